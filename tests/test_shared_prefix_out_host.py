"""nsn_shared_prefix_attention refuses an output that overlaps the queries, before any
launch (fake, never dereferenced addresses)."""
import pytest

from nsn_amd import _lib

A = 1 << 20


@pytest.mark.parametrize("shift", [16, 256, -256, 4 * 8 * 256 - 16, -(4 * 8 * 256 - 16)])
def test_an_output_across_the_queries_is_refused(shift):
    far = 1 << 30
    side = dict(codes=far, norms=far, mins=far, scales=far, factors=far, blocks=far, block_cap=4, tail=far,
                tail_dtype=_lib.DTYPE_F16, tail_cap=64)
    a = _lib.SharedArgs(q=A, q_dtype=_lib.DTYPE_BF16, batch=4, heads_q=8, heads_kv=2, prefixes=2, scale=0.1, bits=3,
                        prefix_k=_lib.KVSide(**side), prefix_v=_lib.KVSide(**side), k=_lib.KVSide(**side),
                        v=_lib.KVSide(**side), seq_len=far, max_seq_len=100, prefix_splits=1, n_splits=4, workspace=far,
                        out=A + shift, out_dtype=_lib.DTYPE_BF16, status=far)
    assert _lib.lib().nsn_shared_prefix_attention(a, None) == _lib.NSN_EINVAL
