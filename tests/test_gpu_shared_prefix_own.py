"""The own tokens of sequences behind a shared prefix (kernels.shared_prefix_attention):
block counts and lengths that the cache cannot hold.  Which tokens a workgroup's
waves take is checked on the host (test_own_ranges.py); the bounds are those of
test_gpu_shared_prefix.py."""
import pytest
import torch

from tests.test_gpu_shared_prefix import DIM, case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nk,nv", [(-1, -1), (-1000, 0), (0, -1), (3, 3), (1 << 30, 1 << 30)])
@pytest.mark.parametrize("max_seq_len", [40, 2000], ids=["joint", "apart"])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (14, 2)])
def test_own_counts_that_do_not_fit_are_not_read(nk, nv, max_seq_len, hq, hkv):
    """The sequence attends its prefix alone, the others what they did; both the joint
    kernel (short own contexts) and the decode kernel beside it."""
    from nsn_amd import _lib, kernels
    args, dense = case([5, 2], [10, 20, 30, 40], hq, hkv, 3, seed=20)
    q, pk, pv, k, v, seq = args
    clean = kernels.shared_prefix_attention(*args, max_seq_len=max_seq_len)
    check(clean, args, dense)
    k.blocks[1], v.blocks[1] = nk, nv
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernels.shared_prefix_attention(*args, max_seq_len=max_seq_len, check=False, status=st)
    assert int(st.item()) == _lib.ST_CAPACITY
    for b in (0, 2, 3):
        assert torch.equal(out[b], clean[b])
    none = torch.zeros((hkv, 0, DIM), dtype=torch.float64, device="cuda")
    check(out, args, (dense[0], dense[1], [dense[2][0], none, *dense[2][2:]], [dense[3][0], none, *dense[3][2:]]))
