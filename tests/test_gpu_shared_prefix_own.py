"""The own tokens of sequences behind a shared prefix (kernels.shared_prefix_attention):
block counts that the cache cannot hold, several blocks for each wave of the joint
kernel, sequences without a prefix.  Which tokens a workgroup's waves take is
checked on the host (test_own_ranges.py); the bounds are those of
test_gpu_shared_prefix.py."""
import pytest
import torch

from nsn_amd.kernels import PackedKV
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


# own contexts that the joint kernel takes (up to max(10, streams / 6) blocks of the
# longest), of several packed blocks for each of its four waves, and just past it
@pytest.mark.parametrize("bits", [3, 5])
@pytest.mark.parametrize("hq,hkv,own", [(4, 1, [640, 639]), (7, 1, [640, 577]), (8, 1, [641, 640]), (2, 1, [333, 640])])
def test_several_own_blocks_a_wave(hq, hkv, own, bits):
    from nsn_amd import kernels
    for tail in (torch.float16, torch.bfloat16):
        args, dense = case([5], own, hq, hkv, bits, tail=tail, seed=21)
        out = kernels.shared_prefix_attention(*args)
        check(out, args, dense)
        assert torch.equal(kernels.shared_prefix_attention(*args), out)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (32, 8), (56, 8)])
@pytest.mark.parametrize("longest", [1344, 1345])
def test_many_streams_with_longer_own_contexts(hq, hkv, longest):
    """16 sequences x 8 kv-heads: 21 blocks are the joint kernel's, 22 the decode kernel's."""
    from nsn_amd import kernels
    own = [longest] + [600 + 47 * i for i in range(15)]
    args, dense = case([3, 9], own, hq, hkv, 3, seed=22)
    out = kernels.shared_prefix_attention(*args)
    check(out, args, dense)
    assert torch.equal(kernels.shared_prefix_attention(*args), out)


def test_a_row_beside_an_empty_one_without_a_prefix():
    """Sequences 2 and 3 continue an empty prefix: 2 holds nothing, 3 attends its own tokens alone."""
    from nsn_amd import _lib, kernels
    for own in ([0, 40, 0, 3], [70, 1, 0, 150]):
        args, dense = case([6, 0], own, 4, 2, 3, seed=23)
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = kernels.shared_prefix_attention(*args, max_seq_len=max(own), status=st, check=False)
        assert int(st.item()) == _lib.ST_EMPTY and bool((out[2] == 0).all())
        q, _, _, _, _, seq = args
        rows = (0, 1, 3)
        for b in rows:
            pick = [[dense[i][b // 2]] for i in (0, 1)] + [[dense[i][b]] for i in (2, 3)]
            pk, pv = (PackedKV(s.codes[p:p + 1], s.norm[p:p + 1], s.min[p:p + 1], s.scale[p:p + 1], s.factor[p:p + 1],
                               s.blocks[p:p + 1], None, s.bits) for s, p in ((args[1], b // 2), (args[2], b // 2)))
            check(out[b:b + 1], (q[b:b + 1], pk, pv, args[3], args[4], seq[b:b + 1]), pick)


@pytest.mark.parametrize("max_seq_len", [40, 2000], ids=["joint", "apart"])
def test_the_output_may_be_the_queries_memory(max_seq_len):
    from nsn_amd import kernels
    from nsn_amd.errors import IntegrityError
    args, dense = case([5, 2], [10, 20, 30, 40], 14, 2, 3, seed=24)
    q = args[0]
    want = kernels.shared_prefix_attention(*args, max_seq_len=max_seq_len)
    room = torch.empty((6, 14, DIM), dtype=q.dtype, device="cuda")
    room[1:5] = q
    for out in (room[:4], room[2:]):
        with pytest.raises(IntegrityError, match="overlaps"):
            kernels.shared_prefix_attention(room[1:5], *args[1:], max_seq_len=max_seq_len, out=out)
    got = kernels.shared_prefix_attention(*args, max_seq_len=max_seq_len, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
