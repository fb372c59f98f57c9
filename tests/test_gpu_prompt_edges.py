"""Prompt attention at the edges of its contract: offsets of sequences that repeat
rows, values that are not finite, an output in the queries' place.  The bounds
are those of test_gpu_prompt.py."""
import pytest
import torch

from tests.test_gpu_prompt import check, make

pytestmark = pytest.mark.gpu


def offsets(*cu):
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2)])
def test_sequences_behind_a_decrease_are_left_out(hq, hkv):
    """[0, N) again and again: the first one is whole, whatever the others would cover."""
    from nsn_amd import _lib, kernels
    N = 1280
    q, k, v, cu = make([N], hq, hkv, torch.bfloat16, 31)
    want = kernels.prompt_attention(q, k, v, cu)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    for many in (offsets(0, N, 0, N, 0, N), offsets(*[0, N] * 3000)):
        st.zero_()
        out = torch.full_like(q, 9.0)
        kernels.prompt_attention(q, k, v, many, status=st, check=False, out=out)
        assert int(st.item()) == _lib.ST_CAPACITY
        assert torch.equal(out, want)


@pytest.mark.parametrize("at", [0, 40, 63, 64, 70, 149])
def test_a_decrease_among_many_sequences(at):
    from nsn_amd import _lib, kernels
    lens = [3 + (5 * i) % 17 for i in range(150)]
    q, k, v, cu = make(lens, 4, 2, torch.float16, 32)
    want = kernels.prompt_attention(q, k, v, cu)
    keep = int(cu[at])
    bad = cu.clone()
    bad[at + 1:] -= int(cu[at + 1]) - keep + 1          # sequence `at` would end a row before it starts
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    kernels.prompt_attention(q, k, v, bad, status=st, check=False, out=out)
    assert int(st.item()) & _lib.ST_CAPACITY
    assert torch.equal(out[:keep], want[:keep]) and bool((out[keep:] == 9).all())
    check(want, q, k, v, lens)


def test_offsets_that_leave_the_rows_leave_one_sequence_out():
    from nsn_amd import _lib, kernels
    q, k, v, cu = make([30, 40, 50], 4, 2, torch.bfloat16, 33)
    want = kernels.prompt_attention(q, k, v, cu)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad, rows in ((offsets(-1, 30, 70, 120), slice(30, 120)), (offsets(0, 30, 70, 121), slice(0, 70))):
        st.zero_()
        out = torch.full_like(q, 9.0)
        kernels.prompt_attention(q, k, v, bad, status=st, check=False, out=out)
        assert int(st.item()) == _lib.ST_CAPACITY
        assert torch.equal(out[rows], want[rows])
        out[rows] = 9.0
        assert bool((out == 9).all())
