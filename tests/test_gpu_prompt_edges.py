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


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 4), (5, 1)])
def test_the_output_may_take_the_queries_place(hq, hkv, dt):
    """Over clean values, and where later tokens hold inf and NaN: those tiles are computed twice."""
    from nsn_amd import kernels
    lens = [230, 1, 400, 64]
    for at in (None, 63, 150, 229, 500):
        q, k, v, cu = make(lens, hq, hkv, dt, 34)
        if at is not None:
            v[at, :, 5], v[at, :, 77], k[at + 1, 0, 9] = float("inf"), float("nan"), float("nan")
        st, again = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
        want = kernels.prompt_attention(q, k, v, cu, status=st, check=False)
        got = kernels.prompt_attention(q, k, v, cu, status=again, check=False, out=q)
        assert got.data_ptr() == q.data_ptr()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and torch.equal(st, again)
        assert bool(torch.isfinite(want).all()) == (at is None)


def test_outputs_beside_and_inside_the_inputs():
    from nsn_amd import kernels
    from nsn_amd.errors import IntegrityError
    lens, hq, hkv = [100, 28], 4, 2
    q, k, v, cu = make(lens, hq, hkv, torch.float16, 35)
    want = kernels.prompt_attention(q, k, v, cu)
    # right behind the queries, and in a gap of strided keys
    room = torch.empty((2 * 128, hq, 128), dtype=torch.float16, device="cuda")
    room[:128] = q
    assert torch.equal(kernels.prompt_attention(room[:128], k, v, cu, out=room[128:]), want)
    wide = torch.zeros(128 * (1 << 17), dtype=torch.float16, device="cuda")
    k2 = wide.as_strided((128, hkv, 128), (1 << 17, 128, 1))
    k2.copy_(k)
    gap = wide[256:256 + q.numel()].view(q.shape)
    assert torch.equal(kernels.prompt_attention(q, k2, v, cu, out=gap), want)
    # rows shared with an input
    room[1:129] = q
    for a, b, c, out in ((room[1:129], k, v, room[:128]), (q, k2, v, wide[:q.numel()].view(q.shape))):
        with pytest.raises(IntegrityError, match="shares rows"):
            kernels.prompt_attention(a, b, c, cu, out=out)
    same = make(lens, 4, 4, torch.float16, 36)
    for out in same[1:3]:
        with pytest.raises(IntegrityError, match="shares rows"):
            kernels.prompt_attention(*same, out=out)


def classes(v, at, n, hq):
    """[n, hq, 128] of what values past fp32 leave of the outputs: 0 finite, 1 inf, -1 -inf, 2 NaN, by a running scan."""
    x = v[at:at + n].repeat_interleave(hq // v.shape[1], 1)
    plus, minus, nan = ((f.cumsum(0) > 0) for f in (x == float("inf"), x == float("-inf"), torch.isnan(x)))
    out = plus.int() - minus.int()
    out[nan | (plus & minus)] = 2
    return out


def classes_of(out):
    c = (out == float("inf")).int() - (out == float("-inf")).int()
    c[torch.isnan(out)] = 2
    return c


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 4), (5, 1)])
@pytest.mark.parametrize("marks", [
    [(0, 3, INF), (0, 4, -INF), (0, 5, NAN)], [(70, 3, -INF)], [(229, 3, -INF)],
    [(20, 3, INF), (90, 3, INF), (200, 3, -INF), (10, 40, -INF), (11, 40, INF), (64, 41, -INF), (300, 41, NAN)],
    [(63, 9, -INF), (64, 9, -INF), (63, 10, NAN), (128, 11, INF), (129, 12, -INF), (191, 13, NAN), (192, 14, -INF)]],
    ids=["first", "middle", "last", "several", "borders"])
@pytest.mark.parametrize("sharp", [False, True])
def test_an_attended_value_past_the_numbers_keeps_its_sign_and_kind(marks, hq, hkv, dt, sharp):
    """An inf in V is an inf of its sign in every output that attends it, whatever its
    weight, a NaN (or both signs) a NaN: in the query's own block and in later ones."""
    from nsn_amd import kernels
    lens = [320, 20]
    q, k, v, cu = make(lens, hq, hkv, dt, 37)
    if sharp:
        q = q * 60       # most weights are below 2^-149
    clean = kernels.prompt_attention(q, k, v, cu)
    for tok, ch, x in marks:
        v[tok, :, ch] = x
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernels.prompt_attention(q, k, v, cu, status=st, check=False)
    want = torch.cat([classes(v, 0, 320, hq), classes(v, 320, 20, hq)])
    assert torch.equal(classes_of(out), want.int())
    assert torch.equal(out[want == 0], clean[want == 0])


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_an_inf_survives_larger_scores_behind_it(dt):
    """Token 1's weight falls past fp32's range when token 150's score is seen, three blocks on."""
    from nsn_amd import kernels
    q, k, v, cu = make([200], 4, 2, dt, 38)
    q[:] = 8.0
    k[:] = 0.0
    k[150] = 8.0          # a score of 128 * 64 * scale = 724
    clean = kernels.prompt_attention(q, k, v, cu)
    v[1, :, 2], v[1, :, 3] = -INF, INF
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = kernels.prompt_attention(q, k, v, cu, status=st, check=False)
    want = classes(v, 0, 200, 4)
    assert torch.equal(classes_of(out), want)
    assert torch.equal(out[want == 0], clean[want == 0])
