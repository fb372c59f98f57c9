"""Decode behind a shared prefix whose V tokens differ by orders of magnitude: every
bound is relative to what the row attends, not to the largest value of the prefix.

Tolerance, per output value: as in test_gpu_shared_prefix.py with A = sum_t p_t |v_t|,
but for the terms that hold the prefix's values in fp16, with F = sum_t p_t f_V[t]:
a direction's 2^-17 counts for each token as far as it is attended, 2^-17 F, and a
weight times f_V is rounded by 2^-11 of itself (in A) or 2^-25 of a unit that the
row's largest such product exceeds 2^11 times: n 2^-36 F.  ds is the largest error
of a score among the tokens whose weight passes 2^-40 (the others stay below
n 2^-39 of the row)."""
import math

import pytest
import torch

from tests.test_gpu_shared_prefix import DIM, SCALE, U, packed

pytestmark = pytest.mark.gpu


def encode(x, bits):
    """x [P, heads, n, 128] (n a multiple of 64) as (PackedKV, restored [P][heads, n, 128] in 64 bits)."""
    from nsn_amd import cache, codec
    P, heads, n, _ = x.shape
    kv, _ = cache.pack_sequences(x, [n] * P, bits=bits, tail_dtype=torch.float16)
    grp = {"codes": kv.codes[:, :, :n // 64].contiguous(),
           "metas": tuple(t[:, :, :n // 64].contiguous().reshape(P, heads, n // 64, *s) for t, s in
                          ((kv.norm, (64, 1)), (kv.min, (1, DIM)), (kv.scale, (1, DIM))))}
    return kv, list(codec.restore_group(grp, torch.float32).double())


def check(got, q, pk, pv, pkd, pvd, kd, vd):
    B, hq, _ = q.shape
    P, hkv, n = len(pkd), pkd[0].shape[0], pkd[0].shape[1]
    for b in range(B):
        p = b // (B // P)
        K, V = torch.cat((pkd[p], kd[b]), 1), torch.cat((pvd[p], vd[b]), 1)
        qq = q[b].double().reshape(hkv, hq // hkv, DIM)
        w = torch.softmax((qq @ K.transpose(1, 2)) * SCALE, -1)
        o, A = w @ V, w @ V.abs()
        fk, fv = (s.factor[p, :, :n // 64].reshape(hkv, 1, n).double() for s in (pk, pv))
        F = (w[..., :n] * fv).sum(-1, keepdim=True)
        ds = ((qq.abs() @ pkd[p].abs().transpose(1, 2)) * 2.0 ** -11
              + qq.abs().sum(-1, keepdim=True) * fk * 2.0 ** -17) * SCALE
        ds = torch.where(w[..., :n] > 2.0 ** -40, ds, torch.zeros_like(ds)).amax(-1, keepdim=True)
        tol = ((2 * ds + 2 * 2.0 ** -11 + 2.0 ** -14 + 2.0 ** -15) * A + (2.0 ** -17 + n * 2.0 ** -36) * F
               + U[got.dtype] * o.abs() + 2.0 ** -24 * A.amax(-1, keepdim=True) + 1e-30)
        err = (got[b].double().reshape(o.shape) - o).abs()
        assert bool((err <= tol).all()), f"sequence {b}: max err/tol {(err / tol).max().item():.3f}"


def run(q, kx, vx, bits, own, seed, qdt=torch.bfloat16, odt=torch.bfloat16, vscale=1.0):
    from nsn_amd import kernels
    g = torch.Generator(device="cuda").manual_seed(seed)
    hkv = kx.shape[1]
    pk, pkd = encode(kx.half(), bits)
    pv, pvd = encode(vx.half(), bits)
    k, kd = packed(g, own, hkv, bits, torch.float16)
    v, vd = packed(g, own, hkv, bits, torch.float16)
    v.tail.mul_(vscale)
    vd = [x * vscale for x in vd] if vscale else [torch.zeros_like(x) for x in vd]
    seq = torch.tensor(own, dtype=torch.int32, device="cuda")
    for most in (None, 1):   # (1: one split, so that a wave walks several blocks)
        out = kernels.shared_prefix_attention(q.to(qdt), pk, pv, k, v, seq, out_dtype=odt, max_prefix_blocks=most)
        check(out, q.to(qdt), pk, pv, pkd, pvd, kd, vd)


def drawn(seed, P, B, hq, hkv, n):
    """Positive queries, and keys that an all-ones direction moves up or down for every query."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")   # noqa: E731
    return rnd(B, hq, DIM).abs() * 0.5 + 0.5, rnd(P, hkv, n, DIM) * 0.3, rnd(P, hkv, n, DIM)


HEADS = [(2, 2), (14, 2), (32, 4)]


@pytest.mark.parametrize("bits", [3, 5])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("at", [0, 31, 32, 700, 1279])
def test_an_outlier_that_no_row_attends(at, hq, hkv, bits):
    """One V token 2^15 times the others' norm, its key far below every other score; one
    token in 100 takes 2^8 times the weight of each of the others, which carry the row."""
    q, kx, vx = drawn(at, 1, 9, hq, hkv, 1280)
    kx = kx * 0.02 + 0.1
    kx[:, :, 50::100] += 0.57    # q . k scale about 5.7 more
    kx[:, :, at] = -6.0          # about -60
    vx = vx * 0.3 + 1.0
    vx /= vx.norm(dim=-1, keepdim=True)
    vx[:, :, at] *= 2.0 ** 15
    run(q, kx, vx, bits, [5, 1, 20, 3, 9, 60, 2, 33, 1], 41, odt=torch.float16, vscale=0.0)


@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("order", ["falling", "rising", "mixed"])
@pytest.mark.parametrize("attended", ["all", "small", "large"])
def test_norms_over_many_orders(hq, hkv, order, attended):
    """Norms from 2^-7 to 2^12 in blocks, with scores that favour nothing, the small or the large tokens."""
    n = 4096
    q, kx, vx = drawn(3, 1, 6, hq, hkv, n)
    kx = kx * 0.02 + 0.1
    kx[:, :, 50::100] += 0.57
    vx = vx * 0.3 + 1.0
    e = torch.linspace(-7, 12, n // 64, device="cuda").round()
    if order == "falling":
        e = e.flip(0)
    elif order == "mixed":
        e = e[torch.randperm(n // 64, generator=torch.Generator().manual_seed(1)).cuda()]
    vx *= torch.exp2(e.repeat_interleave(64))[None, None, :, None] / DIM ** 0.5
    if attended != "all":
        kx += (e.repeat_interleave(64) * (0.12 if attended == "large" else -0.12))[None, None, :, None]
    run(q, kx, vx, 3, [1, 2, 3, 4, 5, 6], 42, odt=torch.float16, vscale=0.0)


@pytest.mark.parametrize("odt", [torch.float16, torch.bfloat16])
def test_small_values_behind_zero_ones(odt):
    """V is exactly 0 for the first blocks and 2^-10 behind them: the small ones keep their bits."""
    q, kx, vx = drawn(4, 2, 8, 8, 2, 1280)
    vx[:, :, :320] = 0.0
    vx[:, :, 320:] *= 2.0 ** -10
    vx[1] = 0.0
    run(q, kx, vx, 3, [1] * 8, 43, odt=odt, vscale=0.0)


@pytest.mark.parametrize("hq,hkv", HEADS)
def test_scores_that_rise_and_fall_by_hundreds(hq, hkv):
    """Every block's scores 40 above (or below) the last one's, past every rescaling of the sums."""
    n = 1280
    for sign in (1, -1):
        q, kx, vx = drawn(5, 1, 5, hq, hkv, n)
        step = torch.arange(n // 64, device="cuda").repeat_interleave(64) * (sign * 4.5)
        kx = kx * 0.1 + (step / 10)[None, None, :, None]
        vx *= torch.exp2((torch.arange(n, device="cuda") % 13) - 6.0)[None, None, :, None]
        run(q, kx, vx, 3, [1, 1, 2, 1, 1], 44)


def test_factors_of_either_sign():
    """A token's factor enters as it is: with its sign turned, in K and V, the token enters with its sign turned."""
    from nsn_amd import kernels
    q, kx, vx = drawn(6, 1, 4, 8, 2, 640)
    g = torch.Generator(device="cuda").manual_seed(45)
    pk, pkd = encode(kx.half(), 3)
    pv, pvd = encode((vx * 300).half(), 3)
    own = [1, 2, 3, 4]
    k, kd = packed(g, own, 2, 3, torch.float16)
    v, vd = packed(g, own, 2, 3, torch.float16)
    turned = (torch.rand(640, generator=g, device="cuda") < 0.5).double()
    for side, dense in ((pk, pkd), (pv, pvd)):
        sign = (1 - 2 * turned).reshape(1, 1, 10, 64)
        side.factor.mul_(sign.float())
        dense[0] *= (1 - 2 * turned)[None, :, None]
    seq = torch.tensor(own, dtype=torch.int32, device="cuda")
    out = kernels.shared_prefix_attention(q.bfloat16(), pk, pv, k, v, seq)
    pk.factor.abs_(), pv.factor.abs_()      # (the bound takes magnitudes)
    check(out, q.bfloat16(), pk, pv, pkd, pvd, kd, vd)
