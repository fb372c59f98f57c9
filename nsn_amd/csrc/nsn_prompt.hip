// Causal attention over whole prompts of different lengths laid end to end
// (gfx950): query i of a sequence attends its tokens 0 .. i.
//
//   out[i, h] = sum_{j <= i} p_j v[j, h / G],  p = softmax_j(scale q[i, h] . k[j, h / G])
//
// The reference has no call of this form: it runs one sequence's prompt through
// the model's dense attention (loop_kv_ac08_attention.py:46-96 keeps the
// original forward for prompts).
//
// A row is one query of one of the kv-head's G q-heads, rows query-major (row
// = query * G + head), and a tile 128 consecutive rows: its queries span 128 /
// G tokens, so that one pass over K and V serves the whole group and little is
// computed past the diagonal.  A workgroup of 4 waves takes a tile, 32 rows a
// wave, over blocks of 64 tokens:
//   S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 MFMA; the C layout of S^T is
//   the B layout of P^T for a permuted token order, so P stays in registers;
//   softmax online in the log2 domain (running maximum and sum per row).
// K and V rows go straight to LDS by DMA, one block ahead, into two stages; V
// is transposed as it is read (read_column).  Two workgroups share a CU (64 KB
// of LDS and half the registers each): the two waves of a SIMD belong to
// different ones, so that one's products meet the other's softmax, and one's
// start and end the other's blocks.
//
// Values that are not finite behind a query (padding, a poisoned later token)
// would reach it as 0 times inf: a tile whose output is not finite is done once
// more with such values marked (output_marked).  Finite data pays one barrier and
// one look at its output a tile for it; looking at V's diagonal blocks instead
// cost 4 % of the ragged case.
//
// What bounds it.  Four prompts of 8192 tokens, 16 heads: 1055 to 1095 us, 1042 to
// 1004 TFLOP/s (a 16384^3 library product reaches 1345 on this card); 16 ragged
// prompts of 100 to 2000 tokens, 32:8 heads: 219 to 229 us, 786 to 752 TFLOP/s.
// MFMA are busy 54 % of the SIMDs' cycles at 1.8 GHz, VALU issue 46 %, LDS carries
// 32 KB of operands a wave and block; left out, the K reads are worth 19 %, the DMA
// 15 %, the products 21 %, the exponentials 5 %, the barrier 1 %.  Tiles of 256 rows
// on 8 waves (half the DMA; the two waves of a SIMD kept half a block apart) took
// 1067 and 241 us where these took 1037 and 222.
//
// Work: tiles are numbered by their place in their sequence, the last places
// of all sequences first (the causal work grows with the place), and a
// workgroup finds its (sequence, place) from the offsets on the device.
#include <type_traits>

#include "nsn_rows.hpp"
#include "nsn_tile.hpp"
#include "nsn_wave.hpp"

namespace nsn {
namespace prompt {

using namespace tile;
using wave::wave_max;
using wave::wave_sum;

constexpr int kWaves = 4;
constexpr int kRows = 32 * kWaves;                  // rows of a tile
constexpr int kHalf = kBlockTok * kDim * 2;         // bytes of one side of a stage
constexpr int kStages = 2;
template <int DT> constexpr uint16_t kInf = DT == NSN_DTYPE_BF16 ? 0x7F80 : 0x7C00;
constexpr uint16_t kLargest = 0x7F7F;               // bf16's largest value
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
constexpr int64_t kMaxStride = 1 << 22;             // elements: 64 rows stay within a 32-bit byte offset

struct PromptParams {
    const uint16_t *q, *k, *v;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;     // token and head strides, elements
    uint16_t *out;                                  // [tokens, heads_q, 128]
    int64_t tokens;
    int seqs, heads_q, heads_kv, group;
    float qscale;                                   // scale * log2(e)
    const int32_t *cu;                              // [seqs + 1]
    int32_t *status;
};

// The 16-byte chunk c of token row t sits at chunk position c ^ swz(t) of its
// 256-byte row.  K: an S^T operand read (32 rows, one chunk) takes 16 rows a
// pass, at 16 different slots.  V: read_column reads 4 rows x 64 bytes a pass,
// which (t & 3) << 2 puts into four different quarters of the row.
__device__ __forceinline__ int k_swz(int t) { return t & 15; }
__device__ __forceinline__ int v_swz(int t) { return ((t & 3) << 2) | ((t >> 2) & 3); }

// Sequence s of the first `seqs` as the kernel uses it: its first token and
// length; one whose offsets decrease or leave the token rows has none (and is flagged).
__device__ __forceinline__ void sequence(const PromptParams &p, int s, int seqs, int32_t &start, int32_t &n, bool &bad,
                                         bool &decreases) {
    start = n = 0;
    decreases = false;
    if (s >= seqs) return;
    const int32_t a = p.cu[s], b = p.cu[s + 1];
    decreases = b < a;
    if (a < 0 || decreases || b > p.tokens) {
        bad = true;
        return;
    }
    start = a;
    n = b - a;
}
__device__ __forceinline__ int32_t tiles_of(const PromptParams &p, int32_t n) {
    return static_cast<int32_t>((static_cast<int64_t>(n) * p.group + kRows - 1) / kRows);
}

// Tile t of all sequences' tiles, the last places first: its sequence's first
// token and length and its place z.  False: no such tile.  Sequences behind a
// decrease of the offsets may repeat earlier ones' rows: they are left out, so
// that no row has two tiles and the tiles are no more than the grid's.
__device__ __forceinline__ bool find_tile(const PromptParams &p, int32_t t, bool first_wg, int32_t &start, int32_t &n,
                                          int32_t &z) {
    const int l = threadIdx.x & 63;
    bool bad = false, decreases;
    int seqs = p.seqs;
    auto cut = [&](int s0, int32_t &m) {   // after sequences s0 + l: none from the first decrease on
        const uint64_t at = __ballot(decreases);
        if (at == 0) return;
        seqs = s0 + __ffsll(static_cast<unsigned long long>(at)) - 1;
        if (s0 + l >= seqs) m = 0;
    };
    int32_t st0, n0;
    sequence(p, l, seqs, st0, n0, bad, decreases);
    cut(0, n0);
    const int32_t t0 = tiles_of(p, n0);
    int32_t top = wave_max(t0);
    for (int s = 64; s < seqs; s += 64) {
        int32_t a, m;
        sequence(p, s + l, seqs, a, m, bad, decreases);
        cut(s, m);
        top = max(top, wave_max(tiles_of(p, m)));
    }
    if (first_wg && __ballot(bad) && l == 0) raise_status(p.status, NSN_ST_CAPACITY);
    auto above = [&](int32_t place) {   // tiles at places >= place
        int32_t c = wave_sum(max(0, t0 - place));
        for (int s = 64; s < seqs; s += 64) {
            int32_t a, m;
            sequence(p, s + l, seqs, a, m, bad, decreases);
            c += wave_sum(max(0, tiles_of(p, m) - place));
        }
        return c;
    };
    if (top == 0 || t >= above(0)) return false;
    int32_t lo = 0, hi = top, fhi = 0;   // above(lo) > t >= above(hi) = fhi
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) / 2, f = above(mid);
        if (f > t) {
            lo = mid;
        } else {
            hi = mid;
            fhi = f;
        }
    }
    z = lo;
    int32_t r = t - fhi;   // the r-th sequence with more than z tiles
    for (int s = 0; s < seqs; s += 64) {
        int32_t a = st0, m = n0;
        if (s) sequence(p, s + l, seqs, a, m, bad, decreases);
        const uint64_t has = __ballot(tiles_of(p, m) > z);
        const int32_t c = __popcll(has);
        if (r >= c) {
            r -= c;
            continue;
        }
        const int32_t rank = __popcll(has & ((1ull << l) - 1));
        const int lane = __ffsll(static_cast<unsigned long long>(__ballot(((has >> l) & 1) && rank == r))) - 1;
        start = __builtin_amdgcn_readlane(a, lane);
        n = __builtin_amdgcn_readlane(m, lane);
        return true;
    }
    return false;
}

// One tile; true: it is to be done again, marked (written: this wave's rows
// are out and stay).  LO (bf16): the softmax weights enter the PV product and the
// sums as bf16 hi + lo (~2^-17 relative) instead of one bf16 rounding, for the
// tiles whose first queries attend a handful of tokens, where one weight's
// rounding moves the output by up to 2^-9 of |v|.
template <int DT, bool LO>
__device__ __forceinline__ bool attend_tile(const PromptParams &p, uint8_t (&stg)[kStages][2 * kHalf], int &again, int kvh,
                                            int64_t start, int32_t n, int32_t z, bool marked, bool &written) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   // (nothing of a tile is kept for its second time)
    asm volatile("" : "+s"(z));
    const int l = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = l & 31, h = l >> 5;
    // ---- DMA: instruction i of a side fills rows 4i .. 4i + 3 (lane l: row 4i
    // + l / 16, position l % 16); a wave issues i = 4 wave .. 4 wave + 3 of each
    // side, at offsets that stay the same from block to block.  Rows past the
    // sequence repeat its last token (masked).
    const int drow = 16 * wave + (l >> 4), pos = l & 15;
    const uint32_t kb = static_cast<uint32_t>(p.k_ts) * 2, vb = static_cast<uint32_t>(p.v_ts) * 2;
    const uint16_t *kbase = p.k + start * p.k_ts + kvh * p.k_hs, *vbase = p.v + start * p.v_ts + kvh * p.v_hs;
    uint32_t koff[4], voff[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int row = drow + 4 * x;
        koff[x] = row * kb + 16u * (pos ^ k_swz(row));
        voff[x] = row * vb + 16u * (pos ^ v_swz(row));
    }
    auto stage = [&](int j) __attribute__((always_inline)) {
        const int t0 = j * kBlockTok;
        const int last = n - 1 - t0;
        uint8_t *dst = stg[j % kStages] + 4096 * wave;
        const uint16_t *ks = kbase + static_cast<int64_t>(t0) * p.k_ts, *vs = vbase + static_cast<int64_t>(t0) * p.v_ts;
        if (last >= kBlockTok - 1) {   // (uniform)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                dma16s(ks, koff[x], dst + 1024 * x);
                dma16s(vs, voff[x], dst + 1024 * x + kHalf);
            }
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int row = drow + 4 * x;
                const uint32_t past = static_cast<uint32_t>(row > last ? row - last : 0);
                dma16s(ks, koff[x] - past * kb, dst + 1024 * x);
                dma16s(vs, voff[x] - past * vb, dst + 1024 * x + kHalf);
            }
        }
    };
    stage(0);
    if (tid == 0 && !marked) again = 0;   // (before the first block's barrier)

    int G = p.group;
    asm volatile("" : "+s"(G));   // (the divisions wait until the fetch is on its way)
    const int rows = n * G;                      // (< 2^30 + G, by the host's bound on the grid)
    const int r0 = z * kRows, rw = r0 + 32 * wave;
    const int r = rw + col, rr = r < rows ? r : rows - 1;
    const int qi = rr / G;
    const int64_t head = static_cast<int64_t>(kvh) * G + (rr - qi * G);
    const int q_last = ((r0 + kRows < rows ? r0 + kRows : rows) - 1) / G;
    const int nblk = q_last / kBlockTok + 1;
    // this wave's queries: blocks [0, jend) reach them, the mask starts at the first one's block
    const int w_first = rw / G, w_last = ((rw + 32 < rows ? rw + 32 : rows) - 1) / G;
    const int jend = rw < rows ? w_last / kBlockTok + 1 : 0, jfull = rw < rows ? (w_first + 1) / kBlockTok : 0;

    // ---- Q fragments (B operand of S^T = K Q^T): row rw + l % 32, channels 16 ks + 8 h ..
    u32x4 qf[8];
    const uint16_t *qrow = p.q + (start + qi) * p.q_ts + head * p.q_hs + 8 * h;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) qf[ks] = *reinterpret_cast<const u32x4 *>(qrow + 16 * ks);

    f32x16 acc[4];   // O^T tiles: channels 32 ct + 8 (i / 4) + 4 h + i % 4 of the lane's row
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[ct][i] = 0.f;
    float m_run = -INFINITY, lsum = 0.f;   // (lsum: this lane's half of the row's tokens)

    // S^T[token][row]: register i of s[tt] holds token 32 tt + 8 (i / 4) + 4 h + i % 4
    f32x16 s[2];
    const int kx = 16 * (h ^ (col & 15));
    auto scores = [&](int j) __attribute__((always_inline)) {
        const uint8_t *kj = stg[j % kStages] + 256 * col;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[tt][i] = 0.f;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const u32x4 a = *reinterpret_cast<const u32x4 *>(kj + 8192 * tt + (kx ^ (32 * ks)));
                s[tt] = mfma<DT>(a, qf[ks], s[tt]);
            }
        mfma_order<16, 1>();
        __builtin_amdgcn_s_setprio(0);
    };
    u32x4 pb[4];              // P^T B operands of the 16-token steps (LO: the bf16 hi parts)
    u32x4 pl[LO ? 4 : 1];
    auto softmax = [&](int j, bool masked) __attribute__((always_inline)) {
        if (masked) {
            const int lim = qi - j * kBlockTok;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * tt + 8 * (i >> 2) + 4 * h + (i & 3) > lim) s[tt][i] = -INFINITY;
        }
        float mx = max2f(s[0][15], s[1][15]);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const float a0 = max3f(s[tt][0], s[tt][1], s[tt][2]), a1 = max3f(s[tt][3], s[tt][4], s[tt][5]);
            const float a2 = max3f(s[tt][6], s[tt][7], s[tt][8]), a3 = max3f(s[tt][9], s[tt][10], s[tt][11]);
            const float a4 = max3f(s[tt][12], s[tt][13], s[tt][14]);
            mx = max3f(mx, max3f(a0, a1, a2), max2f(a3, a4));
        }
        mx = halves_max(mx) * p.qscale;   // (the queries stay exact: scores scale here and inside the exponent)
        if (__builtin_amdgcn_ballot_w64(mx > m_run + kLazy)) {
            const float mnew = fmaxf(m_run, mx);
            float alpha = (m_run == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - mnew);
            if (marked) alpha = fmaxf(alpha, 0x1p-126f);   // (an inf stays one: no 0 times it)
            lsum *= alpha;
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) acc[ct] *= alpha;
            m_run = mnew;
        }
        const float msafe = (m_run == -INFINITY) ? 0.f : m_run;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float v = s[c >> 1][8 * (c & 1) + 2 * e + x];
                    w[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(v, p.qscale, -msafe));
                }
                if constexpr (LO) split_bf16(w[0], w[1], hi[e], lo[e]);
                else hi[e] = pk<DT>(w[0], w[1]);
                // the row sum takes the rounded weights that the PV product uses
                lsum = add_pair<DT>(hi[e], lsum);
                if constexpr (LO) lsum = add_pair<DT>(lo[e], lsum);
            }
            pb[c] = u32x4{hi[0], hi[1], hi[2], hi[3]};
            if constexpr (LO) pl[c] = u32x4{lo[0], lo[1], lo[2], lo[3]};
        }
    };
    // O^T[channel][row] += V^T P^T over the block's four 16-token steps.  Lane
    // l of a read addresses token 16 c + 8 x + 4 h + (l % 16) / 4, channels 32
    // ct + 16 ((l / 16) % 2) + 4 (l % 4) .. + 3.
    uint32_t vx[4];
    {
        const int i = l & 15, tr = i >> 2;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
            vx[ct] = kHalf + 256 * (4 * h + tr) + 64 * (ct ^ tr) + 16 * ((2 * ((l >> 4) & 1) + ((i & 3) >> 1)) ^ h) + 8 * (i & 1);
    }
    auto output = [&](int j) __attribute__((always_inline)) {
        const uint8_t *vj = stg[j % kStages];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int ct = 0; ct < 4; ++ct) {
                const u32x2 a0 = read_column(vj + vx[ct] + 4096 * c);
                const u32x2 a1 = read_column(vj + (vx[ct] ^ 32) + 4096 * c + 2048);   // (x = 1: the slot's bit 1)
                const u32x4 a = {a0[0], a0[1], a1[0], a1[1]};
                acc[ct] = mfma<DT>(a, pb[c], acc[ct]);
                if constexpr (LO) acc[ct] = mfma<DT>(a, pl[c], acc[ct]);
            }
        mfma_order<16, LO ? 2 : 1, 2>();
        __builtin_amdgcn_s_setprio(0);
    };

    // The mask takes a token out of the scores; its weight is an exact 0, and 0
    // times a finite value adds nothing, but times inf or NaN it would.  Here such
    // a value leaves the product, and for every row that attends it further ones
    // add (bf16's largest)^2, past fp32's range: once with its sign for an inf
    // (whatever its weight, which is positive), with both for a NaN.  Only a tile
    // whose output was not finite takes this path, a second time through its blocks.
    auto output_marked = [&](int j) __attribute__((always_inline)) {
        const uint8_t *vj = stg[j % kStages];
        int lim = qi - j * kBlockTok;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
            asm volatile("" : "+v"(lim));   // (the marks of the rows are made again: they would not fit the registers)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                __builtin_amdgcn_sched_barrier(0);
                const u32x2 a0 = read_column(vj + vx[ct] + 4096 * c);
                const u32x2 a1 = read_column(vj + (vx[ct] ^ 32) + 4096 * c + 2048);
                u32x4 a = {a0[0], a0[1], a1[0], a1[1]}, plus, minus, attended;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t pair = a[e];
                    const u16x2 past = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, pair & 0x7fff7fffu),
                                                                     u16x2{kInf<DT> - 1, kInf<DT> - 1});
                    const u16x2 one = __builtin_elementwise_min(past, u16x2{1, 1});   // 1 where not finite
                    const u16x2 nan = __builtin_elementwise_min(past - one, u16x2{1, 1});
                    const u16x2 negative = __builtin_bit_cast(u16x2, pair) >> u16x2{15, 15};
                    plus[e] = __builtin_bit_cast(uint32_t, (one & (nan | (negative ^ u16x2{1, 1}))) * u16x2{kLargest, kLargest});
                    minus[e] = __builtin_bit_cast(uint32_t, (one & (nan | negative)) * u16x2{kLargest | 0x8000, kLargest | 0x8000});
                    a[e] &= __builtin_bit_cast(uint32_t, one - u16x2{1, 1});
                    const int i = 8 * (c & 1) + 2 * e, t = 32 * (c >> 1) + 8 * (i >> 2) + 4 * h + (i & 3);
                    attended[e] = (t <= lim ? kLargest : 0u) | (t + 1 <= lim ? uint32_t{kLargest} << 16 : 0u);
                }
                acc[ct] = mfma<DT>(a, pb[c], acc[ct]);
                if constexpr (LO) acc[ct] = mfma<DT>(a, pl[c], acc[ct]);
                asm volatile("" : "+v"(lim));
                acc[ct] = mfma<NSN_DTYPE_BF16>(plus, attended, acc[ct]);
                acc[ct] = mfma<NSN_DTYPE_BF16>(minus, attended, acc[ct]);
            }
        }
    };

    // ---- the blocks.  Block j is taken when it has landed and every wave has
    // left block j - 1, whose stage block j + 1 then goes into.
    auto begin = [&](int j) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (j + 1 < nblk) stage(j + 1);
        __builtin_amdgcn_sched_barrier(0);
    };
    int j = 0;
    for (; !LO && !marked && j < jfull; ++j) {   // (a tile of first queries has at most one such block a wave)
        begin(j);
        scores(j);
        softmax(j, false);
        output(j);
    }
    for (; j < nblk; ++j) {   // the diagonal (a loop of its own: the other one carries no mask), all blocks of a marked tile
        begin(j);
        if (j >= jend) continue;
        scores(j);
        softmax(j, true);
        if (marked) output_marked(j);
        else output(j);
    }

    // ---- O = O^T / sum.  A wave with a value that is not finite writes nothing
    // the first time: the output may lie in the queries' place, which it reads again.
    const float rl = 1.f / halves_sum(lsum);
    bool bad = false;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[ct][i] *= rl;
            bad |= !finite(acc[ct][i]);
        }
    const bool redo = __builtin_amdgcn_ballot_w64(bad && r < rows) != 0;   // (uniform)
    if (r < rows && (marked ? !written : !redo)) {
        int ro = r;   // (its query and head once more: kept across the blocks they cost a spill)
        asm volatile("" : "+v"(ro));
        const int qo = ro / G;
        uint16_t *dst = p.out + ((start + qo) * p.heads_q + static_cast<int64_t>(kvh) * G + (ro - qo * G)) * kDim + 8 * h;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                // the lane's 4 channels of c and of c + 1 against those of lane ^ 32: 8 channels of one
                uint32_t w[2][2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int i = 4 * (c + x);
                    w[x][0] = pk<DT>(acc[ct][i], acc[ct][i + 1]);
                    w[x][1] = pk<DT>(acc[ct][i + 2], acc[ct][i + 3]);
                }
                const auto a = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                const auto b = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                *reinterpret_cast<u32x4 *>(dst + 32 * ct + 8 * c) = u32x4{a[0], b[0], a[1], b[1]};
            }
    }
    if (marked) {
        if (bad && r < rows && !written) raise_status(p.status, NSN_ST_NONFINITE_OUTPUT);
        return false;
    }
    written = !redo;
    if (redo && l == 0) again = 1;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();   // (also: every wave has left the stages)
    asm volatile("" ::: "memory");
    return again != 0;
}

template <int DT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void prompt_kernel(PromptParams p) {
    __shared__ __align__(16) uint8_t stg[kStages][2 * kHalf];
    __shared__ int again;
    const uint32_t hkv = static_cast<uint32_t>(p.heads_kv);
    const int kvh = static_cast<int>(blockIdx.x % hkv);   // (fastest: a kv-head's tiles meet in few L2s)
    int32_t start, n, z;
    if (!find_tile(p, static_cast<int32_t>(blockIdx.x / hkv), blockIdx.x == 0 && threadIdx.x < 64, start, n, z)) return;
    // queries up to the 64th: weights as hi + lo
    const bool first = DT == NSN_DTYPE_BF16 && static_cast<int64_t>(z) * kRows < static_cast<int64_t>(kBlockTok) * p.group;
    bool written = false;
    for (bool marked = false, more = true; more; marked = true) {
        if (first) more = attend_tile<DT, DT == NSN_DTYPE_BF16>(p, stg, again, kvh, start, n, z, marked, written);
        else more = attend_tile<DT, false>(p, stg, again, kvh, start, n, z, marked, written);
        more = more && !marked;
    }
}

}  // namespace prompt
}  // namespace nsn

using namespace nsn;

extern "C" int nsn_prompt_attention(const nsn_prompt_args *a, nsn_stream_t stream) {
    using namespace nsn::prompt;
    if (!a || a->tokens < 0 || a->seqs < 0 || a->heads_q <= 0 || a->heads_kv <= 0 || a->heads_q % a->heads_kv)
        return NSN_EINVAL;
    if (a->dtype != NSN_DTYPE_F16 && a->dtype != NSN_DTYPE_BF16) return NSN_EINVAL;
    if (!(a->scale > 0.f) || !__builtin_isfinite(a->scale)) return NSN_EINVAL;
    if (a->tokens == 0 || a->seqs == 0) return NSN_OK;
    if (!a->q || !a->k || !a->v || !a->out || !a->cu_seqlens) return NSN_EINVAL;
    for (const void *ptr : {a->q, a->k, a->v, static_cast<const void *>(a->out)})
        if (reinterpret_cast<uintptr_t>(ptr) & 15u) return NSN_EINVAL;
    for (int64_t st : {a->q_token_stride, a->q_head_stride, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                       a->v_head_stride})
        if (st < 0 || (st & 7) || st > kMaxStride) return NSN_EINVAL;
    constexpr int64_t kMaxGrid = 1 << 22;   // workgroups (2^31 threads)
    const int64_t group = a->heads_q / a->heads_kv;
    // a sequence's last tile may be partly filled; empty sequences have none
    if (a->tokens > 0x7fffffff || a->seqs > 0x7fffff00 || group > kRows * kMaxGrid / a->tokens) return NSN_EINVAL;
    const int64_t tiles = a->tokens * group / kRows + (a->seqs < a->tokens ? a->seqs : a->tokens);
    if (tiles > kMaxGrid / a->heads_kv) return NSN_EINVAL;   // (more rows than memory holds)
    // the output in the queries' place, row for row, or apart from all inputs
    const uintptr_t lo = reinterpret_cast<uintptr_t>(a->out), hi = lo + a->tokens * a->heads_q * kDim * 2;
    auto meets = [&](const void *x, int64_t heads, int64_t ts, int64_t hs) {
        return rows_meet(reinterpret_cast<uintptr_t>(x), a->tokens, heads, 2 * ts, 2 * hs, kDim * 2, lo, hi);
    };
    const bool in_place = a->q == a->out && (a->tokens == 1 || a->q_token_stride == a->heads_q * kDim) &&
                          (a->heads_q == 1 || a->q_head_stride == kDim);
    if ((!in_place && meets(a->q, a->heads_q, a->q_token_stride, a->q_head_stride)) ||
        meets(a->k, a->heads_kv, a->k_token_stride, a->k_head_stride) ||
        meets(a->v, a->heads_kv, a->v_token_stride, a->v_head_stride))
        return NSN_EINVAL;
    PromptParams p{};
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k);
    p.v = static_cast<const uint16_t *>(a->v);
    p.q_ts = a->q_token_stride;
    p.q_hs = a->q_head_stride;
    p.k_ts = a->k_token_stride;
    p.k_hs = a->k_head_stride;
    p.v_ts = a->v_token_stride;
    p.v_hs = a->v_head_stride;
    p.out = static_cast<uint16_t *>(a->out);
    p.tokens = a->tokens;
    p.seqs = static_cast<int>(a->seqs);
    p.heads_q = static_cast<int>(a->heads_q);
    p.heads_kv = static_cast<int>(a->heads_kv);
    p.group = static_cast<int>(group);
    p.qscale = a->scale * kLog2e;
    p.cu = a->cu_seqlens;
    p.status = a->status;
    const dim3 grid(static_cast<unsigned>(tiles * a->heads_kv));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (a->dtype == NSN_DTYPE_BF16) hipLaunchKernelGGL(prompt_kernel<NSN_DTYPE_BF16>, grid, dim3(64 * kWaves), 0, st, p);
    else hipLaunchKernelGGL(prompt_kernel<NSN_DTYPE_F16>, grid, dim3(64 * kWaves), 0, st, p);
    return hipGetLastError() == hipSuccess ? NSN_OK : NSN_ELAUNCH;
}
