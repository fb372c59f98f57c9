// Decode attention of sequences that continue a shared packed prefix (gfx950).
//
// One query token per (sequence, q-head).  The fan sequences of a prefix attend
// its packed blocks and, each, their own packed blocks and tail:
//
//   out = sum_t p_t v_t,  p = softmax(scale q . k_t) over prefix and own tokens
//
// The prefix is read once for all of its sequences: their query heads that
// share a kv-head are the rows of one product, fan * G of them.  The own tokens
// take the decode kernel's arithmetic (nsn_segment.hpp); the softmax states of
// both (partials of maximum, weight sum and weighted values) are joined by the
// kernel that follows.  No counterpart in the reference, whose decode reads a
// whole cache per sequence (loop_kv_vf01_kernel.py:56-139).
//
// Prefix kernel.  A workgroup takes 32 * NT rows (NT 1 or 2) of one (prefix,
// kv-head) and a share of its blocks; each of its 8 waves walks a contiguous
// part of the share by itself, in steps of 32 tokens, without barriers:
//   - codes come by DMA, 32 tokens ahead, into the wave's own LDS; a block's
//     metadata with its first half;
//   - K is dequantised in registers straight into the A operand of S^T = K Q^T
//     (32 x 32 x 16 MFMA, fp16): a lane holds one token and 64 channels, code
//     z as the fp16 subnormal z 2^(k-24), and d 2^-7 = (z 2^(k-24)) (s 2^(17-k)) +
//     m 2^-7 is one packed fma per two values.  It rounds d to 2^-11 of itself,
//     below |d| = 2^-7 to 2^-18 (so is a smaller minimum); s 2^17 stays finite for
//     s < 1/2 (an encoder's scales are at most 2/7);
//   - queries are scaled per row by a power of two into fp16's upper range:
//     bf16 and fp16 queries enter exactly (values below 2^-29 of their row's
//     largest lose bits);
//   - the token factor f_K multiplies the fp32 score, f_V the softmax weight,
//     which is then rounded to fp16 once: to 2^-11, or 2^-36 of the row's largest
//     product so far (see kTop); sums and the softmax state are fp32;
//   - V is dequantised like K into the A operand of O^T += V^T P^T: a lane holds
//     4 channels and, per product, 8 tokens in the order of S^T's registers.
// One dequantised operand feeds NT products (two: 32 rows more cost the softmax
// and the products only; 128 rows a wave do not fit the registers).  The waves'
// states are joined in LDS, a workgroup leaves one partial per row; the grid is
// one workgroup per CU (their LDS), whatever the rows and prefixes.
//
// What bounds it.  16 sequences x 32:8 heads behind 32704 3-bit tokens (64 rows
// x 511 blocks x 8 kv-heads, 30 MB): 25.3 us, 1.2 TB/s and 340 TFLOP/s.  Of it
// 3.5 us are the first 32 tokens of all 2048 waves (fetched at once), 15 us
// two blocks a wave -- about 560 VALU instructions and 64 exponentials a half
// beside 32 MFMA, but VALU issue fills only 38 % of the launch's cycles, and the
// first block takes twice the second's time -- and 5 us the join and the partials.
// One loop body for both halves (17 KB of code, no spills) took it from 34.7 to
// 25.8 us, one fma instead of a multiply and an fma and reads a step ahead to
// 24.3; a unit of its own for each row's weights costs 0.6 to 1.
#include "nsn_segment.hpp"
#include "nsn_own_ranges.hpp"
#include "nsn_tile.hpp"
#include "nsn_unpack.hpp"
#include "nsn_wave.hpp"

namespace nsn {
namespace prefix {

using namespace tile;
using unpack::kunpack;
using unpack::Layout;

constexpr int kWaves = 8;
constexpr int kPartStride = 132;
constexpr int kMinBlocks = kWaves;    // blocks of a split, at least: one per wave
constexpr float kLn2 = 0.6931471805599453f;

struct Side {
    const uint8_t *codes;
    const uint16_t *mins, *scales;
    const float *factors;
    const int32_t *blocks;
    int64_t block_cap;
};

struct PrefixParams {
    const uint16_t *q;          // [batch, heads_q, 128]
    int q_bf16;
    int64_t heads_q, heads_kv;
    int group, fan, row_tiles, splits;
    float scale;
    Side k, v;
    float *part;                // [batch, heads_q, splits, 132]
    int32_t *status;
};

// Splits of a prefix of nb blocks: the waves of a split have a block each at least.
__host__ __device__ __forceinline__ int splits_of(int64_t nb, int splits) {
    const int64_t most = (nb + kMinBlocks - 1) / kMinBlocks;
    return static_cast<int>(most < splits ? most : splits);
}
// The prefix's blocks, 0 where the counts do not fit the cache.
__device__ __forceinline__ int prefix_blocks(const Side &k, const Side &v, int64_t p, bool &bad) {
    const int32_t nk = k.blocks[p], nv = v.blocks[p];
    bad = nk != nv || nk < 0 || nk > k.block_cap || nk > v.block_cap;
    return bad ? 0 : nk;
}

// LDS of a wave: two stages of 32 tokens ([K codes | V codes]), two of a
// block's metadata, the block's K scale and min in operand order.
template <int BITS> struct Shape {
    static constexpr int HALF = 32 * 16 * BITS;          // code bytes of 32 tokens, one side
    static constexpr int STAGE = 2 * HALF;
    static constexpr int KMIN = 0, KSCALE = 256, VMIN = 512, VSCALE = 768, KF = 1024, VF = 1280, META = 1536;
    static constexpr int KOP = 512;                      // [16 groups of 8 channels][8 scales | 8 mins]
    static constexpr int WAVE = 2 * STAGE + 2 * META + KOP;
};
template <int NT> struct Lds {
    static constexpr int ROWS = 32 * NT;
    static constexpr int QP = 272;                       // query row pitch: 17 slots of 16 bytes, so that an operand
                                                         // read (32 rows, one chunk) takes 32 different ones
    static constexpr int Q = ROWS * QP;
    static constexpr int ML = kWaves * ROWS * 8;         // the waves' (maximum, sum) per row
    static constexpr int AREA = ROWS * kPartStride * 4;  // a wave's values, rows 33 slots of 16 bytes apart
};
template <int BITS, int NT> constexpr int lds_bytes() {
    const int loop = Lds<NT>::Q + kWaves * Shape<BITS>::WAVE, join = Lds<NT>::ML + 4 * Lds<NT>::AREA;
    return loop > join ? loop : join;
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f16x2 as_h2(uint32_t x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ uint32_t as_u(f16x2 x) { return __builtin_bit_cast(uint32_t, x); }
// Codes as fp16 subnormals z 2^(k-24) -> (m + z s) 2^-kDown, given s 2^(24-kDown-k)
// and m 2^-kDown: one rounding.
constexpr int kDown = 7;
__device__ __forceinline__ uint32_t dequant(uint32_t codes, f16x2 s, f16x2 m) {
    return as_u(__builtin_elementwise_fma(as_h2(codes), s, m));
}

// The unit 2^off in which a row's softmax weights are held.  A weight times f_V
// is rounded to fp16.  The largest such product is put into [2^11, 2^12) (kTopTo)
// when it passes 2^15 (kTop), the first one above 0 at once: a rounding is then
// 2^-11 of its product or 2^-36 of the row's largest, whatever V holds at tokens
// that the row does not attend.  The weights alone stay in fp32's range by their
// scores: they are put to 2^36 when they pass 2^60, which leaves room for any f_V
// of an encoder (2^-25 to 2^17); a first product below 2^-30 counts as that.
constexpr float kTop = 32768.f, kScoreMax = 60.f, kScoreTo = 36.f;
constexpr int kTopTo = 11, kLeast = -30;

// 4 channels of tokens a (low half) and b (high half), given each token's
// 4 * BITS code bits in the low bits of a word: channel c at bit kV4[c].
template <int BITS> struct V4;
template <> struct V4<3> {
    static constexpr int k[4] = {0, 3, 6, 6};
    static __device__ __forceinline__ void pair(uint32_t a, uint32_t b, uint32_t (&D)[4]) {
        const uint32_t X = perm(b, a, 0x05040100u);
        D[0] = X & 0x00070007u;
        D[1] = X & 0x00380038u;
        D[2] = X & 0x01C001C0u;
        D[3] = (X >> 3) & 0x01C001C0u;
    }
};
template <> struct V4<5> {
    static constexpr int k[4] = {0, 5, 5, 2};
    static __device__ __forceinline__ void pair(uint32_t a, uint32_t b, uint32_t (&D)[4]) {
        const uint32_t X = perm(b, a, 0x05040100u), Y = perm(b, a, 0x06050201u);   // bits 0..15, 8..23
        D[0] = X & 0x001F001Fu;
        D[1] = X & 0x03E003E0u;
        D[2] = (X >> 5) & 0x03E003E0u;
        D[3] = (Y >> 5) & 0x007C007Cu;
    }
};

template <int BITS, int NT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void prefix_kernel(PrefixParams p) {
    using S = Shape<BITS>;
    using L = Lds<NT>;
    using LY = Layout<BITS>;
    __shared__ __align__(16) uint8_t smem[lds_bytes<BITS, NT>()];
    __shared__ float c1_s[L::ROWS];
    const int tid = threadIdx.x, l = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = l & 31, h = l >> 5;

    // grid: (unit, row tile), unit = (split, prefix, kv-head), kv-head fastest
    const uint32_t hkv = static_cast<uint32_t>(p.heads_kv);
    const uint32_t units = gridDim.x / static_cast<uint32_t>(p.row_tiles);
    const int rt = static_cast<int>(blockIdx.x / units);
    const uint32_t u = blockIdx.x - static_cast<uint32_t>(rt) * units;
    const int kvh = static_cast<int>(u % hkv);
    const uint32_t ps = u / hkv;
    const int split = static_cast<int>(ps % static_cast<uint32_t>(p.splits));
    const int64_t pre = ps / static_cast<uint32_t>(p.splits);
    const int rows = p.fan * p.group, r0 = rt * L::ROWS;
    auto head_row = [&](int r) {   // row r's (sequence, q-head) of [batch, heads_q]
        const int i = r / p.group;
        return (pre * p.fan + i) * p.heads_q + static_cast<int64_t>(kvh) * p.group + (r - i * p.group);
    };

    bool bad_counts;
    const int nb = prefix_blocks(p.k, p.v, pre, bad_counts);
    if (bad_counts && tid == 0) raise_status(p.status, NSN_ST_CAPACITY);
    const int splits = splits_of(nb, p.splits);
    if (split >= splits) return;
    const uint32_t share = static_cast<uint32_t>(nb) / static_cast<uint32_t>(splits);
    const int extra = nb - static_cast<int>(share) * splits;
    const int s0 = split * static_cast<int>(share) + (split < extra ? split : extra);
    const int sn = static_cast<int>(share) + (split < extra);   // (the wave's part: below 2^28)
    const int b0 = s0 + (sn * wave) / kWaves, b1 = s0 + (sn * (wave + 1)) / kWaves;

    // ---- DMA of the wave's codes and metadata
    uint8_t *const ws = smem + L::Q + wave * S::WAVE;
    uint8_t *const meta = ws + 2 * S::STAGE;
    uint32_t *const kop = reinterpret_cast<uint32_t *>(meta + 2 * S::META);
    const int64_t kr = (pre * p.heads_kv + kvh) * p.k.block_cap, vr = (pre * p.heads_kv + kvh) * p.v.block_cap;
    const uint8_t *const kcodes = p.k.codes + kr * 2 * S::HALF, *const vcodes = p.v.codes + vr * 2 * S::HALF;
    const int q16 = l & 15;
    const uint16_t *msrc = ((l < 16) ? p.k.mins + kr * kDim : (l < 32) ? p.k.scales + kr * kDim
                          : (l < 48) ? p.v.mins + vr * kDim : p.v.scales + vr * kDim) + 8 * q16;
    const float *fsrc = ((l < 16) ? p.k.factors + kr * kBlockTok : p.v.factors + vr * kBlockTok) + 4 * q16;
    auto stage = [&](int g) __attribute__((always_inline)) {   // half g = 2 * block + (0 | 1)
        const int64_t at = static_cast<int64_t>(g) * S::HALF;
        uint8_t *const dst = ws + (g & 1) * S::STAGE;
#pragma unroll
        for (int i = 0; i < (S::HALF + 1023) / 1024; ++i)
            if (1024 * i + 16 * l < S::HALF) {   // (the last one: half the lanes)
                dma16s(kcodes + at + 1024 * i, 16u * l, dst + 1024 * i);
                dma16s(vcodes + at + 1024 * i, 16u * l, dst + S::HALF + 1024 * i);
            }
        if (!(g & 1)) {
            uint8_t *const md = meta + ((g >> 1) & 1) * S::META;
            dma16(msrc + static_cast<uint64_t>(static_cast<uint32_t>(g >> 1)) * kDim, md);
            if (l < 32) dma16(fsrc + static_cast<uint64_t>(static_cast<uint32_t>(g >> 1)) * kBlockTok, md + S::KF);
        }
    };
    if (b0 < b1) stage(2 * b0);

    // ---- queries: row r0 + tid / 8, 16 channels a thread, into LDS in operand
    // order: chunk 2 ks + h holds channels 64 h + 8 ks + chE[e]
    if (tid < 8 * L::ROWS) {
        const int row = tid >> 3, part = tid & 7, r = r0 + row;
        const bool valid = r < rows;
        const uint4 *qp = reinterpret_cast<const uint4 *>(p.q + head_row(valid ? r : rows - 1) * kDim + 16 * part);
        const uint4 w0 = qp[0], w1 = qp[1];
        const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        float x[16], mx = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint16_t b = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
            x[e] = valid ? (p.q_bf16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b)) : 0.f;
            mx = fmaxf(mx, fabsf(x[e]));
            bad |= !finite(x[e]);
        }
        if (bad) raise_status(p.status, NSN_ST_NONFINITE_ATTN_INPUT);
        mx = fmaxf(mx, __shfl_xor(mx, 1));
        mx = fmaxf(mx, __shfl_xor(mx, 2));
        mx = fmaxf(mx, __shfl_xor(mx, 4));
        // sigma: max|q| 2^sigma in [2^14, 2^15)
        int e2 = 0;
        (void)frexpf(mx, &e2);
        int sigma = (mx > 0.f && finite(mx)) ? 15 - e2 : 0;
        sigma = sigma < -100 ? -100 : (sigma > 100 ? 100 : sigma);
        const float pw = ldexpf(1.f, sigma);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int grp = 2 * part + g, ks = grp & 7, hh = grp >> 3;
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = pk<NSN_DTYPE_F16>(x[8 * g + LY::chE[2 * i]] * pw, x[8 * g + LY::chE[2 * i + 1]] * pw);
            *reinterpret_cast<u32x4 *>(smem + row * L::QP + 16 * (2 * ks + hh)) = u32x4{o[0], o[1], o[2], o[3]};
        }
        if (part == 0) c1_s[row] = p.scale * kLog2e * ldexpf(1.f, kDown - sigma);
    }
    __syncthreads();

    // acc and lsum hold weights times 2^-off: a power of two of its own for each row,
    // as far below the largest weight times f_V seen as fp16 allows (see kTop)
    float c1[NT], off[NT], top[NT], lsum[NT];
    f32x16 acc[NT][4];   // O^T: register i of tile ct is channel 4 (8 (i / 4) + 4 h + i % 4) + ct of the lane's row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        c1[nt] = c1_s[32 * nt + col];
        off[nt] = -INFINITY;
        top[nt] = 0.f;
        lsum[nt] = 0.f;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[nt][ct][i] = 0.f;
    }

    // where channels 2 l, 2 l + 1 of the K scales and mins go in operand order
    int kpos[2];
    float kpow[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int c = 2 * l + x;
        int e = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) e = LY::chE[i] == (c & 7) ? i : e;
        int ke = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ke = i == e ? LY::kE[i] : ke;
        kpos[x] = (c >> 3) * 16 + e;
        kpow[x] = static_cast<float>(1 << (24 - kDown - ke));
    }
    const uint8_t *const qrow = smem + col * L::QP + 16 * h;
    // V: the lane's channels 4 col .. 4 col + 3 start at code bit 4 * BITS * col of a token row
    constexpr int ROWB = 16 * BITS;
    const int vdw = (4 * BITS * col) >> 5;
    const uint32_t vsh = static_cast<uint32_t>(4 * BITS * col) & 31u;

    f16x2 vs[4], vm[4];
    for (int g = 2 * b0; g < 2 * b1; ++g) {   // half g & 1 of block g / 2
        const int tt = g & 1;
        const uint8_t *mt = meta + ((g >> 1) & 1) * S::META;
        const uint8_t *st = ws + tt * S::STAGE;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // half g is in
        if (g + 1 < 2 * b1) stage(g + 1);
        if (tt == 0) {
            const uint32_t km = *reinterpret_cast<const uint32_t *>(mt + S::KMIN + 4 * l);
            const uint32_t ksc = *reinterpret_cast<const uint32_t *>(mt + S::KSCALE + 4 * l);
            uint16_t *ko = reinterpret_cast<uint16_t *>(kop);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                ko[kpos[x]] = f32_to_f16_bits(h16(ksc, x) * kpow[x]);
                ko[kpos[x] + 8] = f32_to_f16_bits(h16(km, x) * (1.f / (1 << kDown)));
            }
            const uint2 sm = *reinterpret_cast<const uint2 *>(mt + S::VSCALE + 8 * col);
            const uint2 mm = *reinterpret_cast<const uint2 *>(mt + S::VMIN + 8 * col);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t sel = (c & 1) ? 0x03020302u : 0x01000100u;
                const uint32_t sw = c < 2 ? sm.x : sm.y, mw = c < 2 ? mm.x : mm.y;
                const _Float16 up = static_cast<_Float16>(static_cast<float>(1 << (24 - kDown - V4<BITS>::k[c])) / 4.f);
                const _Float16 four = static_cast<_Float16>(4.f), down = static_cast<_Float16>(1.f / (1 << kDown));
                vs[c] = as_h2(perm(sw, sw, sel)) * f16x2{up, up} * f16x2{four, four};   // (up * 4 is past fp16's range)
                vm[c] = as_h2(perm(mw, mw, sel)) * f16x2{down, down};
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the operand-order K scales, this wave's own)
        }
        // ---- S^T = K Q^T: token 32 tt + col, channels 64 h + 8 ks ..
        f32x16 s[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[nt][i] = 0.f;
        // The operands of step ks + 1 are read while step ks is computed (left to
        // the compiler, every step waits for its own reads).
        const uint8_t *kc = st + col * ROWB + h * (ROWB / 2);
        uint32_t code[2 * BITS];
#pragma unroll
        for (int w = 0; w < 2 * BITS; ++w) code[w] = *reinterpret_cast<const uint32_t *>(kc + 4 * w);
        u32x4 sc[2], mn[2], qb[2][NT];
        auto fetch = [&](int ks) __attribute__((always_inline)) {
            sc[ks & 1] = *reinterpret_cast<const u32x4 *>(kop + 8 * (8 * h + ks));
            mn[ks & 1] = *reinterpret_cast<const u32x4 *>(kop + 8 * (8 * h + ks) + 4);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                qb[ks & 1][nt] = *reinterpret_cast<const u32x4 *>(qrow + 32 * L::QP * nt + 32 * ks);
        };
        fetch(0);
#pragma unroll
        for (int kq = 0; kq < 2; ++kq) {
            uint32_t c4[BITS];
#pragma unroll
            for (int w = 0; w < BITS; ++w) c4[w] = code[BITS * kq + w];
            u32x4 B[4];
            kunpack(c4, B);
#pragma unroll
            for (int k4 = 0; k4 < 4; ++k4) {
                const int ks = 4 * kq + k4;
                if (ks < 7) fetch(ks + 1);
                __builtin_amdgcn_sched_barrier(0);
                u32x4 a;
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = dequant(B[k4][i], as_h2(sc[ks & 1][i]), as_h2(mn[ks & 1][i]));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt] = mfma<NSN_DTYPE_F16>(a, qb[ks & 1][nt], s[nt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // ---- softmax: register i holds token 32 tt + 8 (i / 4) + 4 h + i % 4
        float fk[16], fv[16];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 a = *reinterpret_cast<const float4 *>(mt + S::KF + 4 * (32 * tt + 8 * c + 4 * h));
            const float4 b = *reinterpret_cast<const float4 *>(mt + S::VF + 4 * (32 * tt + 8 * c + 4 * h));
            fk[4 * c] = a.x; fk[4 * c + 1] = a.y; fk[4 * c + 2] = a.z; fk[4 * c + 3] = a.w;
            fv[4 * c] = b.x; fv[4 * c + 1] = b.y; fv[4 * c + 2] = b.z; fv[4 * c + 3] = b.w;
        }
        float mx[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[nt][i] *= fk[i];
            const float a0 = max3f(s[nt][0], s[nt][1], s[nt][2]), a1 = max3f(s[nt][3], s[nt][4], s[nt][5]);
            const float a2 = max3f(s[nt][6], s[nt][7], s[nt][8]), a3 = max3f(s[nt][9], s[nt][10], s[nt][11]);
            const float a4 = max3f(s[nt][12], s[nt][13], s[nt][14]);
            mx[nt] = max3f(max3f(a0, a1, a2), max2f(a3, a4), s[nt][15]) * c1[nt];   // (of the lane's half of the tokens)
        }
        // the V words of 16 tokens: lane's tokens 16 c + 4 h .. + 3 and 16 c + 8
        // + 4 h .. + 3 of the half, two dwords each; the first 16 behind the
        // last exponentials, the others behind the first products
        uint32_t vw[8][2];
        auto fetch_v = [&](int c) __attribute__((always_inline)) {
            const uint8_t *vc = st + S::HALF + (16 * c + 4 * h) * ROWB + 4 * vdw;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t *w = reinterpret_cast<const uint32_t *>(vc + (8 * (k >> 2) + (k & 3)) * ROWB);
                vw[k][0] = w[0];
                vw[k][1] = w[1];
            }
        };
        u32x4 pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt == NT - 1) {   // (where the other rows' scores have left their registers)
                __builtin_amdgcn_sched_barrier(0);
                fetch_v(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            auto rescale = [&](float to) __attribute__((always_inline)) {   // to: -inf only where off is
                const float r = off[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(off[nt] - to);
                off[nt] = to;
                lsum[nt] *= r;
                if (g > 2 * b0) {   // (no sums in the first half)
#pragma unroll
                    for (int ct = 0; ct < 4; ++ct) acc[nt][ct] *= r;
                }
                return r;
            };
            if (__builtin_amdgcn_ballot_w64(mx[nt] > off[nt] + kScoreMax)) {
                const float both = halves_max(mx[nt]);
                rescale(both > off[nt] + kScoreMax ? both - kScoreTo : off[nt]);
            }
            const float o = off[nt] == -INFINITY ? 0.f : off[nt];
            float ls[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][i], c1[nt], -o));
                ls[i & 1] += w;
                s[nt][i] = w * fv[i];
            }
            lsum[nt] += ls[0] + ls[1];
            float x;   // (of the lane's half of the tokens)
            {
                auto mag = [&](int i) { return __builtin_fabsf(s[nt][i]); };   // (a modifier of the maximum)
                const float a0 = max3f(mag(0), mag(1), mag(2)), a1 = max3f(mag(3), mag(4), mag(5));
                const float a2 = max3f(mag(6), mag(7), mag(8)), a3 = max3f(mag(9), mag(10), mag(11));
                const float a4 = max3f(mag(12), mag(13), mag(14));
                x = max3f(max3f(a0, a1, a2), max2f(a3, a4), mag(15));
            }
            if (__builtin_amdgcn_ballot_w64(x > top[nt])) {
                x = halves_max(x);
                const bool over = x > top[nt];
                int e = static_cast<int>(__float_as_uint(x) >> 23) - 127;   // x in [2^e, 2^(e + 1))
                e = e < kLeast ? kLeast : e;
                const float r = rescale(over ? off[nt] + static_cast<float>(e - kTopTo) : off[nt]);
                top[nt] = over ? kTop : top[nt];
#pragma unroll
                for (int i = 0; i < 16; ++i) s[nt][i] *= r;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) pb[nt][c][e] = pk<NSN_DTYPE_F16>(s[nt][8 * c + 2 * e], s[nt][8 * c + 2 * e + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
        // ---- O^T += V^T P^T, two steps of 16 tokens
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = __builtin_amdgcn_alignbit(vw[k][1], vw[k][0], vsh);
            if (c == 0) fetch_v(1);
            __builtin_amdgcn_sched_barrier(0);
            u32x4 a[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t D[4];
                V4<BITS>::pair(f[2 * k], f[2 * k + 1], D);
#pragma unroll
                for (int ct = 0; ct < 4; ++ct) a[ct][k] = dequant(D[ct], vs[ct], vm[ct]);
            }
#pragma unroll
            for (int ct = 0; ct < 4; ++ct)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[nt][ct] = mfma<NSN_DTYPE_F16>(a[ct], pb[nt][c], acc[nt][ct]);
        }
    }

    // ---- join the waves' states: every wave scales its own to the rows' maxima,
    // waves 4-7 hand theirs to 0-3, and the four sums are added row by row
    __syncthreads();   // (Q and the stages are free; no DMA is in flight)
    float2 *ml = reinterpret_cast<float2 *>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float lt = halves_sum(lsum[nt]);
        if (h == 0) ml[wave * L::ROWS + 32 * nt + col] = float2{off[nt], lt};
    }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w * L::ROWS + 32 * nt + col].x);
        const float a = (off[nt] == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(off[nt] - M) * (1 << kDown);
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) acc[nt][ct] *= a;
    }
    float *const area = reinterpret_cast<float *>(smem + L::ML + (wave & 3) * L::AREA);
    auto at = [&](int nt, int i) {
        return reinterpret_cast<float4 *>(area + (32 * nt + col) * kPartStride + 4 * (8 * (i >> 2) + 4 * h + (i & 3)));
    };
    auto put = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                *at(nt, i) = float4{acc[nt][0][i], acc[nt][1][i], acc[nt][2][i], acc[nt][3][i]};
    };
    if (wave >= 4) put();
    __syncthreads();
    if (wave < 4) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float4 x = *at(nt, i);
                acc[nt][0][i] += x.x;
                acc[nt][1][i] += x.y;
                acc[nt][2][i] += x.z;
                acc[nt][3][i] += x.w;
            }
        put();   // (a lane rewrites what it has read itself)
    }
    __syncthreads();
    // row 2 k + h of a wave's L::ROWS / 8: 32 lanes x 16 bytes
#pragma unroll
    for (int k = 0; k < L::ROWS / kWaves / 2; ++k) {
        const int row = wave * (L::ROWS / kWaves) + 2 * k + h;
        if (r0 + row >= rows) continue;
        float4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4 *>(smem + L::ML + w * L::AREA + row * kPartStride * 4 + 16 * col);
            o.x += x.x;
            o.y += x.y;
            o.z += x.z;
            o.w += x.w;
        }
        float *dst = p.part + (head_row(r0 + row) * p.splits + split) * kPartStride;
        *reinterpret_cast<float4 *>(dst + 4 + 4 * col) = o;
        if (col == 0) {
            float M = -INFINITY, Z = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w * L::ROWS + row].x);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float2 v = ml[w * L::ROWS + row];
                Z += v.y * ((v.x == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(v.x - M));   // (0 * NaN stays NaN)
            }
            *reinterpret_cast<float4 *>(dst) = float4{M * kLn2, Z, 0.f, 0.f};
        }
    }
}

// Join of a (sequence, q-head)'s partials: the prefix's, then its own (their
// count behind them, as the decode kernel leaves it).  8 groups of 32 lanes
// take every eighth partial, a lane 4 channels.
struct MergeParams {
    const float *pre, *own;
    const int32_t *counts;
    Side k, v;
    int64_t heads_q;
    int fan, splits, n_splits;
    void *out;
    int32_t *status;
};
constexpr int kGroups = 8;
// Channels 4 lane .. + 3 of a (sequence, q-head): U / Z, zero where nothing was attended.
template <int ODT>
__device__ __forceinline__ void finish(const float4 &U, float Z, int total, int64_t bh, int lane, const MergeParams &p) {
    if (total == 0) {
        Z = 1.f;
        if (lane == 0) raise_status(p.status, NSN_ST_EMPTY);
    }
    const float o[4] = {U.x / Z, U.y / Z, U.z / Z, U.w / Z};
    uint16_t *dst = static_cast<uint16_t *>(p.out) + bh * kDim + 4 * lane;
    *reinterpret_cast<u32x2 *>(dst) = u32x2{pack16<ODT>(o[0], o[1]), pack16<ODT>(o[2], o[3])};
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 4; ++c) bad |= !finite(Elem<ODT>::load(Elem<ODT>::store(o[c])));
    if (bad) raise_status(p.status, NSN_ST_NONFINITE_OUTPUT);
}
// A softmax state over partials: maximum, weight sum, 4 channels of weighted values.
constexpr int kJoin = 8;   // partials in flight
struct Softmax {
    float m = -INFINITY, z = 0.f;
    float4 u{0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void raise(float to) {
        const float a = (m == -INFINITY) ? 0.f : expf(m - to);   // (0 * NaN stays NaN)
        z *= a;
        u.x *= a;
        u.y *= a;
        u.z *= a;
        u.w *= a;
        m = to;
    }
    __device__ __forceinline__ void weigh(float ms, float zs, const float4 &us) {   // ms <= m
        const float a = (ms == -INFINITY) ? 0.f : expf(ms - m);
        z = __builtin_fmaf(zs, a, z);
        u.x = __builtin_fmaf(us.x, a, u.x);
        u.y = __builtin_fmaf(us.y, a, u.y);
        u.z = __builtin_fmaf(us.z, a, u.z);
        u.w = __builtin_fmaf(us.w, a, u.w);
    }
    __device__ __forceinline__ void add(float ms, float zs, const float4 &us) {
        raise(fmaxf(m, ms));
        weigh(ms, zs, us);
    }
    // partials first, first + step, .. < n of the row at src
    __device__ __forceinline__ void join(const float *src, int first, int step, int n, int lane) {
        for (int s0 = first; s0 < n; s0 += step * kJoin) {
            float2 v[kJoin];
            float4 w[kJoin];
            float to = m;
#pragma unroll
            for (int i = 0; i < kJoin; ++i) {
                v[i] = float2{-INFINITY, 0.f};
                w[i] = float4{0.f, 0.f, 0.f, 0.f};
                if (s0 + step * i < n) {
                    const float *ps = src + static_cast<int64_t>(s0 + step * i) * kPartStride;
                    v[i] = *reinterpret_cast<const float2 *>(ps);
                    w[i] = *reinterpret_cast<const float4 *>(ps + 4 + 4 * lane);
                }
            }
#pragma unroll
            for (int i = 0; i < kJoin; ++i) to = fmaxf(to, v[i].x);
            raise(to);
#pragma unroll
            for (int i = 0; i < kJoin; ++i) weigh(v[i].x, v[i].y, w[i]);
        }
    }
};

template <int ODT>
__global__ __launch_bounds__(256) void prefix_merge_kernel(MergeParams p) {
    __shared__ float red_m[kGroups], red_z[kGroups];
    __shared__ float4 red_u[kGroups][32];
    const int64_t bh = blockIdx.x;
    const int grp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bool bad_counts;
    const int np = splits_of(prefix_blocks(p.k, p.v, bh / p.heads_q / p.fan, bad_counts), p.splits);
    int no = p.counts[bh];
    no = no < 0 ? 0 : (no > p.n_splits ? p.n_splits : no);   // (in bounds whatever the count)
    Softmax x;
    x.join(p.pre + bh * p.splits * kPartStride, grp, kGroups, np, lane);
    x.join(p.own + bh * p.n_splits * kPartStride, grp, kGroups, no, lane);
    if (lane == 0) {
        red_m[grp] = x.m;
        red_z[grp] = x.z;
    }
    red_u[grp][lane] = x.u;
    __syncthreads();
    if (grp != 0) return;
    for (int g = 1; g < kGroups; ++g) x.add(red_m[g], red_z[g], red_u[g][lane]);
    finish<ODT>(x.u, x.z, np + no, bh, lane, p);
}

// Own tokens and join in one kernel, for short own contexts: a workgroup per
// (sequence, kv-head), whose waves 0 .. kOwnWaves - 1 take a range of the own
// tokens each (the decode kernel's segment, partials to the workspace) while
// waves kOwnWaves .. 7 join the prefix's partials of its q-heads; then both are
// joined.  Against the decode kernel and the merge above it saves a launch and
// the decode kernel's search for its work, and loses where a wave walks many
// blocks (see own_blocks).
constexpr int kOwnWaves = 4;
// The most 64-token blocks of an own context that pay so: with few workgroups
// the decode kernel's waves finish a long one sooner, with many they are full
// anyway.  Measured behind 2048 tokens, apart -> fused: 2 x 8 kv-heads x 600
// own tokens 23.1 -> 21.5 us, x 1000 23.2 -> 26.2; 4 x 16 x 600 23.3 -> 22.8, x
// 1000 23.7 -> 27.4; 16 x 8 x 40 26.8 -> 22.9, x 1000 30.7 -> 31.0, x 2000 32.9
// -> 34.9; 48 x 4 x 1000 39.9 -> 34.9, x 2000 46.8 -> 39.5; 64 x 4 (5 bits) x
// 1000 39.2 -> 35.9, x 3000 52.8 -> 50.2.
inline int64_t own_blocks(int64_t streams) { return streams / 6 > 10 ? streams / 6 : 10; }
template <int BITS, int QDT, int GRP, bool TBF, int ODT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void own_merge_kernel(
    fast::FastParams p, MergeParams g) {
    using S = fast::LdsShape<BITS, GRP>;
    __shared__ u32x4 s_afrag[kOwnWaves][S::ROWS * 16 + 1];
    __shared__ uint32_t s_pbuf[kOwnWaves][S::ROWS * 36 + 4];
    __shared__ uint32_t s_k0[kOwnWaves][S::NBW], s_k1[kOwnWaves][S::NBW], s_v0[kOwnWaves][S::NBW], s_v1[kOwnWaves][S::NBW];
    __shared__ uint32_t s_m0[kOwnWaves][S::MW], s_m1[kOwnWaves][S::MW];
    __shared__ float red_m[kGroups], red_z[kGroups];
    __shared__ float4 red_u[kGroups][32];
    const int tid = threadIdx.x, l = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 31, G = p.group, per = kGroups / G;   // groups of 32 lanes that share a q-head's partials
    const uint32_t hkv = static_cast<uint32_t>(p.heads_kv);
    const int b = static_cast<int>(blockIdx.x / hkv), kvh = static_cast<int>(blockIdx.x % hkv);
    // the sequence's own tokens: none where its counts do not fit the cache
    const OwnRanges own(p.seq_len[b], p.k.blocks ? p.k.blocks[b] : 0, p.v.blocks ? p.v.blocks[b] : 0,
                        {p.k.block_cap, p.k.tail ? p.k.tail_cap : 0},
                        {p.v.block_cap, p.v.tail ? p.v.tail_cap : 0});
    if (own.over && tid == 0 && kvh == 0) raise_status(p.status, NSN_ST_CAPACITY);
    auto cut = [&](int k) { return own.cut(k, kOwnWaves); };
    int count = 0, slot = 0;   // (non-empty ranges, those before this wave's)
#pragma unroll
    for (int k = 0; k < kOwnWaves; ++k) {
        const int used = cut(k) < cut(k + 1);
        slot += k < wave ? used : 0;
        count += used;
    }
    const int64_t bh0 = static_cast<int64_t>(b) * p.heads_q + static_cast<int64_t>(kvh) * G;
    bool bad_counts;
    const int np = splits_of(prefix_blocks(g.k, g.v, b / g.fan, bad_counts), g.splits);
    if (wave < kOwnWaves) {
        for (int i = l; i < S::ROWS * 16 + 1; i += 64) s_afrag[wave][i] = u32x4{0u, 0u, 0u, 0u};
        for (int i = l; i < S::ROWS * 36 + 4; i += 64) s_pbuf[wave][i] = 0u;
        fast::lds_sync();
        if (cut(wave) < cut(wave + 1)) {
            const fast::Lds<BITS, GRP> sh{s_afrag[wave], s_pbuf[wave], s_k0[wave], s_k1[wave],
                                          s_v0[wave],    s_v1[wave],   s_m0[wave], s_m1[wave]};
            fast::segment<BITS, QDT, false, GRP, TBF>(p, sh, b, kvh, cut(wave), cut(wave + 1), own.nk, own.nv, slot, count,
                                                       l);
        }
    } else {   // 2 * (kWaves - kOwnWaves) == kGroups groups of 32 lanes
        const int grp = (tid >> 5) - 2 * kOwnWaves, head = grp / per;
        Softmax x;
        if (head < G) x.join(g.pre + (bh0 + head) * g.splits * kPartStride, grp % per, per, np, lane);
        if (lane == 0) {
            red_m[grp] = x.m;
            red_z[grp] = x.z;
        }
        red_u[grp][lane] = x.u;
    }
    __syncthreads();   // (the partials of the workgroup's waves are in memory)
    const int head = tid >> 5;
    if (head >= G) return;
    Softmax x;
    x.join(g.own + (bh0 + head) * g.n_splits * kPartStride, 0, 1, count, lane);
    for (int k = head * per; k < (head + 1) * per; ++k) x.add(red_m[k], red_z[k], red_u[k][lane]);
    finish<ODT>(x.u, x.z, np + count, bh0 + head, lane, g);
}

constexpr int row_tile(int64_t rows) { return rows > 32 ? 64 : 32; }

}  // namespace prefix
}  // namespace nsn

using namespace nsn;

// Splits of a prefix's blocks: one round of workgroups, one per CU.
extern "C" int nsn_shared_prefix_splits(int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t prefixes,
                                        int64_t max_prefix_blocks) {
    using namespace nsn::prefix;
    if (batch <= 0 || heads_kv <= 0 || heads_q <= 0 || heads_q % heads_kv || prefixes <= 0 || batch % prefixes) return 1;
    const int64_t rows = batch / prefixes * (heads_q / heads_kv);
    const int64_t units = prefixes * heads_kv * ((rows + row_tile(rows) - 1) / row_tile(rows));
    int64_t s = 256 / units;
    const int64_t most = (max_prefix_blocks + kMinBlocks - 1) / kMinBlocks;
    s = s < most ? s : most;
    return static_cast<int>(s < 1 ? 1 : s);
}

extern "C" int64_t nsn_shared_prefix_workspace_floats(int64_t batch, int64_t heads_q, int prefix_splits, int n_splits) {
    if (batch <= 0 || heads_q <= 0 || prefix_splits <= 0 || n_splits <= 0) return 0;
    const int64_t own = nsn_attention_workspace_floats(batch, heads_q, n_splits);
    return (own + 3) / 4 * 4 + batch * heads_q * prefix_splits * nsn::prefix::kPartStride;
}

extern "C" int nsn_shared_prefix_attention(const nsn_shared_args *a, nsn_stream_t stream) {
    using namespace nsn::prefix;
    if (!a || !a->q || !a->seq_len || !a->workspace || !a->out || !a->status) return NSN_EINVAL;
    if (a->batch <= 0 || a->heads_kv <= 0 || a->heads_q <= 0 || a->heads_q % a->heads_kv || a->prefixes <= 0 ||
        a->batch % a->prefixes || a->max_seq_len <= 0 || a->prefix_splits < 1 || a->n_splits < 2)
        return NSN_EINVAL;
    if (a->bits != 3 && a->bits != 5) return NSN_EINVAL;
    if (!(a->scale > 0.f) || !__builtin_isfinite(a->scale)) return NSN_EINVAL;
    if (a->q_dtype != NSN_DTYPE_F16 && a->q_dtype != NSN_DTYPE_BF16) return NSN_EINVAL;
    if (a->out_dtype != NSN_DTYPE_F16 && a->out_dtype != NSN_DTYPE_BF16) return NSN_EINVAL;
    for (const void *ptr : {a->q, static_cast<const void *>(a->out), static_cast<const void *>(a->workspace)})
        if (reinterpret_cast<uintptr_t>(ptr) & 15u) return NSN_EINVAL;
    // the output in the queries' place, or apart from them (the joint kernel's
    // workgroups write while others read)
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(a->q), o0 = reinterpret_cast<uintptr_t>(a->out);
    if (a->heads_q > (1 << 23) / a->batch) return NSN_EINVAL;
    const uintptr_t bytes = static_cast<uintptr_t>(a->batch * a->heads_q) * kDim * 2;
    if (q0 != o0 && q0 < o0 + bytes && o0 < q0 + bytes) return NSN_EINVAL;
    for (const nsn_kv_side *s : {&a->prefix_k, &a->prefix_v}) {
        if (!s->blocks || s->block_cap <= 0 || s->block_cap > (1 << 25)) return NSN_EINVAL;
        for (const void *ptr : {static_cast<const void *>(s->codes), static_cast<const void *>(s->mins),
                                static_cast<const void *>(s->scales), static_cast<const void *>(s->factors)})
            if (!ptr || (reinterpret_cast<uintptr_t>(ptr) & 15u)) return NSN_EINVAL;
    }
    const int64_t group = a->heads_q / a->heads_kv, fan = a->batch / a->prefixes;
    const int64_t rows = fan * group;
    if (rows > (1 << 24)) return NSN_EINVAL;
    const int tile = row_tile(rows);
    const int64_t row_tiles = (rows + tile - 1) / tile;
    const int64_t wgs = a->prefixes * a->heads_kv * row_tiles;
    if (a->prefix_splits > (1 << 22) || wgs > (1 << 22) / a->prefix_splits) return NSN_EINVAL;
    // the own tokens' checks refuse before anything is launched
    nsn_attn_args o{};
    o.q = a->q;
    o.q_dtype = a->q_dtype;
    o.batch = a->batch;
    o.heads_q = a->heads_q;
    o.heads_kv = a->heads_kv;
    o.scale = a->scale;
    o.seq_len = a->seq_len;
    o.max_seq_len = a->max_seq_len;
    o.bits = a->bits;
    o.k_mode = NSN_KV_PACKED;
    o.k = a->k;
    o.v = a->v;
    o.kernel = NSN_ATTN_FAST;
    o.n_splits = a->n_splits;
    o.partials = a->workspace;
    o.status = a->status;
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    fast::FastParams f{};
    bool tbf;
    int rc = fast::fast_params(&o, f, tbf);
    if (rc != NSN_OK) return rc;
    const bool fused = f.nb_max <= own_blocks(a->batch * a->heads_kv) && a->n_splits >= kOwnWaves;
    if (!fused) {
        rc = launch_attn_fast(&o, st);
        if (rc != NSN_OK) return rc;
    }
    const int64_t own = nsn_attention_workspace_floats(a->batch, a->heads_q, a->n_splits);
    PrefixParams p{};
    p.q = static_cast<const uint16_t *>(a->q);
    p.q_bf16 = a->q_dtype == NSN_DTYPE_BF16;
    p.heads_q = a->heads_q;
    p.heads_kv = a->heads_kv;
    p.group = static_cast<int>(group);
    p.fan = static_cast<int>(fan);
    p.row_tiles = static_cast<int>(row_tiles);
    p.splits = a->prefix_splits;
    p.scale = a->scale;
    auto side = [](const nsn_kv_side &s) { return Side{s.codes, s.mins, s.scales, s.factors, s.blocks, s.block_cap}; };
    p.k = side(a->prefix_k);
    p.v = side(a->prefix_v);
    p.part = a->workspace + (own + 3) / 4 * 4;
    p.status = a->status;
    const dim3 grid(static_cast<unsigned>(wgs * a->prefix_splits));
#define NSN_PREFIX_LAUNCH(B_, N_) hipLaunchKernelGGL((prefix_kernel<B_, N_>), grid, dim3(64 * kWaves), 0, st, p)
    if (a->bits == 3) {
        if (tile == 64) NSN_PREFIX_LAUNCH(3, 2);
        else NSN_PREFIX_LAUNCH(3, 1);
    } else {
        if (tile == 64) NSN_PREFIX_LAUNCH(5, 2);
        else NSN_PREFIX_LAUNCH(5, 1);
    }
#undef NSN_PREFIX_LAUNCH
    if (hipGetLastError() != hipSuccess) return NSN_ELAUNCH;
    MergeParams m{};
    m.pre = p.part;
    m.own = a->workspace;
    m.counts = reinterpret_cast<const int32_t *>(a->workspace + a->batch * a->heads_q * a->n_splits * kPartStride);
    m.k = p.k;
    m.v = p.v;
    m.heads_q = a->heads_q;
    m.fan = p.fan;
    m.splits = p.splits;
    m.n_splits = a->n_splits;
    m.out = a->out;
    m.status = a->status;
    if (fused) {
        const dim3 ogrid(static_cast<unsigned>(a->batch * a->heads_kv));
        const bool bf = a->q_dtype == NSN_DTYPE_BF16, obf = a->out_dtype == NSN_DTYPE_BF16;
#define NSN_OWN_LAUNCH3(B_, Q_, G_, T_, O_) \
    hipLaunchKernelGGL((own_merge_kernel<B_, Q_, G_, T_, O_>), ogrid, dim3(64 * kWaves), 0, st, f, m)
#define NSN_OWN_LAUNCH2(B_, Q_, G_, T_)                               \
    do {                                                              \
        if (obf) NSN_OWN_LAUNCH3(B_, Q_, G_, T_, NSN_DTYPE_BF16);     \
        else NSN_OWN_LAUNCH3(B_, Q_, G_, T_, NSN_DTYPE_F16);          \
    } while (0)
#define NSN_OWN_LAUNCH1(B_, Q_, G_)                                   \
    do {                                                              \
        if (tbf) NSN_OWN_LAUNCH2(B_, Q_, G_, true);                   \
        else NSN_OWN_LAUNCH2(B_, Q_, G_, false);                      \
    } while (0)
#define NSN_OWN_LAUNCH(B_, Q_)                                        \
    do {                                                              \
        if (group <= 4) NSN_OWN_LAUNCH1(B_, Q_, 4);                   \
        else NSN_OWN_LAUNCH1(B_, Q_, 8);                              \
    } while (0)
        if (a->bits == 3) {
            if (bf) NSN_OWN_LAUNCH(3, NSN_DTYPE_BF16);
            else NSN_OWN_LAUNCH(3, NSN_DTYPE_F16);
        } else {
            if (bf) NSN_OWN_LAUNCH(5, NSN_DTYPE_BF16);
            else NSN_OWN_LAUNCH(5, NSN_DTYPE_F16);
        }
#undef NSN_OWN_LAUNCH
#undef NSN_OWN_LAUNCH1
#undef NSN_OWN_LAUNCH2
#undef NSN_OWN_LAUNCH3
        return hipGetLastError() == hipSuccess ? NSN_OK : NSN_ELAUNCH;
    }
    const dim3 mgrid(static_cast<unsigned>(a->batch * a->heads_q));
    if (a->out_dtype == NSN_DTYPE_BF16) hipLaunchKernelGGL(prefix_merge_kernel<NSN_DTYPE_BF16>, mgrid, dim3(256), 0, st, m);
    else hipLaunchKernelGGL(prefix_merge_kernel<NSN_DTYPE_F16>, mgrid, dim3(256), 0, st, m);
    return hipGetLastError() == hipSuccess ? NSN_OK : NSN_ELAUNCH;
}
