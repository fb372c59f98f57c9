// A sequence's own tokens as the waves of one workgroup share them, behind a
// shared prefix (nsn_prefix.hip).  Integer arithmetic only: it runs on the host
// as well, where its ranges are checked for every kind of count.
#pragma once

#include <stdint.h>

namespace nsn {
namespace prefix {

constexpr int kOwnBlock = 64;   // tokens of a packed block

struct OwnCapacity {
    int64_t blocks, tail;       // of one side; tail 0: it has none
};

// Tokens 0 .. T - 1 in ranges of equal cost: a packed token 1, a dense one 3
// (read without the prefetch); packed cuts at blocks, dense ones at 16 tokens.
struct OwnRanges {
    int32_t T, nk, nv;          // usable tokens and packed blocks: all 0 where the counts do not fit
    bool over;                  // they did not
    int32_t packed, dense;
    int64_t cost;

    __host__ __device__ OwnRanges(int32_t tokens, int32_t blocks_k, int32_t blocks_v,
                                                  const OwnCapacity &k, const OwnCapacity &v)
        : T(tokens), nk(blocks_k), nv(blocks_v), over(!fits(tokens, blocks_k, k) || !fits(tokens, blocks_v, v)) {
        if (over) T = nk = nv = 0;
        T = T > 0 ? T : 0;
        const int32_t both = nk < nv ? nk : nv;
        packed = both > T / kOwnBlock ? T : both * kOwnBlock;
        cost = packed + 3 * static_cast<int64_t>(T - packed);
        dense = nk == nv ? 16 : kOwnBlock;   // (one side packed: still in blocks)
    }
    static __host__ __device__ bool fits(int32_t tokens, int32_t blocks, const OwnCapacity &c) {
        if (blocks < 0 || blocks > c.blocks) return false;
        const int64_t rest = static_cast<int64_t>(tokens) - static_cast<int64_t>(blocks) * kOwnBlock;
        return rest <= c.tail || rest <= 0;
    }
    // first token of range i of n (i == n: the end)
    __host__ __device__ int32_t cut(int i, int n) const {
        const int64_t c = cost * i / n;
        if (i == n) return T;
        if (c <= packed) return static_cast<int32_t>(c) / kOwnBlock * kOwnBlock;
        const int32_t d = (static_cast<int32_t>((c - packed) / 3) + dense - 1) / dense * dense;   // (< T, to 64 above)
        return d < T - packed ? packed + d : T;
    }
};

}  // namespace prefix
}  // namespace nsn
