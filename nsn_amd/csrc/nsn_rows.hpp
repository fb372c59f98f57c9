// Strided rows against a span of memory, for the host's argument checks.
#pragma once

#include <stdint.h>

namespace nsn {

// Whether one of the [tokens, heads] rows of `bytes` bytes at x (token and head
// strides in bytes, not negative) meets the bytes from lo to hi (hi > lo).
inline bool rows_meet(uintptr_t x, int64_t tokens, int64_t heads, int64_t token_stride, int64_t head_stride,
                      int64_t bytes, uintptr_t lo, uintptr_t hi) {
    if (x >= hi || x + (tokens - 1) * token_stride + (heads - 1) * head_stride + bytes <= lo) return false;   // (as a rule)
    for (int64_t h = 0; h < heads; ++h) {
        const uintptr_t head = x + h * head_stride;
        int64_t t = 0;   // the first token whose row ends behind lo
        if (head + bytes <= lo) {
            if (token_stride == 0) continue;
            t = static_cast<int64_t>(lo - bytes - head) / token_stride + 1;
        }
        if (t < tokens && head + t * token_stride < hi) return true;
    }
    return false;
}

}  // namespace nsn
