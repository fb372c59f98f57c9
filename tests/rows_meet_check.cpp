/*
 * rows_meet (nsn_amd/csrc/nsn_rows.hpp) against every byte of every row: rows of
 * 16 bytes at token and head strides that overlap, repeat, interleave or leave
 * gaps, and spans that start and end anywhere around them.
 *
 *   usage: rows_meet_check
 * Prints the number of cases and mismatches; exit status 1 on a mismatch.
 */
#include <cstdio>
#include <initializer_list>

#include "../nsn_amd/csrc/nsn_rows.hpp"

int main() {
    constexpr int64_t kBytes = 16;
    constexpr uintptr_t x = 1000;
    long cases = 0, bad = 0;
    for (int64_t tokens : {1, 2, 5})
        for (int64_t heads : {1, 2, 3})
            for (int64_t ts : {0, 8, 16, 48, 64, 200})
                for (int64_t hs : {0, 8, 16, 24, 100})
                    for (uintptr_t lo = x - 40; lo < x + 1100; lo += 4)
                        for (uintptr_t size : {1, 16, 20, 128, 700}) {
                            bool want = false;
                            for (int64_t t = 0; t < tokens; ++t)
                                for (int64_t h = 0; h < heads; ++h) {
                                    const uintptr_t row = x + t * ts + h * hs;
                                    want = want || (row < lo + size && row + kBytes > lo);
                                }
                            ++cases;
                            bad += want != nsn::rows_meet(x, tokens, heads, ts, hs, kBytes, lo, lo + size);
                        }
    std::printf("%ld cases, %ld mismatches\n", cases, bad);
    return bad != 0;
}
