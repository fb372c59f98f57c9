/*
 * The ranges of a sequence's own tokens behind a shared prefix, for every kind
 * of length and block count, usable or not: a count that the cache cannot hold
 * leaves no token, every range lies in [0, T], the ranges follow each other and
 * end at T, and a token of a packed block or of a tail row that does not exist
 * is in none of them.
 *
 *   usage: own_ranges_check
 * Prints the number of cases and of those with a fault; exit status 1 if any.
 */
#include <cstdio>

#define __host__
#define __device__
#include "../nsn_amd/csrc/nsn_own_ranges.hpp"

using nsn::prefix::OwnCapacity;
using nsn::prefix::OwnRanges;

int main() {
    const int32_t lengths[] = {INT32_MIN, -1000, -1, 0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 640, 641, 1500,
                               1 << 20, INT32_MAX};
    const int32_t counts[] = {INT32_MIN, -1000, -2, -1, 0, 1, 2, 3, 10, 23, 1 << 14, 1 << 25, INT32_MAX};
    const OwnCapacity caps[] = {{0, 0}, {0, 64}, {1, 0}, {4, 16}, {4, 640}, {23, 127}, {1 << 25, 1 << 20}};
    long cases = 0, bad = 0;
    for (int32_t t : lengths)
        for (int32_t nk : counts)
            for (int32_t nv : counts)
                for (const OwnCapacity &k : caps)
                    for (const OwnCapacity &v : caps) {
                        auto holds = [&](int64_t n, const OwnCapacity &c) {
                            return n >= 0 && n <= c.blocks && (t <= 64 * n || t - 64 * n <= c.tail);
                        };
                        const bool usable = holds(nk, k) && holds(nv, v);
                        const OwnRanges r(t, nk, nv, k, v);
                        bool ok = r.over == !usable && r.T == (usable && t > 0 ? t : 0);
                        ok = ok && r.nk == (usable ? nk : 0) && r.nv == (usable ? nv : 0);
                        const int n = 4;
                        ok = ok && r.cut(0, n) == 0 && r.cut(n, n) == r.T;
                        for (int i = 0; i < n; ++i) {
                            const int32_t a = r.cut(i, n), b = r.cut(i + 1, n);
                            ok = ok && a >= 0 && a <= b && b <= r.T;
                        }
                        ++cases;
                        bad += !ok;
                        if (!ok && bad <= 5)
                            std::printf("T %d, blocks %d %d, capacities %lld/%lld %lld/%lld: T %d, ranges %d %d %d %d %d\n", t,
                                        nk, nv, (long long)k.blocks, (long long)k.tail, (long long)v.blocks,
                                        (long long)v.tail, r.T, r.cut(0, n), r.cut(1, n), r.cut(2, n), r.cut(3, n),
                                        r.cut(4, n));
                    }
    std::printf("%ld cases, %ld faults\n", cases, bad);
    return bad != 0;
}
