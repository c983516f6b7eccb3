// max(p - q, 0) of verify_share.h against quotients of whole numbers: within 7 * 2^-53 of the larger of p and q (1 + 2^-50 of that, for the products of roundings) and 2^-60, 0 where the weights and sums are the
// same.  Prints the largest error in multiples of the bound and of 2^-60, or the first that is outside (exit status 1).
#include <cmath>
#include <cstdio>
#include <random>

#include "../../spy_amd/csrc/verify_share.h"

int main() {
    std::mt19937_64 rng(5);
    const auto below = [&](int bits) { return rng() >> (64 - bits); };
    long double worst = 0, steps = 0;
    for (int i = 0; i < 4000000; i++) {
        // a weight of up to 2^44 (the largest token's) in a sum of that and up to 2^62
        const int rest = 1 + (int)(rng() % 62);
        uint64_t w = below(1 + (int)(rng() % 44)) + 1, v = i % 3 == 0 ? w + below(20) : below(1 + (int)(rng() % 44)) + 1;
        v = v < (1ull << 44) ? v : 1ull << 44;
        const uint64_t all = (1ull << 44) + below(rest), other = i % 3 == 0 ? all + below(30) : (1ull << 44) + below(1 + (int)(rng() % 62));
        const uint64_t got = verify_more(w, 1.0 / (double)all, v, 1.0 / (double)other);
        if (verify_more(w, 1.0 / (double)all, w, 1.0 / (double)all) != 0) { std::printf("p - p is not 0\n"); return 1; }
        const __int128 n = (__int128)w * other - (__int128)v * all;
        const long double want = n > 0 ? (long double)n / (long double)all / (long double)other : 0, p = (long double)w / all, q = (long double)v / other;
        const long double off = fabsl(std::ldexp((long double)got, -60) - want), bound = 7 * 0x1p-53L * (1 + 0x1p-50L) * fmaxl(p, q) + 0x1p-60L;
        worst = fmaxl(worst, off / bound);
        steps = fmaxl(steps, off * 0x1p60L);
        if (off > bound) { std::printf("%llu / %llu - %llu / %llu: off by %Lg, bound %Lg\n", (unsigned long long)w, (unsigned long long)all, (unsigned long long)v, (unsigned long long)other, off, bound); return 1; }
    }
    std::printf("%.2Lf %.1Lf\n", worst, steps);
}
