// The searches of csrc/search.cuh on the host.  Prints one line a check that fails, then the number of failures
// and the largest number of evaluations of a search.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <limits>
#include <random>

#include "search.cuh"

static int g_bad = 0;
static long g_most = 0;

static uint32_t key(float x) {
    if (!(x == x)) return 0x007FFFFFu;
    uint32_t u;
    std::memcpy(&u, &x, 4);
    if (x == 0.0f) u = 0;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
static float value(uint32_t k) {
    const uint32_t u = (k & 0x80000000u) ? (k ^ 0x80000000u) : ~k;
    float x;
    std::memcpy(&x, &u, 4);
    return x;
}

// The border of min-p among the keys of a row's logits: largest logit mx, temperature T.  `walk`: key by key from the
// formula's guess, given up after a million steps.
static void border(float mx, double T, double mp, bool walk) {
    long calls = 0;
    auto keeps = [&](uint32_t k) {
        ++calls;
        const float x = value(k);
        if (x == mx) return true;
        const double w = std::exp(((double)x - (double)mx) / T);
        return w >= mp;
    };
    const uint32_t lo = 0x00800000u, hi = key(mx), guess = key((float)((double)mx + T * std::log(mp)));
    uint32_t b;
    if (walk) {
        b = guess < lo ? lo : guess < hi ? guess : hi;
        while (b > lo && calls < 1000000 && keeps(b - 1)) --b;
        while (b < hi && calls < 1000000 && !keeps(b)) ++b;
    } else {
        b = qmm::lowest_kept(lo, hi, guess, keeps);
    }
    const long used = calls;
    if (used > g_most) g_most = used;
    if (used > 66 || !keeps(b) || (b > lo && keeps(b - 1))) {
        ++g_bad;
        std::printf("max %g T %g min-p %.17g: key %08x after %ld evaluations\n", mx, T, mp, b, used);
    }
}

static void borders(bool walk) {
    const float inf = std::numeric_limits<float>::infinity(), tiny = std::numeric_limits<float>::denorm_min();
    // around 0, where keys are dense
    border(0.0f, 1.0, 1.0, walk);
    border(-0.0f, 1.0, 1.0, walk);
    border(1e-20f, 1.0, 1.0, walk);
    border(tiny, 1.0, 1.0, walk);
    border(-tiny, 0.5, 1.0, walk);
    border(5.0f, 1.0, std::exp(-5.0), walk);
    border(4.0f, 0.5, std::exp(-8.0), walk);
    border(8.0f, 0.8, std::exp(-10.0), walk);
    for (float mx : {0.0f, 1.0f, -3.0f, 3e38f, -3e38f, inf, tiny, 1e-30f, 65504.0f})
        for (double T : {1e-30, 1e-6, 0.7, 1.0, 1e6, 1e16, 3e38, (double)inf})
            for (double mp : {1e-300, 1e-30, 0.02, 0.5, 0.999, 1.0 - 1e-16, 1.0}) border(mx, T, mp, walk);
    std::mt19937 rng(1);
    std::normal_distribution<float> n(0.0f, 10.0f);
    std::uniform_real_distribution<double> u(0.0, 1.0);
    for (int i = 0; i < 20000; ++i) {
        const float mx = n(rng);
        const double T = 0.05 + 2 * u(rng);
        border(mx, T, 1e-6 + u(rng) * (1.0 - 1e-6), walk);
    }
}

// How many equal weights w above a mass reach a target, of `inside` of them.  `walk`: one by one from the quotient.
static uint32_t count(double above, double w, double target, uint32_t inside, bool walk) {
    long calls = 0;
    auto reach = [&](uint32_t n) { return ++calls, above + n * w >= target; };
    const double guess = std::fmin(std::fmax(std::ceil((target - above) / w), 1.0), (double)inside);
    uint32_t n = (uint32_t)guess;
    if (walk) {
        while (n > 1 && reach(n - 1)) --n;
        while (n < inside && !reach(n)) ++n;
    } else {
        n = qmm::lowest_kept(1, inside, n, reach);
    }
    if (calls > g_most) g_most = calls;
    if (calls > 66 || n < 1 || n > inside || (n < inside && !reach(n)) || (n > 1 && reach(n - 1))) {
        ++g_bad;
        std::printf("above %.17g w %g target %.17g inside %u: %u after %ld\n", above, w, target, inside, n, calls);
    }
    return n;
}

static void counts(bool walk) {
    // weights below the last bit of the mass above them: any of a whole range of counts gives the same sum
    count(1.0, 1e-22, 1.0 + std::ldexp(1.0, -51), 100000000, walk);
    count(1.0, 1e-25, 1.0 + std::ldexp(1.0, -52), 1u << 30, walk);
    count(3.0, 1e-300, 3.5, 1u << 30, walk);
    count(3.0, 0.0, 3.0, 1000, walk);  // no quotient
    count(3.0, 0.0, 3.5, 1000, walk);
    count(0.0, 0.5, 1e300, 1000, walk);
    std::mt19937 rng(2);
    std::uniform_real_distribution<double> u(0.0, 1.0);
    for (int i = 0; i < 20000; ++i) {
        const uint32_t inside = 1 + rng() % 5000;
        const double w = std::exp(-30.0 * u(rng)), above = u(rng) * 10, target = above + w * inside * u(rng) * 1.01;
        const uint32_t got = count(above, w, target, inside, walk);
        uint32_t first = 1;
        while (i % 20 == 0 && first < inside && !(above + first * w >= target)) ++first;
        if (i % 20 == 0 && got != first) {
            ++g_bad;
            std::printf("count %u, not %u\n", got, first);
        }
    }
}

// Every border and every guess of a short range, at the ends of the keys too.
static void every_border() {
    for (uint32_t base : {0u, 1000u, 0xFFFFFFFFu - 40u})
        for (uint32_t span : {0u, 1u, 2u, 39u})
            for (uint32_t at = base; at <= base + span && at >= base; ++at)
                for (uint32_t guess : {0u, base, base + span / 2, base + span, at, 0xFFFFFFFFu}) {
                    const uint32_t got =
                        qmm::lowest_kept(base, base + span, guess, [&](uint32_t k) { return k >= at; });
                    if (got != at) {
                        ++g_bad;
                        std::printf("border %u of [%u, %u] from %u: %u\n", at, base, base + span, guess, got);
                    }
                    if (at == 0xFFFFFFFFu) break;
                }
    long calls = 0;  // the widest range from its far end
    const uint32_t got = qmm::lowest_kept(0u, 0xFFFFFFFFu, 0xFFFFFFFFu, [&](uint32_t k) { return ++calls, k >= 3; });
    if (got != 3 || calls > 66) {
        ++g_bad;
        std::printf("widest range: %u after %ld\n", got, calls);
    }
}

int main(int argc, char** argv) {
    const bool walk = argc > 1 && argv[1][0] == 'w';
    borders(walk);
    counts(walk);
    if (!walk) every_border();
    std::printf("%d %ld\n", g_bad, g_most);
    return 0;
}
