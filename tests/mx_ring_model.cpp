// A model of one block of the few-row mxfp4 kernel that makes its own planes:
// the TMA warp, the MMA warp, the tensor core behind it, the epilogue and the 16
// converter warps take steps in random order over the barriers' phases.  The
// tensor core reads a k-block's planes when it gets to it, at any time after the
// MMA warp has issued it, and frees the slot then.
//
// Prints one line per run that read wrong planes or came to a stop, and their
// number last.   usage: mx_ring_model <runs> <seed> <early>
// `early` k-blocks are taken to have begun that have not (a mistake to be seen).
#include <cstdio>
#include <cstdlib>
#include <deque>
#include <random>
#include <utility>
#include <vector>

#include "mx_ring.cuh"

namespace {

constexpr int STAGES = 10, ACCS = 2, WARPS = 16, FIRST = 3;

struct Barrier {
    int phase = 0;  // completed phases
    bool test(int parity) const { return (phase & 1) != parity; }
};

struct Run {
    std::mt19937 rng;
    int nk, n_tiles, tile0, tile1, L, fresh;
    Barrier empty[STAGES], full[STAGES], digits[STAGES], acc_full[ACCS], acc_empty[ACCS], started;
    std::pair<int, int> planes[STAGES];  // (item, k-block) a slot's planes are of
    int begun = 0, wrong = 0, early;

    // TMA warp and its copies
    int t_i = 0;
    std::deque<int> copies;
    // MMA warp and the tensor core behind it
    int m_tile, m_kb = 0, m_nt, m_served = 0, m_seg = 0, m_s = 0, m_ph = 0;
    bool m_in = false;
    int made[STAGES] = {};
    struct Issued {
        int slot, item, kb, acc;  // acc >= 0: end of a tile
    };
    std::deque<Issued> issued;
    // epilogue
    int e_seg = 0;
    // converter warps: the k-blocks each makes planes of
    struct Make {
        int i, item, kb;
    };
    std::deque<Make> make[WARPS];
    int seen[WARPS];

    int rnd(int n) { return (int)(rng() % (unsigned)n); }

    Run(unsigned seed, int early_) : rng(seed), early(early_) {
        nk = 1 + rnd(12);
        n_tiles = 1 + rnd(16);
        const int tiles = n_tiles * (1 + rnd(6));
        tile0 = rnd(tiles);
        tile1 = tile0 + 1 + rnd(tiles - tile0);
        L = qmm::f4_ring_slots(true, nk, STAGES);
        fresh = qmm::f4_ring_fresh(true, nk, STAGES);
        m_tile = tile0;
        m_nt = tile0 % n_tiles;
        for (auto& p : planes) p = {-1, -1};
        // one row to an item: `par` warps share the k-blocks of the run
        const int par = WARPS < L ? WARPS : L;
        int i0 = 0, served = 0;
        for (int tile = tile0; tile < tile1; ++tile, i0 += nk) {
            if (tile != tile0 && tile % n_tiles == 0) served = 0;
            if (served++ < fresh)
                for (int kb = 0; kb < nk; ++kb) make[(i0 + kb) % par].push_back({i0 + kb, tile / n_tiles, kb});
        }
        for (int& s : seen) s = -1;
    }

    int total() const { return (tile1 - tile0) * nk; }

    bool tma() {
        if (t_i == total() || (t_i == FIRST && !started.test(0))) return false;
        const int s = t_i % L, turn = t_i / L;
        if (!empty[s].test((turn & 1) ^ 1)) return false;
        copies.push_back(s);
        ++t_i;
        return true;
    }
    bool copy() {
        if (copies.empty()) return false;
        ++full[copies.front()].phase;
        copies.pop_front();
        return true;
    }
    bool mma() {
        if (m_tile == tile1) return false;
        const int b = m_seg % ACCS;
        if (!m_in) {
            if (!acc_empty[b].test(((m_seg / ACCS) & 1) ^ 1)) return false;
            m_in = true;
        }
        if (m_served < fresh && !digits[m_s].test(made[m_s])) return false;
        if (!full[m_s].test(m_ph)) return false;
        if (m_served < fresh) made[m_s] ^= 1;
        ++begun;
        issued.push_back({m_s, m_tile / n_tiles, m_kb, -1});
        if (++m_s == L) {
            m_s = 0;
            m_ph ^= 1;
        }
        if (++m_kb == nk) {
            issued.push_back({0, 0, 0, b});
            m_kb = 0;
            m_in = false;
            ++m_seg;
            ++m_tile;
            ++m_served;
            if (++m_nt == n_tiles) m_nt = m_served = 0;
        }
        return true;
    }
    bool core() {
        if (issued.empty()) return false;
        const Issued x = issued.front();
        issued.pop_front();
        if (x.acc >= 0) {
            ++acc_full[x.acc].phase;
        } else {
            if (planes[x.slot] != std::make_pair(x.item, x.kb)) ++wrong;
            ++empty[x.slot].phase;
        }
        return true;
    }
    bool epilogue() {
        if (e_seg == tile1 - tile0) return false;
        const int b = e_seg % ACCS;
        if (!acc_full[b].test((e_seg / ACCS) & 1)) return false;
        ++acc_empty[b].phase;
        ++e_seg;
        return true;
    }
    bool convert(int w) {
        if (make[w].empty()) return false;
        const Make x = make[w].front();
        const int turn = x.i / L, s = x.i - turn * L;
        if (x.i - seen[w] > L && !qmm::f4_ring_may_wait(begun + early, x.i, L)) return false;
        if (!empty[s].test((turn & 1) ^ 1)) return false;
        seen[w] = x.i;
        planes[s] = {x.item, x.kb};
        ++digits[s].phase;
        if (x.i == 0) ++started.phase;
        make[w].pop_front();
        return true;
    }

    // 0 right, 1 wrong planes, 2 stopped
    int go() {
        // how often each takes a step: the tensor core from now and then to always
        const int slow = 1 + rnd(40);
        int idle = 0;
        while (e_seg < tile1 - tile0) {
            bool any = false;
            switch (rnd(5)) {
                case 0: any = tma(); break;
                case 1: any = copy(); break;
                case 2: any = mma(); break;
                case 3: any = rnd(slow) == 0 && (core() || epilogue()); break;
                default: any = convert(rnd(WARPS));
            }
            idle = any ? 0 : idle + 1;
            if (idle > 200000) return 2;
        }
        return wrong ? 1 : 0;
    }
};

}  // namespace

int main(int argc, char** argv) {
    const int runs = argc > 1 ? std::atoi(argv[1]) : 400;
    const unsigned seed = argc > 2 ? (unsigned)std::atoi(argv[2]) : 0;
    const int early = argc > 3 ? std::atoi(argv[3]) : 0;
    int bad = 0;
    for (int r = 0; r < runs; ++r) {
        Run run(seed + (unsigned)r, early);
        const int rc = run.go();
        if (!rc) continue;
        ++bad;
        std::printf("run %d: %s (%d k-blocks of %d tiles an item, tiles %d..%d)\n", r,
                    rc == 2 ? "stopped" : "wrong planes", run.nk, run.n_tiles, run.tile0, run.tile1);
    }
    std::printf("%d of %d\n", bad, runs);
    return 0;
}
