// The loading warps and the MMA warp of the many-row attention kernel as they wait for one another, walked under random and very uneven
// schedules.  Every wait is by parity, as the hardware's: it passes when the barrier's running phase has the other parity.  A wait must
// pass for the phase that it means, and the walk must end.
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <random>
#include <vector>

#include "lev_attn_ring.h"

static bool g_before;   // the rules without the arrivals of warps that have no box: must be caught

struct Bar {
    int count = 1, pending = 1, tx = 0, done = 0;
    void init(int c) { count = pending = c; }
    void settle() {
        if (pending == 0 && tx == 0) done++, pending = count;
    }
    void arrive(int expect = 0) { tx += expect, pending--, settle(); }
    void bytes(int n) { tx -= n, settle(); }
    bool passes(int parity) const { return (done & 1) != parity; }
};

// one step of an actor: a wait (returns false while it is closed) followed by what is done behind it
struct Op {
    Bar* bar = nullptr;
    int use = 0;   // the wait is for `use` completed phases
    std::function<void()> then;
};
typedef std::vector<Op> Actor;

struct Case {
    int cg, tiles, kv_stages, ring, box_k, box_v;   // boxes: rows of one; 0: a box per slab of 64 columns (packed rows)
    bool copy, q_boxes;
    std::vector<int> steps;   // of each unit
};

static int walk(const Case& C, unsigned seed, int slow) {
    std::mt19937 rng(seed);
    const int units = (int)C.steps.size(), loaders = C.cg * TC_LOAD_WARPS;
    std::vector<Bar> full(C.ring), empty(C.cg * C.ring), q_empty(C.cg), unit_full(2 * C.cg), unit_empty(2 * C.cg);
    Bar q_full;
    const bool arrive_all = !g_before;
    for (auto& b : full) b.init(arrive_all || C.copy ? tc_full_count(C.copy, C.cg) : 1);
    for (auto& b : unit_empty) b.init(TC_LOAD_WARPS);   // the MMA warp and the other two loading warps
    q_full.init(C.q_boxes ? 1 : TC_LOAD_WARPS * C.cg);
    std::vector<Actor> actors(loaders + 2);
    auto boxes = [&](int rank, int w, bool v) {   // that this warp fetches of a stage
        const int rows = C.cg == 2 && !v ? 64 : 128, box = v ? C.box_v : C.box_k;
        const int all = box ? rows / box : (C.cg == 2 && !v ? 4 : 2);
        int n = 0;
        for (int b = w; b < all; b += TC_LOAD_WARPS) n++;
        (void)rank;
        return n;
    };
    auto all_boxes = [&](bool v) {
        int n = 0;
        for (int w = 0; w < TC_LOAD_WARPS; w++) n += boxes(0, w, v);
        return n * C.cg;
    };
    for (int rank = 0; rank < C.cg; rank++)
        for (int w = 0; w < TC_LOAD_WARPS; w++) {
            Actor& a = actors[rank * TC_LOAD_WARPS + w];
            int at = 0;
            for (int k = 0; k < units; k++) {
                const int n = C.steps[k];
                auto load = [&](bool v) {
                    for (int h = 0; h < C.kv_stages; h++, at++) {
                        Bar *e = &empty[rank * C.ring + at % C.ring], *f = &full[at % C.ring];
                        const int mine = boxes(rank, w, v), all = all_boxes(v);
                        a.push_back({e, at / C.ring, [=, &C]() {
                                         if (C.copy) return f->arrive();
                                         if (rank == 0 && w == 0) f->arrive(all);
                                         if (mine) f->bytes(mine);
                                         if (arrive_all && tc_full_arrives(w)) f->arrive();
                                     }});
                    }
                };
                for (int i = 0; i <= n; i++) {
                    if (i < n) load(false);
                    if (i == 0) {
                        const bool waits = arrive_all ? tc_waits_for_queries(C.q_boxes, w) : true;
                        auto put = [=, &C, &q_full]() -> void {
                            if (!C.q_boxes) return q_full.arrive();
                            if (w) return;
                            if (rank == 0) q_full.arrive(C.cg);
                            q_full.bytes(1);
                        };
                        a.push_back({k > 0 && waits ? &q_empty[rank] : nullptr, k, put});
                    }
                    if (C.tiles == 2 ? i < n : i > 0) load(true);
                }
                Bar *f = &unit_full[2 * rank + ((k + 1) & 1)], *e = &unit_empty[2 * rank + ((k + 1) & 1)], *mine = &unit_empty[2 * rank + (k & 1)];
                if (w == 0) a.push_back({k > 0 ? e : nullptr, (k - 1) / 2 + 1, [=]() { f->arrive(); }});
                else a.push_back({nullptr, 0, [=]() { mine->arrive(); }}), a.push_back({f, k / 2 + 1, nullptr});
            }
            if (arrive_all ? tc_waits_for_queries(C.q_boxes, w) : true) a.push_back({&q_empty[rank], units, nullptr});
            for (int s = 0; s < C.ring; s++, at++) a.push_back({&empty[rank * C.ring + at % C.ring], at / C.ring, nullptr});
        }
    // MMA warps: the leader takes the stages, the second CTA's only keeps the units moving
    for (int rank = 0; rank < C.cg; rank++) {
        Actor& a = actors[loaders + rank];
        int at = 0;
        for (int k = 0; k < units; k++) {
            const int n = C.steps[k];
            if (rank == 0) {
                a.push_back({&q_full, k + 1, nullptr});
                auto take = [&]() {
                    for (int h = 0; h < C.kv_stages; h++, at++) {
                        const int s = at % C.ring;
                        a.push_back({&full[s], at / C.ring + 1, [=, &C, &empty]() {
                                         for (int r = 0; r < C.cg; r++) empty[r * C.ring + s].arrive();
                                     }});
                    }
                };
                auto free_q = [&]() {
                    a.push_back({nullptr, 0, [=, &C, &q_empty]() {
                                     for (int r = 0; r < C.cg; r++) q_empty[r].arrive();
                                 }});
                };
                // stages K0 V0 K1 V1 ... (two tiles) or K0 K1 V0 K2 V1 ...; the queries are free behind the last K
                for (int i = 0; i <= n; i++) {
                    if (i < n) take();
                    if (i == (n > 0 ? n - 1 : 0)) free_q();
                    if (C.tiles == 2 ? i < n : i > 0) take();
                }
            }
            Bar *f = &unit_full[2 * rank + ((k + 1) & 1)], *mine = &unit_empty[2 * rank + (k & 1)];
            a.push_back({nullptr, 0, [=]() { mine->arrive(); }});
            a.push_back({f, k / 2 + 1, nullptr});
        }
    }
    std::vector<size_t> pc(actors.size(), 0);
    for (long stuck = 0;;) {
        bool over = true;
        for (size_t i = 0; i < actors.size(); i++) over = over && pc[i] == actors[i].size();
        if (over) return 0;
        size_t i = rng() % actors.size();
        if ((int)i == slow && rng() % 400) i = rng() % actors.size() == 0 ? i : (i + 1) % actors.size();
        if (pc[i] == actors[i].size()) {
            if (++stuck > 2000000) return 1;
            continue;
        }
        const Op& op = actors[i][pc[i]];
        if (op.bar) {
            if (!op.bar->passes((op.use - 1) & 1)) {
                if (++stuck > 2000000) return 1;   // a phase that is over, or one that never comes
                continue;
            }
            if (op.bar->done != op.use) return 2;
        }
        if (op.then) op.then();
        pc[i]++;
        stuck = 0;
    }
}

int main(int argc, char** argv) {
    g_before = argc > 1;
    std::mt19937 rng(7);
    long walks = 0;
    for (int form = 0; form < 400; form++) {
        Case C;
        const int kind = form % 5;   // pairs, two tiles, one tile of 256, one tile of 128, copies
        C.cg = kind == 0 ? 2 : 1;
        C.tiles = kind == 1 ? 2 : 1;
        C.kv_stages = kind == 2 ? 2 : 1;
        C.ring = kind == 3 ? 6 : 5;
        C.copy = kind == 4;
        C.q_boxes = rng() % 2;
        const int boxes[] = {0, 8, 16, 32, 64, 128};
        C.box_v = C.copy ? 128 : boxes[rng() % 6];
        C.box_k = C.box_v > 128 / C.cg ? 128 / C.cg : C.box_v;
        const int units = 1 + rng() % 6;
        for (int u = 0; u < units; u++) C.steps.push_back(rng() % 5 == 0 ? 0 : 1 + rng() % (rng() % 3 ? 4 : 40));
        for (int slow = -1; slow < C.cg * TC_LOAD_WARPS; slow++, walks++)
            if (const int bad = walk(C, rng(), slow)) {
                printf("form %d (cg %d tiles %d ring %d box %d copy %d q_boxes %d) slow %d: %s\n", form, C.cg, C.tiles, C.ring, C.box_v, C.copy, C.q_boxes, slow,
                       bad == 1 ? "does not end" : "a wait passed for another phase");
                return 1;
            }
    }
    printf("%ld walks ok\n", walks);
    return 0;
}
