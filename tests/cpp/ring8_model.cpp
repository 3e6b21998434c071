// Runs the ring of K/V tiles of attend8.cu (csrc/ring8.h) on the CPU: a producer, the warps of one to three teams and
// copies that land in any order, one event at a time, in orders drawn from many seeds, among them ones that hold back one
// tile's copy or one warp as long as anything else can happen.  Prints what went wrong first in each case, and
// returns 1 if anything did:
//   early    a warp took a tile that had not landed
//   late     a copy was begun into a stage that some warp had not read yet
//   twice    an arrival at a barrier that expected none in this phase
//   stuck    nothing could go on
// `ring8_model plain` leaves ring_ready's first question out, which the model has to find.
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <random>
#include <string>
#include <vector>

#include "ring8.h"

using namespace tle;

namespace {

struct Barrier {   // an mbarrier: phases, each complete once so many have arrived and all bytes are there
    int count = 0, pending = 0, copies = 0;
    uint32_t phase = 0;
    void init(int n) { count = pending = n; }
    bool arrive(int n, int more_copies) {
        copies += more_copies;
        if (n > pending) return false;
        pending -= n;
        turn();
        return true;
    }
    void landed() {
        --copies;
        turn();
    }
    void turn() {
        if (pending == 0 && copies == 0) {
            ++phase;
            pending = count;
        }
    }
    bool passed(uint32_t parity) const { return (phase & 1) != parity; }   // as test_wait.parity
};

struct Segment {
    int tiles, rows;
};
struct Case {
    const char* name;
    std::vector<Segment> segs;
    int teams;   // 0: as ring_teams says
};

struct Step {
    int ring;      // -1: the team's barrier
    int arrivals;
};

// What a run holds back: nothing, the copy of tile `which`, or warp `which`.
enum Hold { kNone, kCopy, kWarp };

std::string run(const Case& c, bool asks, unsigned seed, Hold hold, int which) {
    std::mt19937 rng(seed);
    int all = 0;
    std::vector<int> first;
    for (const Segment& s : c.segs) {
        first.push_back(all);
        all += s.tiles;
    }
    const int teams = c.teams ? c.teams : ring_teams(static_cast<int>(c.segs.size()), all, c.segs[0].rows);
    const int in_team = F8_WARPS / teams, warps = in_team * teams;
    // every warp's steps, in order
    std::vector<std::vector<Step>> steps(warps);
    std::vector<int> due(all, 0);   // arrivals that a tile still waits for
    for (int w = 0; w < warps; ++w) {
        const int team = w / in_team, tw = w % in_team;
        for (size_t s = team; s < c.segs.size(); s += teams) {
            const int bits = ring_group_bits(c.segs[s].rows), rg = tw & ((1 << bits) - 1);
            for (int i = tw >> bits; i < c.segs[s].tiles * kSteps; i += ring_workers(in_team, bits, rg)) {
                steps[w].push_back({first[s] + i / kSteps, kArrivals / kSteps >> bits});
                due[first[s] + i / kSteps] += kArrivals / kSteps >> bits;
            }
            steps[w].push_back({-1, 0});
        }
    }
    for (int n = 0; n < all; ++n)
        if (due[n] != kArrivals) return "a tile's arrivals are not " + std::to_string(kArrivals);
    Barrier full[F8_STAGES], empty[F8_STAGES];
    for (int i = 0; i < F8_STAGES; ++i) {
        full[i].init(1);
        empty[i].init(kArrivals);
    }
    int holds[F8_STAGES];   // the tile whose bytes a stage has; -1: none, or bytes on their way
    for (int& h : holds) h = -1;
    int issued = 0, copied = 0;            // tiles begun, and tiles whose copies are on their way or landed
    std::vector<int> flying;               // tiles
    std::vector<size_t> at(warps, 0);
    std::vector<char> reading(warps, 0), waits(warps, 0);   // in a step; at the team's barrier
    size_t seg = 0;
    int in_seg = 0;                        // the producer's place
    struct Event {
        int kind, who;   // 0 a copy lands, 1 the producer, 2 a warp
    };
    std::vector<Event> now, held;
    for (;;) {
        now.clear();
        held.clear();
        auto offer = [&](int kind, int who, bool late) { (late ? held : now).push_back({kind, who}); };
        for (size_t i = 0; i < flying.size(); ++i) offer(0, static_cast<int>(i), hold == kCopy && flying[i] == which);
        int batch = 0;
        if (copied < issued) {
            offer(1, 0, false);
        } else if (seg < c.segs.size()) {
            batch = std::min(kBatch, c.segs[seg].tiles - in_seg);
            bool go = true;
            for (int b = 0; b < batch; ++b) go = go && empty[ring_stage(issued + b)].passed(ring_parity(issued + b) ^ 1);
            if (go) offer(1, 0, false);
        }
        bool done = true;
        for (int w = 0; w < warps; ++w) {
            if (at[w] >= steps[w].size()) continue;
            done = false;
            const Step& s = steps[w][at[w]];
            bool go = false;
            if (reading[w]) {
                go = true;
            } else if (s.ring < 0) {
                go = !waits[w];   // arriving; the last one frees the team
            } else {
                go = ring_ready(
                    s.ring, [&](int ring) { return !asks || issued > ring; },
                    [&](int st, uint32_t parity) { return full[st].passed(parity); });
            }
            if (go) offer(2, w, hold == kWarp && w == which);
        }
        if (done && seg == c.segs.size() && copied == issued && flying.empty()) return "";
        std::vector<Event>& from = now.empty() ? held : now;
        if (from.empty()) return "stuck";
        const Event e = from[rng() % from.size()];
        if (e.kind == 0) {
            const int n = flying[e.who];
            flying.erase(flying.begin() + e.who);
            holds[ring_stage(n)] = n;
            full[ring_stage(n)].landed();
        } else if (e.kind == 1 && copied < issued) {
            const int n = copied++, st = ring_stage(n);
            if (n >= F8_STAGES && due[n - F8_STAGES] != 0) return "late: tile " + std::to_string(n);
            for (int w = 0; w < warps; ++w)
                if (reading[w] && ring_stage(steps[w][at[w]].ring) == st) return "late: tile " + std::to_string(n);
            holds[st] = -1;
            if (!full[st].arrive(1, 1)) return "twice: tile " + std::to_string(n);
            flying.push_back(n);
        } else if (e.kind == 1) {
            issued += batch;
            in_seg += batch;
            if (in_seg == c.segs[seg].tiles) {
                ++seg;
                in_seg = 0;
            }
        } else {
            const int w = e.who;
            const Step& s = steps[w][at[w]];
            if (s.ring < 0) {
                waits[w] = 1;
                const int t0 = w / in_team * in_team;
                bool last = true;
                for (int v = t0; v < t0 + in_team; ++v) last = last && waits[v];
                if (last)
                    for (int v = t0; v < t0 + in_team; ++v) {
                        waits[v] = 0;
                        ++at[v];
                    }
            } else if (!reading[w]) {
                if (holds[ring_stage(s.ring)] != s.ring) return "early: tile " + std::to_string(s.ring) + " by warp " + std::to_string(w);
                reading[w] = 1;
            } else {
                reading[w] = 0;
                due[s.ring] -= s.arrivals;
                if (!empty[ring_stage(s.ring)].arrive(s.arrivals, 0)) return "twice: a step of tile " + std::to_string(s.ring);
                ++at[w];
            }
        }
    }
}

}  // namespace

int main(int argc, char** argv) {
    const bool asks = !(argc > 1 && strcmp(argv[1], "plain") == 0);
    const std::vector<Case> cases = {
        {"one team, 8 rows", {{40, 8}}, 0},
        {"one team, 16 rows", {{40, 16}}, 0},
        {"one team, 32 rows", {{40, 32}}, 0},
        {"one team, three segments", {{30, 8}, {17, 8}, {13, 8}}, 0},
        {"one team, kinds of rows", {{19, 8}, {12, 16}, {25, 32}}, 0},
        {"one team, two segments of 12", {{12, 1}, {12, 1}}, 0},
        {"two teams", {{12, 8}, {5, 8}, {14, 8}, {9, 8}}, 2},
        {"two teams, kinds of rows", {{12, 16}, {7, 8}, {14, 32}, {9, 16}, {6, 8}}, 2},
        {"three teams", {{1, 8}, {2, 8}, {1, 8}, {4, 8}, {3, 8}, {1, 8}, {2, 8}}, 3},
        {"three teams, a long segment", {{1, 8}, {30, 16}, {2, 32}, {1, 8}, {2, 8}, {1, 8}, {3, 8}, {2, 8}}, 3},
    };
    int bad = 0;
    for (const Case& c : cases) {
        int all = 0;
        for (const Segment& s : c.segs) all += s.tiles;
        std::string why;
        for (unsigned seed = 0; seed < 40 && why.empty(); ++seed) why = run(c, asks, seed, kNone, 0);
        for (int n = 0; n < all && why.empty(); ++n)
            for (unsigned seed = 0; seed < 3 && why.empty(); ++seed) why = run(c, asks, 100 + seed, kCopy, n);
        for (int w = 0; w < F8_WARPS && why.empty(); ++w)
            for (unsigned seed = 0; seed < 3 && why.empty(); ++seed) why = run(c, asks, 200 + seed, kWarp, w);
        printf("%s: %s\n", c.name, why.empty() ? "ok" : why.c_str());
        bad += !why.empty();
    }
    return bad != 0;
}
