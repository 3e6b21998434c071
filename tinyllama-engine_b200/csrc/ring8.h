// ring8.h -- the ring of K/V tiles of chunk_few8_kernel (attend8.cu): its
// sizes, who works on what, and when a tile may be looked at.  Plain arithmetic,
// compiled for the host too, where tests/cpp/ring8_model.cpp runs it with
// copies that land in any order.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TLE_RING __host__ __device__ __forceinline__
#else
#define TLE_RING inline
#endif

namespace tle {

constexpr int F8_WARPS = 15;       // and the producer: 16 warps, so that a thread may have 128 registers
constexpr int F8_STAGES = 11;
// Teams: a segment ends with its warps' results joined, so a CTA with several segments of few tiles has 3 teams of 5
// warps, or 2 of 7, that work on segments in turn, each with its own barrier.  One team and as below: 100 x 1 behind 100
// with 8 KV heads (1 tile) 22.3 and 11.9 us, 256 x 1 behind up to 500 (3) 34.3 and 28.0, 64 x 1 behind up to 800 with 8 KV
// heads (5) 24.0 and 19.7, 256 x 1 behind up to 2000 (12) 60.9 and 58.6; behind up to 4000 (24 tiles) 93.7 and 104.8: the
// ring holds too few of them.  Where 4 row groups share 7 warps, 200 x 4 behind 1000 (8 tiles): 113 and 128, so one team.
constexpr int kThreeTeams = 4, kTwoTeams = 16;   // below so many tiles a segment
constexpr int kBatch = 3;          // tiles whose copies are issued at once
constexpr int kRingTile = 128;     // keys of a tile (kChunkTile)
constexpr int kStep = 32;          // keys of a step
constexpr int kSteps = kRingTile / kStep;
constexpr int kArrivals = 4 * kSteps;   // of a stage: a step of each of 1, 2 or 4 row groups arrives for 4, 2 or 1

// The teams of a CTA of n_segs segments with `tiles` tiles in all, the first of them of n_rows rows.
TLE_RING int ring_teams(int n_segs, int tiles, int n_rows) {
    const int each = n_segs > 0 ? (tiles - 1) / n_segs : 0;
    if (each < kThreeTeams) return n_segs < 3 ? n_segs : 3;
    return each < kTwoTeams && n_segs > 2 && n_rows <= 16 ? 2 : 1;
}
// Row groups of 8 rows: 1, 2 or 4 (as a power of two), a team's warps dealt out to them.
TLE_RING int ring_group_bits(int n_rows) { return n_rows <= 8 ? 0 : n_rows <= 16 ? 1 : 2; }
// Warps of row group rg: warp w of the team is the (w >> bits)th of group w % (1 << bits), and takes every so manieth
// step of a segment.
TLE_RING int ring_workers(int in_team, int bits, int rg) { return (in_team - rg + (1 << bits) - 1) >> bits; }

// Tile `ring` of the CTA's tiles, all segments' one after another, lies in this stage; the stage's barriers
// have this parity for it.
TLE_RING int ring_stage(int ring) { return ring % F8_STAGES; }
TLE_RING uint32_t ring_parity(int ring) { return (ring / F8_STAGES) & 1; }

// Whether tile `ring` has landed.  A barrier's parity tells a lap of the ring from the next one only, and a warp
// takes every so manieth step: it may never have met the stage's tile of the lap before, whose copies need not be the
// first to land.  So the stage's barrier is asked only once the producer has begun with tile `ring`
// (begun(ring)), which it does when the stage's last tile has been used by all.
template <class Begun, class Full>
TLE_RING bool ring_ready(int ring, Begun&& begun, Full&& full) {
    return begun(ring) && full(ring_stage(ring), ring_parity(ring));
}

}  // namespace tle
