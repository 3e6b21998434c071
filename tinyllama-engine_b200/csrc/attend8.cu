// attend8.cu -- attention of few new tokens over pages of 8 bits.
//
//   out_h(t) = sum_{j <= p} softmax_j(q_h(t) . k_{h/g}(j) / 8) v_{h/g}(j),
// k(j) = 2^(bk_j - 127) c_j with whole numbers c_j in -128..127, v(j) likewise
// (cache8.cu).  Rows (token t, head h of a KV head's group) and the split of
// the cache over CTAs are the chunk descriptor's: at most kChunkFewRows rows
// an item, 128-row tiles, partial results joined by chunk_merge_kernel.  Items
// of more rows go through chunk_attn_kernel over bf16 pages (stage8_kernel).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "chunk.cuh"
#include "common.cuh"
#include "kernels.h"
#include "ring8.h"
#include "tcgen05.cuh"

namespace tle {

namespace {

// Bound by the K/V bytes, 130 a row and KV head, where sequences are long; by a
// segment's start and end (its q, the joining) where they are short.  Tiles of codes
// come by TMA (a box is 64 or 128 rows of a page, two rows a line, 128-byte
// swizzle), their scales by bulk copies, into a ring that a producer warp keeps
// full across segments; 15 warps take 32-key steps of the tiles, each with its
// own running maximum, sum and output, joined in shared memory at the segment's
// end.
//
// Measured, 32 heads on 4 (us; bytes of K and V a second): 32 x 1 behind 8000 to 16000, bf16, 49.8,
// 4.3 TB/s (the copies alone, no step taken, 40.4); 64 x 1 behind 1023 to 2047, fp32, 19.5, 2.6 TB/s
// (13.6); 1 x 4 behind 700 10.7.  bf16 pages: 71.2, 25.1 and 10.2.  16 to 32 rows cost 2 or 4
// such passes over the codes, one for 8 rows: 32 x 4 behind 2000, bf16, 34.2, where bf16 pages take 20.3 (fp32 34.5 and 31.8).
//
// Tried: 8 to 11 stages, the same; two producers, scales by cp.async, q by copies and records
// read ahead, joining by a warp of its own or one segment late, no gain; 16- and 64-key steps, slower.
//
// The codes become fp16 on their way from shared memory into the fragments of
// m16n8k16 MMAs, exactly (a byte with its sign bit flipped, below the bits of
// 1024, less 1152), and K's and V's powers of two never meet an element: K's
// multiply the scores, V's the weights.  A tcgen05 tile would need the converted
// codes written back to shared memory, and 8 rows would leave it mostly empty.
// Matrices of 8 rows x 16 bytes are loaded as ones of 16-bit pairs, K as they lie
// and V transposed, so that bytes 0 and 2, and 1 and 3, of a register are a
// fragment's pair each: K's by a permutation of the 64 dimensions that q's
// fragments share, V's by two dimensions in turn.
//
// Precision: q (times a power of two per row) and the weights enter as sums of
// two fp16 numbers, 22 bits and rounding: within 2^-23 of a row's largest element,
// twice a rounding to 32 bits (4096 + 1 + 2^-11 becomes 4097).  A row of q whose largest element is below 2^-111 has
// fewer bits: its factor on the scores is then a subnormal number.  The second terms are rows 8 to 15 of the A
// fragments, so they cost no MMA.  Tensor cores cut their running sums off, so
// the output is carried on in 32-bit sums in shared memory every kFlush steps.
//
// The output's weights are 2^(s_j - m) 2^(bv_j - 127) f with a power of two f per row
// that keeps the largest one between 2^6 and 2^15, whatever V's scales are; m is a whole
// number.  So all rescaling is exact; m moves when exceeded by more than
// kMoveThreshold, f when a weight would be above 2^15.
constexpr int F8_THREADS = 32 * (F8_WARPS + 1);
static_assert(kRingTile == kTile, "the ring's tiles");
constexpr int kFlush = 4;          // steps of a warp whose MMAs are summed in a row
constexpr int kQBits = 12;         // the largest element of q in [2^12, 2^13)
constexpr int kWeightBits = 15, kWeightStart = 6;

// Rows of a copy: a tile, or two copies where a page is 64 rows.
__host__ __device__ constexpr int box_of(int page_shift) { return page_shift >= 7 ? kTile : kTile / 2; }

struct Few8Smem {
    uint8_t k[F8_STAGES][kTile * HD];
    uint8_t v[F8_STAGES][kTile * HD];
    uint8_t ks[F8_STAGES][kTile];
    uint8_t vs[F8_STAGES][kTile];
    float o[F8_WARPS][8][HD + 4];   // a warp's result, and its rows' maximum and sum
    float2 ml[F8_WARPS][8];
    uint64_t full[F8_STAGES], empty[F8_STAGES], work_full;
    int issued;                      // tiles that the producer has begun to copy
    Work work[kWorkCache];
};
struct Few8Tma {
    CUtensorMap k, v;   // the layer's codes as [n_pages * n_head_kv][page rows / 2][128], box {128, 32 or 64, 1}
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
// The count of begun tiles, between the producer and the warps: who reads it has seen what came before it.
__device__ __forceinline__ int load_acquire(const int* p) {
    int x;
    asm volatile("ld.acquire.cta.shared::cta.b32 %0, [%1];" : "=r"(x) : "r"(smem_u32(p)) : "memory");
    return x;
}
__device__ __forceinline__ void store_release(int* p, int x) {
    asm volatile("st.release.cta.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(p)), "r"(x) : "memory");
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// lo, hi as the sum of two pairs of fp16 numbers
__device__ __forceinline__ void two_terms(float lo, float hi, uint32_t& t0, uint32_t& t1) {
    t0 = pack_f16(lo, hi);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&t0));
    t1 = pack_f16(lo - f.x, hi - f.y);
}
// The codes in bytes 0 and 2 of u as fp16 numbers: (u & 00ff00ff) ^ 64806480 is 1024 + (code + 128).
__device__ __forceinline__ uint32_t codes_f16(uint32_t u) {
    uint32_t h, r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(h) : "r"(u), "r"(0x00ff00ffu), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));   // - 1152
    return r;
}
// 2^e, -127 <= e <= 127
__device__ __forceinline__ float pow2(int e) {
    return e < -126 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// 2^d for a whole number d <= 0 (or -inf).
__device__ __forceinline__ float pow2_down(float d) {
    return d < -126.f ? 0.f : __uint_as_float(static_cast<uint32_t>(static_cast<int>(d) + 127) << 23);
}

template <class Act>
__global__ void __launch_bounds__(F8_THREADS, 1)
    chunk_few8_kernel(const __grid_constant__ ChunkArgs A, const __grid_constant__ Pool8 P, const __grid_constant__ Few8Tma M) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Few8Smem& S = *reinterpret_cast<Few8Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < F8_STAGES; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], kArrivals);
        }
        mbar_init(&S.work_full, 1);
        S.issued = 0;
        fence_barrier_init();
        prefetch_tmap(&M.k);
        prefetch_tmap(&M.v);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid == 0) fetch_first(A, A.n_ctas + blockIdx.x, &S.work[0]);
    __syncthreads();
    const int seg0 = S.work[0].seg0, seg1 = S.work[0].seg1;
    bool failed = false, fetched = false;
    auto work_of = [&](int i) -> const Work& {
        if (i > seg0 && !fetched) {
            wait_or_flag(&S.work_full, 0, A.err, kErrWaitFull, failed);
            fetched = true;
        }
        return i - seg0 < kWorkCache ? S.work[i - seg0] : *static_cast<const Work*>(A.d.segs + i);
    };
    if (warp == F8_WARPS) {   // producer
        int ring = 0;
        const int box_rows = box_of(P.page_shift);
        const uint64_t policy = l2_evict_first_policy();
        for (int sg = seg0; sg < seg1; ++sg) {
            const Work w = work_of(sg);
            // lane l has the page of box b0 + l: -1 behind the last row, -2 outside the pool
            const int per_tile = kTile / box_rows;
            int b0 = per_tile * w.t0, id = -1;
            auto refill = [&]() {
                const int r = (b0 + lane) * box_rows;
                id = -1;
                if (r < w.kv_len && b0 + lane < per_tile * w.t1) {
                    id = w.pages[r >> P.page_shift];
                    if (static_cast<unsigned>(id) >= static_cast<unsigned>(P.n_pages)) {
                        record_error(A.err, kErrBadPage);
                        id = -2;
                    }
                }
            };
            refill();
            // up to kBatch tiles at once, one a lane: a turn of this loop takes about as long as the tiles' copies do
            for (int n0 = w.t0; n0 < w.t1; n0 += kBatch) {
                const int count = min(kBatch, w.t1 - n0);
                if (per_tile * (n0 + count) - b0 > 32) {
                    b0 = per_tile * n0;
                    refill();
                }
                const int n = n0 + min(lane, count - 1), mine = ring + n - n0, st = ring_stage(mine);
                const int id0 = __shfl_sync(0xffffffffu, id, per_tile * n - b0);
                const int id1 = per_tile == 2 ? __shfl_sync(0xffffffffu, id, per_tile * n - b0 + 1) : -1;
                wait_or_flag(&S.empty[st], ring_parity(mine) ^ 1, A.err, kErrWaitEmpty, failed);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                ring += count;
                if (lane == 0) store_release(&S.issued, ring);
                if (__any_sync(0xffffffffu, id0 == -2 || id1 == -2)) {
                    for (int e = 0; e < count * per_tile; ++e) {
                        const int to = __shfl_sync(0xffffffffu, st, e / per_tile), b = e % per_tile;
                        if (__shfl_sync(0xffffffffu, b ? id1 : id0, e / per_tile) != -2) continue;
                        for (int i = lane; i < box_rows * HD / 16; i += 32) {   // its rows count as zeros
                            reinterpret_cast<uint4*>(S.k[to] + b * box_rows * HD)[i] = make_uint4(0, 0, 0, 0);
                            reinterpret_cast<uint4*>(S.v[to] + b * box_rows * HD)[i] = make_uint4(0, 0, 0, 0);
                        }
                        if (lane < box_rows / 4) {
                            reinterpret_cast<uint32_t*>(S.ks[to] + b * box_rows)[lane] = 0x7f7f7f7fu;
                            reinterpret_cast<uint32_t*>(S.vs[to] + b * box_rows)[lane] = 0x7f7f7f7fu;
                        }
                    }
                    fence_proxy_async_smem();   // before the stage's next copy
                }
                __syncwarp();
                if (lane < count) {
                    mbar_arrive_expect_tx(&S.full[st], ((id0 >= 0) + (id1 >= 0)) * 2 * box_rows * (HD + 1));
                    for (int b = 0; b < per_tile; ++b) {
                        const int page = b ? id1 : id0;
                        if (page < 0) continue;
                        const int z = page * A.n_head_kv + w.kvh, y = (n * kTile + b * box_rows) & ((1 << P.page_shift) - 1);
                        const size_t row = (static_cast<size_t>(z) << P.page_shift) + y;
                        tma_load_3d(S.k[st] + b * box_rows * HD, &M.k, 0, y / 2, z, &S.full[st]);
                        bulk_g2s(S.ks[st] + b * box_rows, P.key_scale + row, box_rows, &S.full[st], policy);
                        tma_load_3d(S.v[st] + b * box_rows * HD, &M.v, 0, y / 2, z, &S.full[st]);
                        bulk_g2s(S.vs[st] + b * box_rows, P.value_scale + row, box_rows, &S.full[st], policy);
                    }
                }
                __syncwarp();
            }
            if (failed) break;
        }
        // no copy may still be in flight when the CTA leaves, after a wait that expired neither
        bool late = false;
        for (int u = ring > F8_STAGES ? ring - F8_STAGES : 0; u < ring; ++u)
            wait_or_flag(&S.full[ring_stage(u)], ring_parity(u), A.err, kErrDrain, late);
        return;
    }
    auto consume = [&]<bool ONE>(int n_teams) {
        const int in_team = ONE ? F8_WARPS : F8_WARPS / n_teams, team = ONE ? 0 : warp / in_team, tw = warp - team * in_team;
        const int every = ONE ? 1 : n_teams;
        if (!ONE && team >= n_teams) return;
        const int g = lane >> 2, t = lane & 3;        // fragment row, and which quarter of it
        const int mi = lane >> 3, li = lane & 7;      // ldmatrix: matrix and row of this lane's address
        // Rows lie in pairs in lines of 128 bytes: chunk q of row r, 16 bytes, is 4 (r % 2) + q of line r / 2 and
        // lies at that ^ (r / 2 % 8).  This lane's row of a step, chunks mi / 2 and mi / 2 + 2:
        uint32_t piece[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = li + 8 * (mi & 1), line = r >> 1;
            piece[h] = line * 2 * HD + ((((r & 1) * 4 + 2 * h + (mi >> 1)) ^ line) << 4);
        }
        static_assert(kChunkFewRows <= 32 && F8_WARPS < 32, "four row groups at most");
        // This lane's elements 16 c + 4 t .. + 3 of row g of the warp's group, ahead of the segment.
        using Raw = std::conditional_t<sizeof(Act) == 4, uint4, uint2>;
        Raw raw[HD / 16];
        auto load_q = [&](const Work& w) {
            const int r = (tw & ((1 << ring_group_bits(w.n_rows)) - 1)) * 8 + g;
            const bool ok = r < w.n_rows;
            const int row = w.row0 + (ok ? r : 0), tok = row_token(A, row), h = row - tok * A.group;
            const Raw* src = reinterpret_cast<const Raw*>(static_cast<const Act*>(A.q) +
                                                          static_cast<int64_t>(w.first + tok) * A.q_stride +
                                                          (w.kvh * A.group + h) * HD) + t;
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) raw[i] = ok ? src[4 * i] : Raw{};
        };
        int ring0 = 0;   // tiles of the segments before
        // (the count read at every step: kept in a register, more of them spill, and 32 x 1 behind 16000 takes 50.4 us, not 49.8)
        auto begun = [&](int ring) {
            uint64_t t_first = 0;
            for (int i = 1; load_acquire(&S.issued) <= ring && !failed; ++i) {
                if (i % 256 == 0) {
                    const uint64_t now = globaltimer();
                    if (t_first == 0) t_first = now;
                    if (now - t_first > kWaitTimeoutNs) {
                        record_error(A.err, kErrWaitFull);
                        failed = true;
                    }
                }
            }
            return !failed;
        };
        auto full = [&](int st, uint32_t parity) {
            wait_or_flag(&S.full[st], parity, A.err, kErrWaitFull, failed);
            return !failed;
        };
        auto segment = [&](const Work& w) {
            // w may lie in either memory: what the steps need of it is held in registers
            const int t0 = w.t0, pos_min = w.pos_min, kv_len = w.kv_len;
            const int gb = ring_group_bits(w.n_rows), rg = tw & ((1 << gb) - 1), kw = tw >> gb;
            const int pos_r = w.pos + row_token(A, w.row0 + min(rg * 8 + g, w.n_rows - 1));
            uint32_t qf[HD / 16][4];   // A fragments: rows g the first terms, rows g + 8 the second
            float c;                   // of the row's scores: 2^e / 8 log2(e), q = 2^e (terms)
            {
                float x[16];
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    if constexpr (sizeof(Act) == 4) {
                        x[4 * i] = __uint_as_float(raw[i].x);
                        x[4 * i + 1] = __uint_as_float(raw[i].y);
                        x[4 * i + 2] = __uint_as_float(raw[i].z);
                        x[4 * i + 3] = __uint_as_float(raw[i].w);
                    } else {
                        x[4 * i] = __uint_as_float(raw[i].x << 16);
                        x[4 * i + 1] = __uint_as_float(raw[i].x & 0xffff0000u);
                        x[4 * i + 2] = __uint_as_float(raw[i].y << 16);
                        x[4 * i + 3] = __uint_as_float(raw[i].y & 0xffff0000u);
                    }
                }
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmax3(most, fabsf(x[i]), 0.f);
                most = fmax3(most, __shfl_xor_sync(0xffffffffu, most, 1), 0.f);
                most = fmax3(most, __shfl_xor_sync(0xffffffffu, most, 2), 0.f);
                const bool fine = most <= 3.4028234e38f;   // otherwise every score is NaN
                // in two powers of two, neither of which leaves the range
                const float pre = most < 0x1p-60f ? 0x1p64f : 1.f;
                const int e = fine && most > 0.f ? static_cast<int>(__float_as_uint(most * pre) >> 23) - 127 - kQBits : 0;
                const float up = fine ? pow2(-e) : 0.f;
                c = fine ? kExpScale * pow2(e) * (1.f / pre) : NAN;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = fine ? x[i] * pre * up : 0.f;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    two_terms(x[4 * ks], x[4 * ks + 2], qf[ks][0], qf[ks][1]);
                    two_terms(x[4 * ks + 1], x[4 * ks + 3], qf[ks][2], qf[ks][3]);
                }
            }
            float m = -INFINITY, l = 0.f;
            int fe = 127;                             // f = 2^fe
            float f = pow2(127), limit = pow2(kWeightBits - 127);
            float o[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            int since = 0;
            bool flushed = false;
            // this lane's dimensions 16 c + 4 t .. + 3 of row g
            auto held = [&](int i) -> float4& { return *reinterpret_cast<float4*>(&S.o[warp][g][16 * i + 4 * t]); };
            auto flush = [&]() {
#pragma unroll
                for (int i = 0; i < HD / 16; ++i) {
                    float4 y = make_float4(o[2 * i][0] + o[2 * i][2], o[2 * i + 1][0] + o[2 * i + 1][2], o[2 * i][1] + o[2 * i][3],
                                           o[2 * i + 1][1] + o[2 * i + 1][3]);
                    if (flushed) {
                        const float4 z = held(i);
                        y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
                    }
                    held(i) = y;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
                flushed = true;
                since = 0;
            };
            auto scale_o = [&](float by) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] *= by;
                if (flushed)
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) {
                        const float4 z = held(i);
                        held(i) = make_float4(z.x * by, z.y * by, z.z * by, z.w * by);
                    }
            };
            // kStep keys from j0 of tile n in stage st; EDGE: some row does not attend to all of the tile.
            auto step = [&]<bool EDGE>(int st, int n, int j0) {
                constexpr int B = kStep / 8, N = kStep / 4;   // blocks of 8 keys; keys of a lane: 2 t, 2 t + 1 of each
                const int key0 = n * kTile + j0;
                if (EDGE && key0 >= kv_len) return;
                if (++since > kFlush) flush();
                const uint32_t kb = smem_u32(S.k[st]) + j0 * HD, vb = smem_u32(S.v[st]) + j0 * HD;
                float sf[B][4];
#pragma unroll
                for (int b2 = 0; b2 < B / 2; ++b2) {
                    // matrices: keys 0-7 and 8-15 of chunks 0, 1; then of 2, 3
                    uint32_t kr[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) ldsm4(kb + 16 * b2 * HD + piece[h], kr[h]);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const uint32_t u = kr[ks >> 1][2 * (ks & 1) + b];
                            if (ks == 0) mma_f16_zero(sf[2 * b2 + b], qf[ks], codes_f16(u), codes_f16(u >> 8));
                            else mma_f16(sf[2 * b2 + b], qf[ks], codes_f16(u), codes_f16(u >> 8));
                        }
                }
                float s[N], vsf[N];
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    const uint32_t kx = *reinterpret_cast<const uint16_t*>(&S.ks[st][j0 + 8 * b + 2 * t]);
                    const uint32_t vx = *reinterpret_cast<const uint16_t*>(&S.vs[st][j0 + 8 * b + 2 * t]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int i = 2 * b + e;
                        s[i] = (sf[b][e] + sf[b][2 + e]) * (__uint_as_float((e ? kx << 15 : kx << 23) & 0x7f800000u) * c);
                        vsf[i] = __uint_as_float((e ? vx << 15 : vx << 23) & 0x7f800000u);
                        if (EDGE && key0 + 8 * b + 2 * t + e > pos_r) {
                            s[i] = -INFINITY;
                            vsf[i] = 0.f;
                        }
                    }
                }
                float mt = s[0];
#pragma unroll
                for (int i = 1; i + 1 < N; i += 2) mt = fmax3(mt, s[i], s[i + 1]);
                mt = fmax3(mt, s[N - 1], s[N - 1]);
                if (__any_sync(0xffffffffu, m == m && !(mt <= m + kMoveThreshold))) {
                    float to = fmax3(mt, __shfl_xor_sync(0xffffffffu, mt, 1), -INFINITY);
                    to = fmax3(to, __shfl_xor_sync(0xffffffffu, to, 2), -INFINITY);
                    float by = 1.f;
                    if (m == m && !(to <= m + kMoveThreshold)) {
                        to = ceilf(to);
                        if (m != -INFINITY) {
                            // weights of the new m are smaller by 2^(m - to): f makes up for it, as far as it goes
                            l *= pow2_down(m - to);
                            const float e = static_cast<float>(fe) + (to - m);
                            by = pow2_down(fminf(127.f - e, 0.f));
                            fe = static_cast<int>(fminf(e, 127.f));
                            f = pow2(fe);
                            limit = pow2(min(kWeightBits - fe, 127));
                        }
                        m = to;
                    }
                    if (__any_sync(0xffffffffu, by != 1.f)) scale_o(by);
                }
                const float m_use = m == -INFINITY ? 0.f : m;   // nothing attended so far: the scores are -inf
                float wt[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float p = ex2_sfu(s[i] - m_use);
                    l += p;
                    wt[i] = p * vsf[i];
                }
                float wm = wt[0];
#pragma unroll
                for (int i = 1; i + 1 < N; i += 2) wm = fmax3(wm, wt[i], wt[i + 1]);
                wm = fmax3(wm, wt[N - 1], wt[N - 1]);
                if (__any_sync(0xffffffffu, !(wm <= limit))) {
                    float to = fmax3(wm, __shfl_xor_sync(0xffffffffu, wm, 1), 0.f);
                    to = fmax3(to, __shfl_xor_sync(0xffffffffu, to, 2), 0.f);
                    float by = 1.f;
                    if (to > limit && to <= 3.4028234e38f) {
                        const int e = max(kWeightStart + 127 - static_cast<int>(__float_as_uint(to) >> 23), -126);
                        by = pow2_down(static_cast<float>(e - fe));
                        fe = e;
                        f = pow2(fe);
                        limit = pow2(min(kWeightBits - fe, 127));
                    }
                    scale_o(by);
                }
#pragma unroll
                for (int b2 = 0; b2 < B / 2; ++b2) {
                    uint32_t vr[2][4], pf[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) ldsm4_t(vb + 16 * b2 * HD + piece[h], vr[h]);
                    two_terms(wt[4 * b2] * f, wt[4 * b2 + 1] * f, pf[0], pf[1]);
                    two_terms(wt[4 * b2 + 2] * f, wt[4 * b2 + 3] * f, pf[2], pf[3]);
#pragma unroll
                    for (int q = 0; q < HD / 16; ++q) {   // chunk q: dimensions 16 q + 2 g (+1)
                        const uint32_t u0 = vr[q >> 1][2 * (q & 1)], u1 = vr[q >> 1][2 * (q & 1) + 1];
                        mma_f16(o[2 * q], pf, codes_f16(u0), codes_f16(u1));
                        mma_f16(o[2 * q + 1], pf, codes_f16(u0 >> 8), codes_f16(u1 >> 8));
                    }
                }
            };
            // the steps of the segment, dealt out to the group's warps
            const int n_steps = (w.t1 - t0) * kSteps, nkw = ring_workers(in_team, gb, rg);
            for (int i = kw; i < n_steps; i += nkw) {
                const int n = t0 + i / kSteps, ring = ring0 + i / kSteps, st = ring_stage(ring);
                ring_ready(ring, begun, full);   // after a wait that expired the warp goes on, in bounds
                __syncwarp();
                if (n * kTile + kTile - 1 > pos_min) step.template operator()<true>(st, n, kStep * (i % kSteps));
                else step.template operator()<false>(st, n, kStep * (i % kSteps));
                __syncwarp();
                if (lane == 0) mbar_arrive_n(&S.empty[st], kArrivals / kSteps >> gb);
            }
            flush();
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (t == 0) S.ml[warp][g] = make_float2(m, l);
            const float back = pow2(-fe);   // to the weights 2^(s - m)
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                const float4 z = held(i);
                held(i) = make_float4(z.x * back, z.y * back, z.z * back, z.w * back);
            }
        };
        if (ONE && seg0 < seg1) load_q(S.work[0]);
        if (warp == (ONE ? F8_WARPS - 1 : 0)) fetch_work(A, seg0, seg1, S.work, &S.work_full);
        if (!ONE && seg0 + team < seg1) load_q(work_of(seg0 + team));
        for (int i = 0; i < team; ++i) ring0 += work_of(seg0 + i).t1 - work_of(seg0 + i).t0;
        for (int sg = seg0 + team; sg < seg1; sg += every) {
            const Work& w = work_of(sg);
            segment(w);
            if (sg + every < seg1) {
                ring0 += w.t1 - w.t0;
                if (!ONE)
                    for (int i = sg + 1; i < sg + every; ++i) ring0 += work_of(i).t1 - work_of(i).t0;
                load_q(work_of(sg + every));
            }
            named_bar_sync(1 + team, 32 * in_team);
            // ---- join the key workers: a row per warp, two columns per lane; lane q has the
            // weight of worker q ----
            const int gb = ring_group_bits(w.n_rows);
            for (int r = tw; r < w.n_rows; r += in_team) {
                const int w0 = r >> 3, rr = r & 7, nkw = ring_workers(in_team, gb, w0);
                const float2 ml = lane < nkw ? S.ml[team * in_team + w0 + (lane << gb)][rr] : make_float2(-INFINITY, 0.f);
                float m_all = ml.x;
#pragma unroll
                for (int d = 1; d < 16; d *= 2) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, d));
                const float fw = ml.x == -INFINITY ? 0.f : ex2_sfu(ml.x - m_all);
                float l_all = fw == 0.f ? 0.f : fw * ml.y;
#pragma unroll
                for (int d = 1; d < 16; d *= 2) l_all += __shfl_xor_sync(0xffffffffu, l_all, d);
                float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < F8_WARPS; ++q) {
                    const float fq = __shfl_sync(0xffffffffu, fw, q);
                    if (q < nkw && fq != 0.f) {
                        const float2 x = *reinterpret_cast<const float2*>(&S.o[team * in_team + w0 + (q << gb)][rr][2 * lane]);
                        acc.x = fmaf(fq, x.x, acc.x);
                        acc.y = fmaf(fq, x.y, acc.y);
                    }
                }
                const float l_row = __shfl_sync(0xffffffffu, l_all, 0), m_row = __shfl_sync(0xffffffffu, m_all, 0);
                const bool empty = l_row == 0.f;   // no row of this segment has a weight
                const float inv = empty ? 0.f : 1.0f / l_row;
                acc = empty ? make_float2(no_weight(w), no_weight(w)) : make_float2(acc.x * inv, acc.y * inv);
                const RowOut<Act> dst = row_out<Act>(A, w, r);
                if (dst.out) store_pair(dst.out + 2 * lane, acc);
                else store_pair(dst.part + 2 * lane, acc);
                if (dst.lse && lane == 0) *dst.lse = empty ? -INFINITY : m_row + log2f(l_row);
            }
            named_bar_sync(1 + team, 32 * in_team);
        }
    };
    const int n_segs = seg1 - seg0;
    const int n_teams = ring_teams(n_segs, n_segs > 0 ? S.work[0].cta_tiles : 0, n_segs > 0 ? S.work[0].n_rows : 0);
    if (n_teams <= 1) consume.template operator()<true>(1);
    else consume.template operator()<false>(n_teams);
}

template <class Act>
cudaError_t launch_few8(const ChunkArgs& a, const Pool8& pool, cudaStream_t stream) {
    Few8Tma m;
    const uint64_t heads = static_cast<uint64_t>(pool.n_pages) * a.n_head_kv, rows = uint64_t{1} << pool.page_shift;
    cudaError_t me = make_tmap_3d_8b(&m.k, pool.key_codes, rows / 2, heads, box_of(pool.page_shift) / 2);
    if (me != cudaSuccess) return me;
    me = make_tmap_3d_8b(&m.v, pool.value_codes, rows / 2, heads, box_of(pool.page_shift) / 2);
    if (me != cudaSuccess) return me;
    constexpr size_t smem = sizeof(Few8Smem) + 1024;
    static_assert(smem <= 232448, "shared memory of one SM");
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        return cudaFuncSetAttribute(chunk_few8_kernel<Act>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    });
    if (e != cudaSuccess) return e;
    Launch L(dim3(a.n_few_ctas), F8_THREADS, smem, stream);
    return cudaLaunchKernelEx(&L.cfg, chunk_few8_kernel<Act>, a, pool, m);
}

}  // namespace

cudaError_t launch_chunk_few8(const ChunkArgs& a, const Pool8& pool, bool act_bf16, cudaStream_t stream) {
    return act_bf16 ? launch_few8<__nv_bfloat16>(a, pool, stream) : launch_few8<float>(a, pool, stream);
}

}  // namespace tle
