// attend8.cu -- attention of few new tokens over pages of 8 bits.
//
//   out_h(t) = sum_{j <= p} softmax_j(q_h(t) . k_{h/g}(j) / 8) v_{h/g}(j),
// k(j) = 2^(bk_j - 127) c_j with whole numbers c_j in -128..127, v(j) likewise
// (cache8.cu).  Rows (token t, head h of a KV head's group) and the split of
// the cache over CTAs are the chunk descriptor's: at most kChunkFewRows rows
// an item, 128-row tiles, partial results joined by chunk_merge_kernel.  Items
// of more rows go through chunk_attn_kernel over bf16 pages (stage8_kernel).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "chunk.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tle {

namespace {

// Bound by the K/V bytes, 130 a row and KV head.  Tiles come by 1-D bulk
// copies (a head's rows of a page are contiguous) into a ring that a producer
// warp keeps full across segments; 16 warps take 16-key steps of the tiles,
// each with its own running maxima, sum and output, joined in shared memory at
// the segment's end.
//
// The codes become fp16 on their way from shared memory into the fragments of
// m16n8k16 MMAs, exactly (the byte with its sign bit flipped, below the bits of
// 1024, less 1152), and K's and V's powers of two never meet an element: K's
// multiply the scores, V's go into the exponent of the weights.  A tcgen05
// tile would need the converted codes written back to shared memory, and 8
// rows would leave it mostly empty.
//
// Which key is column c of a step's first or second 8 is free, and so is the
// order of the 64 dimensions in a product over them: lane (g, t) takes
// K's bytes 16 t .. 16 t + 15 of one key per 8 (one 16-byte load), and V's bytes
// 8 g .. 8 g + 7 of the keys t, t + 4, t + 8, t + 12 of the step (columns 2 t, 2 t + 1
// of either 8), so that no load has bank conflicts and neither K nor V is
// transposed.
//
// Precision: q (times a power of two per row) and the weights enter as sums of
// two fp16 numbers, 22 bits and rounding: within 2^-24 of the largest element,
// as 32-bit arithmetic is.  The second terms are rows 8 to 15 of the A
// fragments, so they cost no MMA.  Tensor cores cut their running sums off, so
// the output is carried on in 32-bit registers every kFlush steps.
//
// The weights of the output are w_j = 2^(s_j + e_j - m2), e_j = bv_j - 127, with a
// running maximum m2 of their own beside m for the sum of 2^(s_j - m): whatever
// V's scales, the largest contribution has the largest weight.  Both maxima are whole
// numbers, so that rescaling is exact, and move only when exceeded by more than
// kMoveThreshold.
constexpr int F8_WARPS = 16;
constexpr int F8_THREADS = 32 * (F8_WARPS + 1);
constexpr int F8_STAGES = 8;
constexpr int kFlush = 8;          // steps of a warp whose MMAs are summed in a row
constexpr int kBox8 = 64;          // rows of a bulk copy: the smallest page
constexpr float kWeightBits = 7.f; // w <= 2^(kWeightBits + kMoveThreshold) = 2^15
constexpr int kQBits = 12;         // the largest element of q in [2^12, 2^13)

struct Stage8 {
    uint8_t k[kTile * HD];
    uint8_t v[kTile * HD];
    uint8_t ks[kTile];
    uint8_t vs[kTile];
};
struct Few8Smem {
    Stage8 st[F8_STAGES];
    float o[F8_WARPS][8][HD + 4];   // a warp's result, and its rows' maximum and sum
    float2 ml[F8_WARPS][8];
    uint64_t full[F8_STAGES], empty[F8_STAGES], work_full;
    Work work[kWorkCache];
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
// The codes in bytes 0 and 2 of u as fp16 numbers.
__device__ __forceinline__ uint32_t codes_f16(uint32_t u) {
    const uint32_t h = (u & 0x00ff00ffu) ^ 0x64806480u;   // 1024 + (code + 128)
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));   // - 1152
    return r;
}
// 2^d for a whole number d <= 0 (or -inf).
__device__ __forceinline__ float pow2_down(float d) {
    return d < -126.f ? 0.f : __uint_as_float(static_cast<uint32_t>(static_cast<int>(d) + 127) << 23);
}
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int t) { return (w >> (8 * t)) & 0xffu; }

template <class Act>
__global__ void __launch_bounds__(F8_THREADS, 1)
    chunk_few8_kernel(const __grid_constant__ ChunkArgs A, const __grid_constant__ Pool8 P) {
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Few8Smem& S = *reinterpret_cast<Few8Smem*>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < F8_STAGES; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], F8_WARPS);
        }
        mbar_init(&S.work_full, 1);
        fence_barrier_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid == 0) fetch_first(A, A.n_ctas + blockIdx.x, &S.work[0]);
    __syncthreads();
    const int seg0 = S.work[0].seg0, seg1 = S.work[0].seg1;
    bool failed = false;
    auto work_of = [&](int i) -> const Work& {
        if (i == seg0 + 1) wait_or_flag(&S.work_full, 0, A.err, kErrWaitFull, failed);
        return i - seg0 < kWorkCache ? S.work[i - seg0] : *static_cast<const Work*>(A.d.segs + i);
    };
    if (warp == F8_WARPS) {   // producer
        int ring = 0;
        const uint64_t policy = l2_evict_first_policy();
        for (int sg = seg0; sg < seg1; ++sg) {
            const Work w = work_of(sg);
            // lane l has the page of box b0 + l: -1 behind the last row, -2 outside the pool
            int b0 = 2 * w.t0, id = -1;
            auto refill = [&]() {
                const int r = (b0 + lane) * kBox8;
                id = -1;
                if (r < w.kv_len && b0 + lane < 2 * w.t1) {
                    id = w.pages[r >> P.page_shift];
                    if (static_cast<unsigned>(id) >= static_cast<unsigned>(P.n_pages)) {
                        record_error(A.err, kErrBadPage);
                        id = -2;
                    }
                }
            };
            refill();
            for (int n = w.t0; n < w.t1; ++n, ++ring) {
                if (2 * n - b0 >= 32) {
                    b0 = 2 * n;
                    refill();
                }
                const int st = ring % F8_STAGES;
                const int ids[2] = {__shfl_sync(0xffffffffu, id, 2 * n - b0), __shfl_sync(0xffffffffu, id, 2 * n - b0 + 1)};
                wait_or_flag(&S.empty[st], ((ring / F8_STAGES) & 1) ^ 1, A.err, kErrWaitEmpty, failed);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                Stage8& T = S.st[st];
                int boxes = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    boxes += ids[b] >= 0;
                    if (ids[b] != -2) continue;
                    for (int i = lane; i < kBox8 * HD / 16; i += 32) {   // its rows count as zeros
                        reinterpret_cast<uint4*>(T.k + b * kBox8 * HD)[i] = make_uint4(0, 0, 0, 0);
                        reinterpret_cast<uint4*>(T.v + b * kBox8 * HD)[i] = make_uint4(0, 0, 0, 0);
                    }
                    if (lane < kBox8 / 4) {
                        reinterpret_cast<uint32_t*>(T.ks + b * kBox8)[lane] = 0x7f7f7f7fu;
                        reinterpret_cast<uint32_t*>(T.vs + b * kBox8)[lane] = 0x7f7f7f7fu;
                    }
                    fence_proxy_async_smem();   // before the stage's next copy
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_expect_tx(&S.full[st], boxes * 2 * (kBox8 * HD + kBox8));
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if (ids[b] < 0) continue;
                        const size_t row = ((static_cast<size_t>(ids[b]) * A.n_head_kv + w.kvh) << P.page_shift) +
                                           (((2 * n + b) * kBox8) & ((1 << P.page_shift) - 1));
                        bulk_g2s(T.k + b * kBox8 * HD, P.key_codes + row * HD, kBox8 * HD, &S.full[st], policy);
                        bulk_g2s(T.ks + b * kBox8, P.key_scale + row, kBox8, &S.full[st], policy);
                        bulk_g2s(T.v + b * kBox8 * HD, P.value_codes + row * HD, kBox8 * HD, &S.full[st], policy);
                        bulk_g2s(T.vs + b * kBox8, P.value_scale + row, kBox8, &S.full[st], policy);
                    }
                }
                __syncwarp();
            }
            if (failed) break;
        }
        // no copy may still be in flight when the CTA leaves, after a wait that expired neither
        bool late = false;
        for (int u = ring > F8_STAGES ? ring - F8_STAGES : 0; u < ring; ++u)
            wait_or_flag(&S.full[u % F8_STAGES], (u / F8_STAGES) & 1, A.err, kErrDrain, late);
        return;
    }
    const int g = lane >> 2, t = lane & 3;   // fragment row, and which quarter of it
    static_assert(kChunkFewRows <= 32 && F8_WARPS % 4 == 0, "four row groups at most");
    // row groups of 8 rows: 1, 2 or 4, each by F8_WARPS / groups warps
    auto row_groups = [](int n_rows) { return n_rows <= 8 ? 1 : n_rows <= 16 ? 2 : 4; };
    // This lane's 16 elements of row g of the warp's group, ahead of the segment.
    constexpr int kRaw = 16 * sizeof(Act) / 16;
    uint4 raw[kRaw];
    auto load_q = [&](const Work& w) {
        const int r = warp % row_groups(w.n_rows) * 8 + g;
        const bool ok = r < w.n_rows;
        const int row = w.row0 + (ok ? r : 0), tok = row_token(A, row), h = row - tok * A.group;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const Act*>(A.q) +
                                                          static_cast<int64_t>(w.first + tok) * A.q_stride +
                                                          (w.kvh * A.group + h) * HD + 16 * t);
#pragma unroll
        for (int i = 0; i < kRaw; ++i) raw[i] = ok ? src[i] : make_uint4(0, 0, 0, 0);
    };
    int ring = 0;
    auto segment = [&](const Work& w) {
        const int rgroups = row_groups(w.n_rows), nkw = F8_WARPS / rgroups;
        const int rg = warp % rgroups, kw = warp / rgroups;
        const int pos_r = w.pos + row_token(A, w.row0 + min(rg * 8 + g, w.n_rows - 1));
        uint32_t qf[HD / 16][4];   // A fragments: rows g the first terms, rows g + 8 the second
        float c;                   // of the row's scores: 2^e / 8 log2(e), q = 2^e (terms)
        {
            float x[16];
            if constexpr (sizeof(Act) == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[4 * i] = __uint_as_float(raw[i].x);
                    x[4 * i + 1] = __uint_as_float(raw[i].y);
                    x[4 * i + 2] = __uint_as_float(raw[i].z);
                    x[4 * i + 3] = __uint_as_float(raw[i].w);
                }
            } else {
                float y[8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    bf16x8(raw[i], y);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[8 * i + e] = y[e];
                }
            }
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmax3(most, fabsf(x[i]), 0.f);
            most = fmax3(most, __shfl_xor_sync(0xffffffffu, most, 1), 0.f);
            most = fmax3(most, __shfl_xor_sync(0xffffffffu, most, 2), 0.f);
            const bool fine = most <= 3.4028234e38f;   // otherwise every score is NaN
            const int e = fine && most > 0.f ? ilogbf(most) - kQBits : 0;
            c = fine ? ldexpf(kExpScale, e) : NAN;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fine ? ldexpf(x[i], -e) : 0.f;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                two_terms(x[4 * ks], x[4 * ks + 1], qf[ks][0], qf[ks][1]);
                two_terms(x[4 * ks + 2], x[4 * ks + 3], qf[ks][2], qf[ks][3]);
            }
        }
        float m = -INFINITY, m2 = -INFINITY, l = 0.f;
        float o[8][4], sum[8][2];   // sum: what o held before
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            sum[j][0] = sum[j][1] = 0.f;
        }
        int since = 0;
        auto flush = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[j][0] += o[j][0] + o[j][2];
                sum[j][1] += o[j][1] + o[j][3];
                o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            }
            since = 0;
        };
        // 16 keys from j0 of tile n in T; EDGE: some row does not attend to all of the tile.
        auto step = [&]<bool EDGE>(const Stage8& T, int n, int j0) {
            const int key0 = n * kTile + j0;
            if (EDGE && key0 >= w.kv_len) return;
            if (++since > kFlush) flush();
            // lane (g, t): of either 8 keys its column g is key (g / 2) + 4 (g % 2) + 8 b of the step
            uint4 kr[2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
                kr[b] = *reinterpret_cast<const uint4*>(T.k + (j0 + (g >> 1) + 4 * (g & 1) + 8 * b) * HD + 16 * t);
            const uint4 ksc = *reinterpret_cast<const uint4*>(T.ks + j0), vsc = *reinterpret_cast<const uint4*>(T.vs + j0);
            uint2 vr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vr[i] = *reinterpret_cast<const uint2*>(T.v + (j0 + t + 4 * i) * HD + 8 * g);
            float sf[2][4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                sf[b][0] = sf[b][1] = sf[b][2] = sf[b][3] = 0.f;
                const uint32_t u[4] = {kr[b].x, kr[b].y, kr[b].z, kr[b].w};
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    mma_f16(sf[b], qf[ks], codes_f16(__byte_perm(u[ks], 0, 0x4140)), codes_f16(__byte_perm(u[ks], 0, 0x4342)));
            }
            // key i of this lane: t + 4 i, columns 2 t + i % 2 of the 8 keys i / 2
            const uint32_t kb[4] = {ksc.x, ksc.y, ksc.z, ksc.w}, vb[4] = {vsc.x, vsc.y, vsc.z, vsc.w};
            float s[4], ev[4], su[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = (sf[i >> 1][i & 1] + sf[i >> 1][2 + (i & 1)]) * c * __uint_as_float(byte_of(kb[i], t) << 23);
                const uint32_t b = byte_of(vb[i], t);
                ev[i] = b == 255u ? NAN : static_cast<float>(static_cast<int>(b) - 127);
                if (EDGE && key0 + t + 4 * i > pos_r) {
                    s[i] = -INFINITY;
                    ev[i] = 0.f;
                }
                su[i] = s[i] + ev[i];
            }
            float mt = fmax3(fmax3(s[0], s[1], s[2]), s[3], s[3]);
            float mu = fmax3(fmax3(su[0], su[1], su[2]), su[3], su[3]);
            const bool grow = (m == m && !(mt <= m + kMoveThreshold)) || (m2 == m2 && !(mu <= m2 + kMoveThreshold));
            if (__any_sync(0xffffffffu, grow)) {
                mt = fmax3(mt, __shfl_xor_sync(0xffffffffu, mt, 1), -INFINITY);
                mt = fmax3(mt, __shfl_xor_sync(0xffffffffu, mt, 2), -INFINITY);
                mu = fmax3(mu, __shfl_xor_sync(0xffffffffu, mu, 1), -INFINITY);
                mu = fmax3(mu, __shfl_xor_sync(0xffffffffu, mu, 2), -INFINITY);
                if (m == m && !(mt <= m + kMoveThreshold)) {
                    const float to = ceilf(mt);
                    l *= pow2_down(m - to);
                    m = to;
                }
                if (m2 == m2 && !(mu <= m2 + kMoveThreshold)) {
                    const float to = ceilf(mu), f = pow2_down(m2 - to);
                    m2 = to;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[j][e] *= f;
                        sum[j][0] *= f;
                        sum[j][1] *= f;
                    }
                }
            }
            // nothing attended so far: all scores are -inf, and their weights 0
            const float m_use = m == -INFINITY ? 0.f : m, shift = (m_use - (m2 == -INFINITY ? 0.f : m2)) + kWeightBits;
            float wt[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float d = s[i] - m_use;
                l += ex2_sfu(d);
                wt[i] = ex2_sfu(d + (ev[i] + shift));
            }
            uint32_t pf[4];
            two_terms(wt[0], wt[1], pf[0], pf[1]);
            two_terms(wt[2], wt[3], pf[2], pf[3]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {   // 4 of the lane's 8 bytes: dimensions 8 g + 4 h ..
                const uint32_t a = h ? vr[0].y : vr[0].x, b = h ? vr[1].y : vr[1].x;
                const uint32_t cc = h ? vr[2].y : vr[2].x, d = h ? vr[3].y : vr[3].x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t pick = e | ((4 + e) << 8);   // byte e of both, in bytes 0 and 2
                    mma_f16(o[4 * h + e], pf, codes_f16(__byte_perm(a, b, pick)), codes_f16(__byte_perm(cc, d, pick)));
                }
            }
        };
        for (int n = w.t0; n < w.t1; ++n, ++ring) {
            const int st = ring % F8_STAGES;
            wait_or_flag(&S.full[st], (ring / F8_STAGES) & 1, A.err, kErrWaitFull, failed);
            __syncwarp();
            const Stage8& T = S.st[st];
            // the step s of the segment (8 a tile) is key worker s % nkw's
            const int first = (n - w.t0) * (kTile / 16);
            for (int j = (kw + nkw - first % nkw) % nkw; j < kTile / 16; j += nkw) {
                if (w.edge(n)) step.template operator()<true>(T, n, 16 * j);
                else step.template operator()<false>(T, n, 16 * j);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.empty[st]);
        }
        flush();
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) S.ml[warp][g] = make_float2(m, l);
        // with the weights 2^(s - m): the dimensions 16 t + j and 16 t + 8 + j
        const float up = m2 - m - kWeightBits;
        const int e = fabsf(up) < 4096.f ? static_cast<int>(up) : 0;   // 0: nothing attended, or NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            S.o[warp][g][16 * t + j] = ldexpf(sum[j][0], e);
            S.o[warp][g][16 * t + 8 + j] = ldexpf(sum[j][1], e);
        }
    };
    if (seg0 < seg1) load_q(S.work[0]);
    if (warp == F8_WARPS - 1) fetch_work(A, seg0, seg1, S.work, &S.work_full);
    for (int sg = seg0; sg < seg1; ++sg) {
        const Work w = work_of(sg);
        segment(w);
        if (sg + 1 < seg1) load_q(work_of(sg + 1));
        named_bar_sync(1, 32 * F8_WARPS);
        // ---- join the key workers: a row per warp, two columns per lane; lane q has the
        // weight of worker q ----
        const int rgroups = row_groups(w.n_rows), nkw = F8_WARPS / rgroups;
        for (int r = warp; r < w.n_rows; r += F8_WARPS) {
            const int w0 = r >> 3, rr = r & 7;
            const float2 ml = lane < nkw ? S.ml[w0 + lane * rgroups][rr] : make_float2(-INFINITY, 0.f);
            float m_all = ml.x;
#pragma unroll
            for (int d = 1; d < F8_WARPS; d *= 2) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, d));
            const float f = ml.x == -INFINITY ? 0.f : ex2_sfu(ml.x - m_all);
            float l_all = f == 0.f ? 0.f : f * ml.y;
#pragma unroll
            for (int d = 1; d < F8_WARPS; d *= 2) l_all += __shfl_xor_sync(0xffffffffu, l_all, d);
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int q = 0; q < F8_WARPS; ++q) {
                const float fq = __shfl_sync(0xffffffffu, f, q);
                if (q < nkw && fq != 0.f) {
                    const float2 x = *reinterpret_cast<const float2*>(&S.o[w0 + q * rgroups][rr][2 * lane]);
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
        named_bar_sync(1, 32 * F8_WARPS);
    }
}

template <class Act>
cudaError_t launch_few8(const ChunkArgs& a, const Pool8& pool, cudaStream_t stream) {
    constexpr size_t smem = sizeof(Few8Smem);
    static_assert(smem <= 232448, "shared memory of one SM");
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        return cudaFuncSetAttribute(chunk_few8_kernel<Act>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    });
    if (e != cudaSuccess) return e;
    Launch L(dim3(a.n_few_ctas), F8_THREADS, smem, stream);
    return cudaLaunchKernelEx(&L.cfg, chunk_few8_kernel<Act>, a, pool);
}

}  // namespace

cudaError_t launch_chunk_few8(const ChunkArgs& a, const Pool8& pool, bool act_bf16, cudaStream_t stream) {
    return act_bf16 ? launch_few8<__nv_bfloat16>(a, pool, stream) : launch_few8<float>(a, pool, stream);
}

}  // namespace tle
