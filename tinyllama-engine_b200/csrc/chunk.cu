// chunk.cu -- chunks of new tokens over a paged KV cache: append (rope + store)
// and causal attention.
//
// Reference semantics per token: rope() src/ops.cpp:1223-1281, then
// attention() src/ops.cpp:1317-1515 at its position, for a batch of chunks
// (generate.cpp:52-59 feeds a prompt one token at a time).  With f_i the
// frequency of pair i and p the token's position,
//   (x'_2i, x'_2i+1) = (x_2i cos a - x_2i+1 sin a, x_2i sin a + x_2i+1 cos a),  a = fl32(p f_i)
//   out_h(t) = sum_{j <= p} softmax_j(q'_h(t) . k_{h/g}(j) / 8) v_{h/g}(j).
#include <cuda.h>
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "chunk.cuh"
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tle {

namespace {

// ---- append -----------------------------------------------------------------
// A warp takes a token, or an equal part of its n_head + 2 n_head_kv heads
// ("units") where there are few tokens, in 16-byte pieces: 8 (bf16) or 16
// (fp32) lanes per head.  Each lane finds sine and cosine of one of the 32
// pairs and fetches those of its own elements from the lanes that have them,
// once for all units.  HBM-bound: each element is read once and written once;
// kAppendBatch pieces per lane are in flight (fp32: 2048 tokens 7.8 us with 10, 10.6 us
// with 4; bf16: 18 k tokens 33 us with 4, 41 us with 8).  18 k tokens bf16: 160.6 MB
// in 31.7 us, 5.1 TB/s (small blocks leave their places to the next ones soon: 256
// threads 33.0 us); 64 single tokens 3.7 us, the launch and one dependent
// load after another.
constexpr int kAppendThreads = 64;
constexpr int kAppendPart = 4;             // pieces of the smallest part of a token
constexpr int kAppendWarps = 148 * 16;   // below so many tokens their heads are spread over several warps

template <class Act, class Pool>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs A, int parts) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int kAppendBatch = sizeof(Act) == 4 ? 10 : 4;
    constexpr int VE = 16 / sizeof(Act);        // elements of a piece
    constexpr int LPH = HD / VE;                // lanes per head
    constexpr int HPW = 32 / LPH;               // heads per piece of a warp
    const int lane = threadIdx.x & 31;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int64_t tok = w / parts;
    if (tok >= A.n_tokens) return;
    const int part = static_cast<int>(w - tok * parts);
    const int units = A.n_head + 2 * A.n_head_kv, kv0 = A.n_head, v0 = A.n_head + A.n_head_kv;
    const int pieces = (units + HPW - 1) / HPW;
    const int j_end = static_cast<int>(static_cast<int64_t>(part + 1) * pieces / parts);
    // before its records: another plan's descriptor may end before this one's do
    if (A.d.hdr->id != A.plan_id) {
        if (lane == 0) record_error(A.err, kErrBadDesc);
        return;
    }
    const ChunkTok tk = A.d.toks[tok];
    const int d0 = lane % LPH * VE;             // this lane's elements of a head
    const Act* q = static_cast<const Act*>(A.q) + tok * A.q_stride + d0;
    const Act* k = static_cast<const Act*>(A.k) + tok * A.k_stride + d0;
    const Act* v = static_cast<const Act*>(A.v) + tok * A.v_stride + d0;
    Act* qo = static_cast<Act*>(A.q_out) + tok * A.n_head * HD + d0;
    // the token's row in the pools
    Pool* kr = nullptr;
    Pool* vr = nullptr;
    const int id = A.d.seqs[tk.seq].pages[tk.pos >> A.page_shift];
    if (static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages)) {
        const size_t row = (static_cast<size_t>(id) << A.page_shift) | (tk.pos & ((1 << A.page_shift) - 1));
        kr = static_cast<Pool*>(A.key_pool) + row * A.n_head_kv * HD + d0;
        vr = static_cast<Pool*>(A.value_pool) + row * A.n_head_kv * HD + d0;
    } else if (lane == 0) {
        record_error(A.err, kErrBadPage);
    }
    float cs[VE / 2], sn[VE / 2];
    if (A.rotate) {
        float s1, c1;
        sincosf(static_cast<float>(tk.pos) * A.inv_freq[lane], &s1, &c1);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            cs[i] = __shfl_sync(0xffffffffu, c1, d0 / 2 + i);
            sn[i] = __shfl_sync(0xffffffffu, s1, d0 / 2 + i);
        }
    }
    for (int j0 = static_cast<int>(static_cast<int64_t>(part) * pieces / parts); j0 < j_end; j0 += kAppendBatch) {
        uint4 x[kAppendBatch];
#pragma unroll
        for (int b = 0; b < kAppendBatch; ++b) {
            const int u = (j0 + b) * HPW + lane / LPH;
            const Act* src = u < kv0 ? q + u * HD : u < v0 ? k + (u - kv0) * HD : v + (u - v0) * HD;
            x[b] = j0 + b < j_end && u < units ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int b = 0; b < kAppendBatch; ++b) {
            const int u = (j0 + b) * HPW + lane / LPH;
            if (j0 + b >= j_end || u >= units) continue;
            float y[VE];
            if constexpr (sizeof(Act) == 2) {
                bf16x8(x[b], y);
            } else {
                y[0] = __uint_as_float(x[b].x);
                y[1] = __uint_as_float(x[b].y);
                y[2] = __uint_as_float(x[b].z);
                y[3] = __uint_as_float(x[b].w);
            }
            if (A.rotate && u < v0) {
#pragma unroll
                for (int i = 0; i < VE / 2; ++i) {
                    const float a = y[2 * i], c = y[2 * i + 1];
                    y[2 * i] = a * cs[i] - c * sn[i];
                    y[2 * i + 1] = a * sn[i] + c * cs[i];
                }
            }
            if (u < kv0) store_n<VE>(qo + u * HD, y);
            else if (kr) store_n<VE>(u < v0 ? kr + (u - kv0) * HD : vr + (u - v0) * HD, y);
        }
    }
}

// ---- attention ----------------------------------------------------------------
// Flash attention on the tcgen05 tensor cores, straight from the page pools.
//
// Rows and tiles: row t g + h of a (chunk, KV head) is query head h of its
// group for token t, so one K/V tile serves every query that shares it.  An
// item is up to 256 rows; a segment is a range of 128-row K/V tiles of an
// item, and a CTA walks the segments that the plan gave it (ChunkPlanner in
// abi.cu: the batch's tiles cut evenly over the SMs, so ragged batches, long
// contexts with few tokens and whole prompts all fill the GPU).
//
// Two chains per CTA, each a softmax warpgroup with its own scores S, running
// maximum, sum and output O in tensor memory.  In an item of more than 128
// rows ("dual") each chain has a row tile and they share every K/V tile; of a
// smaller item both have the same rows and take its blocks of keys
// alternately, and at the segment's end each joins the two results for half
// of the columns.  A chain goes through its blocks (a tile; with fp32
// activations half of one): S = Q K^T, softmax by one thread per row with a
// lazily moved reference maximum, P into TMEM as the A operand of O += P V.
// The next S is there before this block is done.  A scheduler has two softmax
// warps, so what a warp waits for costs time: barriers are probed ahead of
// their use, and between the scores' load and the first store of P there is
// no branch, so that the compiler can overlap maximum, exponentials, sums and
// packing.
// K and V tiles come by TMA (two 64-row boxes, each inside a page, 128-byte
// swizzle): K is K-major, V is read MN-major, so nothing is transposed or
// copied beforehand.
//
// What bounds it: with 64 columns a score costs 256 tensor-core operations and
// one exponential, and the exponential unit (16 a cycle and SM) is the slower of
// the two: 2048 cycles for 256 x 128 scores; a block takes about 2650 (bf16).
// 2048 tokens behind 30000 rows, 32 query on 4 KV heads: 650 us, 800 TFLOP/s; ncu:
// exponential unit 76 % busy, tensor cores 38 %.  Exponentials by polynomial on
// the FMA units, for a part of the scores: 774 us where this took 669.  Four
// softmax warpgroups of 64 rows, or two blocks of 64 keys in flight per chain:
// 881 to 1340 us where this took 700, for registers.  fp32: 777 tokens behind 16000
// rows 279 us, 374 TFLOP/s of three products each, tensor cores 57 % busy.
//
// Precision: bf16 activations: P rounded to bf16 (its sum is not), fp32
// accumulation.  fp32 activations: q and P are cut into three bf16 numbers of
// 8 bits each whose sum is the 24-bit value exactly, so S and O are 32-bit
// sums of exact products; the cost is three times the MMAs.  The tensor cores
// cut their running sums off instead of rounding them (over 16000 rows O came
// out 3e-5 too small), so with fp32 activations O is summed there over
// kFlushBlocks blocks only and from there on in registers.
//
// Rows beyond what a token attends to: a score is masked by selection, but
// P = 0 does not silence a NaN or infinity in V.  Tiles that hold such rows
// for any row of the item ("edge" tiles, the last one or two) therefore pass
// through one warp first: rows behind the last one are zeroed in shared
// memory, and if a row that only some of the item's tokens attend to is not
// finite, the segment's rows are computed again one by one from global memory
// (chunk_row_exact), which reads nothing but the attended rows.  fp32: so are
// rows that came out NaN, since an infinity in K times a zero term of q is NaN
// where 32-bit arithmetic has a score of -inf.
constexpr int CT_THREADS = 512;
constexpr int kChains = 2;
constexpr int kBox = 64;                     // rows per TMA box: the smallest bf16 page
constexpr int kTileHalfs = kTile * HD;       // elements of a K or V tile (16 KB)
template <bool F32>
constexpr int kKeysOf = F32 ? 64 : 128;      // keys of a block
template <bool F32>
constexpr int kBufsOf = F32 ? 2 : 1;         // S and P buffers of a chain
constexpr int kFlushBlocks = 4;              // fp32: blocks whose PV are summed in tensor memory (48 MMAs)
constexpr int kRegsLaunch = 128;
// fp32: the Q loaders hold more (777 tokens behind 16000 rows: 276 us with 72,
// 291 us with 56, 287 us with 80).
template <bool F32>
constexpr int kRegsControl = F32 ? 72 : 56;
template <bool F32>
constexpr int kRegsSoftmax = 2 * kRegsLaunch - kRegsControl<F32>;
static_assert(CT_THREADS == 512, "two warpgroups of either kind: the split uses the launch's registers up");
template <bool F32>
struct ChunkSmem {
    static constexpr int kStages = F32 ? 3 : 4;     // K/V tiles
    static constexpr int kTerms = F32 ? 3 : 1;      // bf16 terms of q and P
    static constexpr int kQBufs = F32 ? 1 : 2;      // Q buffers (segments in flight)
    uint16_t q[kQBufs][2][kTerms][kTileHalfs];      // 16 KB each, SW128 K-major
    uint16_t k[kStages][kTileHalfs];
    uint16_t v[kStages][kTileHalfs];
    uint4 stage[8][256];                            // a softmax warp's results on their way out
    uint64_t kv_full[kStages];
    uint64_t kv_empty[kStages];                   // the PV issuers and the edge warp
    uint64_t v_ok[kStages];                       // edge tiles: V checked
    uint64_t q_full[2], q_free[2];
    uint64_t scanned[2];                            // the segment's edge tiles are checked
    uint64_t seg_end[2];                            // the softmax is done with the segment
    uint64_t joined, read;                          // smaller items: both results there; both read
    uint64_t s_full[kChains][2], s_free[kChains][2], p_full[kChains][2], p_free[kChains][2];
    int bad[2];                                     // the segment has a non-finite masked V row
    uint32_t tmem_base;
    uint64_t work_full;
    Work work[kWorkCache];                          // the CTA's first segments
};

// TMEM columns (all 512): per chain S 128, P 64 and O 64.  fp32: two buffers
// of 64 keys; the first two terms of P lie on the block's S (whose buffer is
// free again after the PV that reads them), the third where bf16 has P.  At
// the end of a smaller item's segment P's columns hold the row's maximum and sum.
constexpr uint32_t col_s(int c, int h) { return 128u * c + 64u * h; }
constexpr uint32_t col_p(int c, int h) { return 256u + 64u * c + 32u * h; }
constexpr uint32_t col_o(int c) { return 384u + 64u * c; }

constexpr uint32_t kIdO = idesc_bf16_f32(kChunkRows, HD) | (1u << 16);   // B (= V) MN-major

// Shared-memory descriptor of 16 rows of V as an MN-major B operand: rows of
// 128 bytes (the 64 columns of N), 8-row swizzle atoms 1024 bytes apart along K.
__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1024u >> 4) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
           (static_cast<uint64_t>(2u) << 61);
}

__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The upper 16 bits of both numbers (bf16 by truncation), as a pair; and what
// truncation leaves of each, exactly.
__device__ __forceinline__ uint32_t top_pair(float lo, float hi) {
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
__device__ __forceinline__ uint64_t rest_pair(float lo, float hi) {
    const uint64_t top = f2(__uint_as_float(__float_as_uint(lo) & 0xffff0000u), __uint_as_float(__float_as_uint(hi) & 0xffff0000u));
    return ffma2(top, f2(-1.0f, -1.0f), f2(lo, hi));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// A value that all lanes have, in a form that the compiler knows to be uniform
// (a warp reduction's result): what feeds an MMA's descriptors and the loops
// around it must not go through per-lane registers, or every MMA waits for
// half a dozen of them to be moved over.
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }
// wait_or_flag for a converged warp, with uniform branches.
__device__ __forceinline__ void wait_uniform(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code, bool& failed) {
    if (failed || __all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return;
    uint64_t t0 = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return;
        const uint64_t t = globaltimer();
        if (t0 == 0) t0 = t;
        if (__any_sync(0xffffffffu, t - t0 > kWaitTimeoutNs)) break;
    }
    record_error(err, code);
    failed = true;
}

struct ChunkTma {
    CUtensorMap k, v;   // the layer's pools as [pool rows][n_head_kv * 64] bf16, box {64, 64}
};

// Element pointer of a row's head in an array of token rows, moved on from row
// to row without a division: `p` at token t0, head h0 of the group.
template <class T>
struct RowWalk {
    T* p;
    int h;
    int64_t wrap;   // from behind a token's last head of the group to the next one's first
    __device__ __forceinline__ RowWalk(const ChunkArgs& A, T* base, int64_t stride, int first, int kvh, int row) {
        const int t = row_token(A, row);
        h = row - t * A.group;
        p = base + static_cast<int64_t>(first + t) * stride + (kvh * A.group + h) * HD;
        wrap = stride - A.group * HD;
    }
    template <int ROWS>
    __device__ __forceinline__ void step(const ChunkArgs& A) {
        p += ROWS * HD;
        for (h += ROWS; h >= A.group; h -= A.group) p += wrap;
    }
};

// Whether any of 8 bf16 numbers has an exponent of all ones.
__device__ __forceinline__ bool not_finite(const uint4 x) {
    auto full = [](uint32_t u) { return ((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
    return (full(x.x) | full(x.y) | full(x.z) | full(x.w)) != 0;
}

// One row of a segment from global memory, attended rows only: the way taken
// when a masked row of V is not finite, or the row's weights are not (see above).
// About 1.5 us a key (777 tokens behind 16000 rows 25 ms): a segment of more than
// a million keys would outlast the other warps' waits, which is reported.
template <class Act>
__device__ __noinline__ void chunk_row_exact(const ChunkArgs& A, const Work& w, int r, RowOut<Act> dst) {
    const int row = w.row0 + r, tok = row_token(A, row), h = w.kvh * A.group + row - tok * A.group;
    const int pos = w.pos + tok;
    const Act* qp = static_cast<const Act*>(A.q) + static_cast<int64_t>(w.first + tok) * A.q_stride + h * HD;
    float q[HD], o[HD];
    for (int d = 0; d < HD; d += 2) {
        const float2 x = load_pair(qp + d);
        q[d] = x.x * kExpScale;
        q[d + 1] = x.y * kExpScale;
        o[d] = o[d + 1] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const size_t rs = static_cast<size_t>(A.n_head_kv) * HD;
    {
        const int end = min(w.t1 * kTile, pos + 1);
        for (int j = w.t0 * kTile; j < end; ++j) {
            const int id = w.pages[j >> A.page_shift];
            const bool ok = static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages);
            const size_t at = ok ? (static_cast<size_t>(id) << A.page_shift) | (j & ((1 << A.page_shift) - 1)) : 0;
            const uint4* kp = reinterpret_cast<const uint4*>(A.key_pool + at * rs + w.kvh * HD);
            const uint4* vp = reinterpret_cast<const uint4*>(A.value_pool + at * rs + w.kvh * HD);
            float s = 0.f;
            for (int c = 0; c < HD / 8; ++c) {
                float f[8];
                bf16x8(ok ? kp[c] : make_uint4(0, 0, 0, 0), f);
                for (int e = 0; e < 8; ++e) s = fmaf(q[8 * c + e], f[e], s);
            }
            const float mn = s > m || s != s ? s : m;   // keeps a NaN
            if (mn == -INFINITY) continue;              // nothing has a weight so far
            const float al = (m == mn) ? 1.f : exp2f(m - mn);
            const float p = exp2f(s - mn);
            m = mn;
            l = l * al + p;
            for (int c = 0; c < HD / 8; ++c) {
                float f[8];
                bf16x8(ok ? vp[c] : make_uint4(0, 0, 0, 0), f);
                for (int e = 0; e < 8; ++e) o[8 * c + e] = fmaf(o[8 * c + e], al, p * f[e]);
            }
        }
    }
    const float inv = m == -INFINITY ? no_weight(w) : 1.0f / l;
    if (dst.lse) *dst.lse = m == -INFINITY ? -INFINITY : m + log2f(l);
    for (int d = 0; d < HD; d += 8) {
        float x[8];
        for (int e = 0; e < 8; ++e) x[e] = o[d + e] * inv;
        if (dst.out) store8(dst.out + d, x);
        else store8(dst.part + d, x);
    }
}

// A producer warp: the K/V tiles of segments [seg0, seg1) in order into a ring
// of stages; a box (64 rows, within a page) by TMA each.
template <int STAGES, class F>
__device__ __forceinline__ void produce_tiles(const ChunkArgs& A, const ChunkTma& M, int seg0, int seg1, F&& work_of,
                                              uint16_t (*k)[kTileHalfs], uint16_t (*v)[kTileHalfs], uint64_t* full,
                                              uint64_t* empty, bool& failed) {
    const int lane = threadIdx.x & 31;
    const int pool_rows = A.pool_pages << A.page_shift;   // a box from here on is all zeros
    int ring = 0;
    for (int sg = seg0; sg < seg1; ++sg) {
        const Work w = work_of(sg);
        // lane l holds where box b0 + l starts
        int b0 = 2 * w.t0, y = 0;
        auto refill = [&]() {
            const int r = (b0 + lane) * kBox;
            y = pool_rows;
            if (r < w.kv_len && b0 + lane < 2 * w.t1) {
                const int id = w.pages[r >> A.page_shift];
                if (static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages))
                    y = (id << A.page_shift) + (r & ((1 << A.page_shift) - 1));
                else
                    record_error(A.err, kErrBadPage);
            }
        };
        refill();
        for (int n = w.t0; n < w.t1; ++n, ++ring) {
            if (2 * n - b0 >= 32) {
                b0 = 2 * n;
                refill();
            }
            const int st = ring % STAGES;
            const int y0 = __shfl_sync(0xffffffffu, y, 2 * n - b0);
            const int y1 = __shfl_sync(0xffffffffu, y, 2 * n - b0 + 1);
            wait_or_flag(&empty[st], ((ring / STAGES) & 1) ^ 1, A.err, kErrWaitEmpty, failed);
            if (lane == 0 && !failed) {
                mbar_arrive_expect_tx(&full[st], 2 * kTileHalfs * 2);
                tma_load_2d(k[st], &M.k, w.kvh * HD, y0, &full[st]);
                tma_load_2d(k[st] + kBox * HD, &M.k, w.kvh * HD, y1, &full[st]);
                tma_load_2d(v[st], &M.v, w.kvh * HD, y0, &full[st]);
                tma_load_2d(v[st] + kBox * HD, &M.v, w.kvh * HD, y1, &full[st]);
            }
            __syncwarp();
        }
    }
    // no copy may still be in flight when the CTA leaves
    for (int u = ring > STAGES ? ring - STAGES : 0; u < ring && !failed; ++u)
        wait_or_flag(&full[u % STAGES], (u / STAGES) & 1, A.err, kErrDrain, failed);
}

// Warp roles (512 threads, one CTA per SM):
//   warps 0, 1  issue S of chain 0, 1; warps 2, 3 issue PV (apart, so that
//               neither stream waits for the other's operands);
//   warps 4-11  softmax, a warpgroup per chain, one TMEM lane (= row) per thread;
//   warp 12     TMA producer of K/V tiles, all segments in order;
//   warp 13     V of the edge tiles;
//   warps 14-15 Q rows into shared memory (bf16 terms, swizzled).
template <bool F32>
__global__ void __launch_bounds__(CT_THREADS, 1)
    chunk_attn_kernel(const __grid_constant__ ChunkArgs A, const __grid_constant__ ChunkTma M) {
    using Smem = ChunkSmem<F32>;
    using Act = std::conditional_t<F32, float, __nv_bfloat16>;
    constexpr int CT_STAGES = Smem::kStages, kTerms = Smem::kTerms, kQBufs = Smem::kQBufs, kKeys = kKeysOf<F32>, kBufs = kBufsOf<F32>;
    constexpr int kBlocks = kTile / kKeys;   // of a tile
    constexpr uint32_t kIdS = idesc_bf16_f32(kChunkRows, kKeys);
    constexpr int kRegsC = kRegsControl<F32>, kRegsS = kRegsSoftmax<F32>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < CT_STAGES; ++i) {
            mbar_init(&S.kv_full[i], 1);
            mbar_init(&S.kv_empty[i], kChains + 1);
            mbar_init(&S.v_ok[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.q_full[i], 2);          // one arrival per loader warp
            mbar_init(&S.q_free[i], kChains);
            mbar_init(&S.scanned[i], 1);
            mbar_init(&S.seg_end[i], 4 * kChains);   // one per softmax warp
        }
        mbar_init(&S.work_full, 1);
        mbar_init(&S.joined, 4 * kChains);
        mbar_init(&S.read, 4 * kChains);
        for (int c = 0; c < kChains; ++c)
            for (int h = 0; h < 2; ++h) {
                mbar_init(&S.s_full[c][h], 1);
                mbar_init(&S.s_free[c][h], 4);
                mbar_init(&S.p_full[c][h], 4);
                mbar_init(&S.p_free[c][h], 1);
            }
        fence_barrier_init();
        prefetch_tmap(&M.k);
        prefetch_tmap(&M.v);
    }
    if (warp == 0) {
        tmem_alloc(&S.tmem_base, 512);
        tmem_relinquish();
    }
    // everything below reads what earlier kernels on the stream wrote
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid == 0) fetch_first(A, blockIdx.x, &S.work[0]);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int seg0 = S.work[0].seg0, seg1 = S.work[0].seg1;
    const uint32_t tmem = S.tmem_base;
    bool failed = false;
    auto work_of = [&](int i) -> const Work& {
        if (i == seg0 + 1) wait_or_flag(&S.work_full, 0, A.err, kErrWaitFull, failed);
        return i - seg0 < kWorkCache ? S.work[i - seg0] : *static_cast<const Work*>(A.d.segs + i);
    };

    if (wg == 0) {
        regs_dealloc<kRegsC>();
        const int c = uniform(warp & 1);   // the chain
        const uint32_t tm = uniform(tmem);
        int ring = 0, x = 0;   // K/V tiles and own blocks so far
        const int n_seg = uniform(seg1 - seg0);
        const uint32_t k0 = uniform(smem_u32(S.k[0])), v0 = uniform(smem_u32(S.v[0])), q0 = uniform(smem_u32(S.q[0][0][0]));
        if (uniform(warp) < 2) {
            // ------------------------------ S = Q K^T ------------------------------
            for (int k = 0; k < n_seg; ++k) {
                const int b = k % kQBufs;
                const Work w = work_of(seg0 + k);
                const int t0 = uniform(w.t0), t1 = uniform(w.t1), kv_len = uniform(w.kv_len);
                const int dual = uniform(static_cast<int>(w.dual()));
                const uint32_t qa = q0 + (b * 2 + (dual ? c : 0)) * (kTerms * kTileHalfs * 2);
                wait_uniform(&S.q_full[b], (k / kQBufs) & 1, A.err, kErrWaitFull, failed);
                bool any = false;
                for (int n = t0; n < t1; ++n, ++ring) {
                    const int st = ring % CT_STAGES;
                    wait_uniform(&S.kv_full[st], (ring / CT_STAGES) & 1, A.err, kErrWaitFull, failed);
                    for (int u = 0; u < kBlocks && n * kTile + u * kKeys < kv_len; ++u) {
                        if (!dual && (((n - t0) * kBlocks + u) & 1) != c) continue;
                        const int h = x % kBufs;
                        // the buffer: its last scores read (bf16), its last P multiplied (fp32)
                        if (x >= kBufs)
                            wait_uniform(F32 ? &S.p_free[c][h] : &S.s_free[c][h], (x / kBufs - 1) & 1, A.err, kErrWaitMma, failed);
                        tc_fence_after();
                        const uint64_t dk = sw128_desc(k0 + (st * kTileHalfs + u * kKeys * HD) * 2), dq = sw128_desc(qa);
                        const uint32_t tS = tm + col_s(c, h);
                        if (elect_one()) {
#pragma unroll
                            for (int term = kTerms - 1; term >= 0; --term)   // the smallest first
#pragma unroll
                                for (int kk = 0; kk < HD / 16; ++kk)
                                    umma_bf16(tS, dq + term * ((kTileHalfs * 2) >> 4) + 2 * kk, dk + 2 * kk, kIdS,
                                              term < kTerms - 1 || kk > 0);
                            umma_commit(&S.s_full[c][h]);
                        }
                        __syncwarp();
                        ++x;
                        any = true;
                    }
                }
                // Q may be replaced once these MMAs are done
                if (any) {
                    if (elect_one()) umma_commit(&S.q_free[b]);
                } else if (lane == 0) {
                    mbar_arrive(&S.q_free[b]);
                }
                __syncwarp();
            }
        } else {
            // ------------------------------ O += P V -------------------------------
            uint32_t v_par = 0;   // parity of the next v_ok of each stage
            for (int k = 0; k < n_seg; ++k) {
                const Work w = work_of(seg0 + k);
                const int t0 = uniform(w.t0), t1 = uniform(w.t1), kv_len = uniform(w.kv_len), pos_min = uniform(w.pos_min);
                const int dual = uniform(static_cast<int>(w.dual()));
                uint32_t acc = 0;   // the segment's first block overwrites O, fp32: every kFlushBlocks-th
                const int x_first = x;
                for (int n = t0; n < t1; ++n, ++ring) {
                    const int st = ring % CT_STAGES;
                    const bool edge = n * kTile + kTile - 1 > pos_min;
                    const uint32_t par = (v_par >> st) & 1;
                    if (edge) v_par ^= 1u << st;
                    // our blocks of this tile: u0, u0 + du, ..., below u1
                    const int u0 = dual ? 0 : (c + (n - t0) * kBlocks) & 1, du = dual ? 1 : 2;
                    const int u1 = min(kBlocks, (kv_len - n * kTile + kKeys - 1) / kKeys);
                    if (u0 >= u1) {
                        wait_uniform(&S.kv_full[st], (ring / CT_STAGES) & 1, A.err, kErrWaitFull, failed);
                        if (lane == 0) mbar_arrive(&S.kv_empty[st]);
                        __syncwarp();
                        continue;
                    }
                    if (edge) wait_uniform(&S.v_ok[st], par, A.err, kErrWaitFull, failed);
                    for (int u = u0; u < u1; u += du, ++x) {
                        const int h = x % kBufs;
                        if (F32 && (x - x_first) % kFlushBlocks == 0) acc = 0;
                        wait_uniform(&S.p_full[c][h], (x / kBufs) & 1, A.err, kErrWaitMma, failed);
                        tc_fence_after();
                        const uint64_t dv = v_desc(v0 + (st * kTileHalfs + u * kKeys * HD) * 2);
                        const uint32_t tP = tm + col_p(c, h), tS = tm + col_s(c, h), tO = tm + col_o(c);
                        if (elect_one()) {
#pragma unroll
                            for (int term = kTerms - 1; term >= 0; --term) {
                                const uint32_t tp = term == kTerms - 1 ? tP : tS + 32u * term;
#pragma unroll
                                for (int kk = 0; kk < kKeys / 16; ++kk)
                                    umma_bf16_tmem_a(tO, tp + 8 * kk, dv + (2048 >> 4) * kk, kIdO,
                                                     term < kTerms - 1 || kk > 0 ? 1u : acc);
                            }
                            umma_commit(&S.p_free[c][h]);
                            if (u + du >= u1) umma_commit(&S.kv_empty[st]);
                        }
                        __syncwarp();
                        acc = 1;
                    }
                }
            }
            for (int y = max(0, x - kBufs); y < x; ++y)   // MMAs done before TMEM is freed
                wait_uniform(&S.p_free[c][y % kBufs], (y / kBufs) & 1, A.err, kErrDrain, failed);
        }
    } else if (wg == 3) {
        regs_dealloc<kRegsC>();
        if (warp == 12) {
            produce_tiles<CT_STAGES>(A, M, seg0, seg1, work_of, S.k, S.v, S.kv_full, S.kv_empty, failed);
        } else if (warp == 13) {
            // -------------------------- V of the edge tiles ----------------------------
            fetch_work(A, seg0, seg1, S.work, &S.work_full);
            int ring = 0;
            for (int sg = seg0; sg < seg1; ++sg) {
                const int k = sg - seg0;
                const Work w = work_of(sg);
                // the flag was last read by the segment before the last one
                if (k >= 2) wait_or_flag(&S.seg_end[k & 1], ((k - 2) >> 1) & 1, A.err, kErrWaitMma, failed);
                if (lane == 0) S.bad[k & 1] = 0;
                __syncwarp();
                for (int n = w.t0; n < w.t1; ++n, ++ring) {
                    const int st = ring % CT_STAGES;
                    wait_or_flag(&S.kv_full[st], (ring / CT_STAGES) & 1, A.err, kErrWaitFull, failed);
                    if (w.edge(n)) {
                        bool bad = false;
                        const int some = max(0, w.pos_min + 1 - n * kTile);   // from here on not for every row
                        const int none = w.kv_len - n * kTile;                // from here on for none
                        uint4* v = reinterpret_cast<uint4*>(S.v[st]);
                        for (int e = (some & ~3) * 8 + lane; e < kTile * 8; e += 32) {
                            const int jl = e >> 3;
                            if (jl >= none) v[e] = make_uint4(0, 0, 0, 0);
                            else if (jl >= some) {
                                bad |= not_finite(v[e]);
                            }
                        }
                        if (__any_sync(0xffffffffu, bad) && lane == 0) S.bad[k & 1] = 1;
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&S.v_ok[st]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.kv_empty[st]);
                }
                if (lane == 0) mbar_arrive(&S.scanned[k & 1]);
            }
        } else {
            // ------------------------------ Q loaders ----------------------------------
            const int lw = warp - 14;
            for (int sg = seg0; sg < seg1; ++sg) {
                const int k = sg - seg0, b = k % kQBufs;
                const Work w = work_of(sg);
                if (k >= kQBufs) wait_or_flag(&S.q_free[b], ((k / kQBufs) - 1) & 1, A.err, kErrWaitEmpty, failed);
                // 8 lanes per row, 4 rows per step, the warps alternate; rows behind the
                // last one stay as they are: nobody looks at their scores
                const int ch = lane & 7, r0 = 4 * lw + (lane >> 3);
                for (int m = 0; m < (w.dual() ? 2 : 1); ++m) {
                    RowWalk<const Act> at(A, static_cast<const Act*>(A.q) + ch * 8, A.q_stride, w.first, w.kvh,
                                          w.row0 + m * kChunkRows + r0);
                    const int left = w.n_rows - m * kChunkRows - r0;   // steps of 8 rows while below
                    const int off = r0 * HD + ((ch ^ r0) << 3);        // the chunk's place; 8 rows on it is the same
                    const int steps = min(16, (w.n_rows - m * kChunkRows + 7) / 8);
                    if constexpr (!F32) {
#pragma unroll 4
                        for (int j = 0; j < steps; ++j) {
                            if (8 * j < left)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                                 smem_u32(&S.q[b][m][0][off + j * 8 * HD])),
                                             "l"(at.p)
                                             : "memory");
                            at.template step<8>(A);
                        }
                    } else {
#pragma unroll 1
                        for (int j0 = 0; j0 < steps; j0 += 4) {
                            float4 x[4][2];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float4* src = reinterpret_cast<const float4*>(at.p);
                                x[j][0] = x[j][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (8 * (j0 + j) < left) {
                                    x[j][0] = src[0];
                                    x[j][1] = src[1];
                                }
                                at.template step<8>(A);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int at_q = off + (j0 + j) * 8 * HD;
                                float* f = reinterpret_cast<float*>(x[j]);
#pragma unroll
                                for (int term = 0; term < kTerms; ++term) {
                                    *reinterpret_cast<uint4*>(&S.q[b][m][term][at_q]) =
                                        make_uint4(top_pair(f[0], f[1]), top_pair(f[2], f[3]), top_pair(f[4], f[5]),
                                                   top_pair(f[6], f[7]));
#pragma unroll
                                    for (int c = 0; c < 4; ++c) f2_split(rest_pair(f[2 * c], f[2 * c + 1]), f[2 * c], f[2 * c + 1]);
                                }
                            }
                        }
                    }
                }
                if constexpr (!F32) cp_async_wait_all();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.q_full[b]);
            }
        }
    } else {
        // ------------------------------ softmax ------------------------------------
        regs_alloc<kRegsS>();
        const int c = wg - 1;
        const int lr = tid & 127;                      // TMEM lane
        const uint32_t tL = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t tO = tL + col_o(c);
        int x = 0;        // own blocks so far (barrier phases)
        int n_joins = 0;  // segments of smaller items so far
        bool s_ready = false;   // S of block x is there
        auto add_o = [&](auto& sum) {
#pragma unroll
            for (int q = 0; q < HD / 32; ++q) {
                float o[32];
                tmem_ld32(tO + 32 * q, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) sum[32 * q + e] += o[e];
            }
        };
        for (int sg = seg0; sg < seg1; ++sg) {
            const int k = sg - seg0;
            const Work& w = work_of(sg);   // read again where needed: registers are short here
            const bool dual = w.dual();
            const int pos_min = w.pos_min;
            const int r = dual ? kChunkRows * c + lr : lr;   // row of the item
            const int my_pos = w.pos + row_token(A, w.row0 + min(r, w.n_rows - 1));
            float m_ref = -INFINITY;                   // reference maximum, log2 units
            float l_run = 0.f;
            [[maybe_unused]] float o_sum[F32 ? HD : 1];   // O of the blocks before the last flush
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < HD; ++e) o_sum[e] = 0.f;
            }
            const int x0 = x;
            const int key0 = w.t0 * kTile, key_end = min(w.t1 * kTile, w.kv_len);
            // Block x from key on; EDGE: some of its keys are masked for some row.
            auto block = [&]<bool EDGE>(int key) {
                const int h = x % kBufs;
                const uint32_t tS = tL + col_s(c, 0) + 64u * h, tP = tL + col_p(c, 0) + 32u * h;
                if (!s_ready) wait_or_flag(&S.s_full[c][h], (x / kBufs) & 1, A.err, kErrWaitMma, failed);
                __syncwarp();
                tc_fence_after();
                float s[kKeys];
#pragma unroll
                for (int q = 0; q < kKeys / 32; ++q) tmem_ld32(tS + 32 * q, *reinterpret_cast<float(*)[32]>(&s[32 * q]));
                tmem_wait_ld();
                if constexpr (!F32) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.s_free[c][h]);   // the MMA may overwrite S
                }
                if constexpr (EDGE) {
                    const int left = my_pos - key;   // the block's last attended key
#pragma unroll
                    for (int e = 0; e < kKeys; ++e)
                        if (e > left) s[e] = -INFINITY;
                }
                float mc[kKeys / 8];
#pragma unroll
                for (int q = 0; q < kKeys / 8; ++q) {
                    float m = fmax3(s[8 * q], s[8 * q + 1], s[8 * q + 2]);
                    m = fmax3(m, s[8 * q + 3], s[8 * q + 4]);
                    m = fmax3(m, s[8 * q + 5], s[8 * q + 6]);
                    mc[q] = fmax3(m, s[8 * q + 7], m);
                }
                float mt = fmax3(fmax3(mc[0], mc[1], mc[2]), fmax3(mc[3], mc[4], mc[5]), fmax3(mc[6], mc[7], mc[7]));
                if constexpr (kKeys == 128)
                    mt = fmax3(mt, fmax3(fmax3(mc[8], mc[9], mc[10]), mc[11], mc[12]), fmax3(mc[13], mc[14], mc[15]));
                mt *= kExpScale;
                const bool move = m_ref == m_ref && !(mt <= m_ref + kMoveThreshold);   // to a NaN too, never from one
                const float alpha = move ? ex2_sfu(m_ref - mt) : 1.f;                  // 0 from -inf
                m_ref = move ? mt : m_ref;
                const bool any_move = __any_sync(0xffffffffu, move);
                const float m_use = m_ref == -INFINITY ? 0.f : m_ref;   // nothing attended so far: weights 0
                const uint64_t sc2 = f2(kExpScale, kExpScale), negm2 = f2(-m_use, -m_use);
                // probed now, needed further down: the last PV, and the next block's S
                const bool p_done = F32 || x == 0 || mbar_test_wait(&S.p_free[c][0], (x - 1) & 1);
                s_ready = mbar_test_wait(&S.s_full[c][(x + 1) % kBufs], ((x + 1) / kBufs) & 1);
#pragma unroll
                for (int e = 0; e < kKeys / 2; ++e)
                    f2_split(ffma2(f2(s[2 * e], s[2 * e + 1]), sc2, negm2), s[2 * e], s[2 * e + 1]);
#pragma unroll
                for (int e = 0; e < kKeys; ++e) s[e] = ex2_sfu(s[e]);
                uint64_t lsum2[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
                for (int e = 0; e < kKeys / 2; ++e) lsum2[e & 3] = fadd2(lsum2[e & 3], f2(s[2 * e], s[2 * e + 1]));
                float lsum0, lsum1;
                f2_split(fadd2(fadd2(lsum2[0], lsum2[1]), fadd2(lsum2[2], lsum2[3])), lsum0, lsum1);
                l_run = l_run * alpha + (lsum0 + lsum1);
                [[maybe_unused]] uint32_t pk[kKeys / 2];
                if constexpr (!F32) {
#pragma unroll
                    for (int e = 0; e < kKeys / 2; ++e) pk[e] = pack_bf16(s[2 * e], s[2 * e + 1]);
                }
                // P and O may be touched once the last PV is done (fp32: P lies where only
                // an earlier PV could be reading, and S was issued after that)
                if (!p_done) wait_or_flag(&S.p_free[c][0], (x - 1) & 1, A.err, kErrWaitMma, failed);
                __syncwarp();
                if constexpr (F32) {
                    if (x > x0 && (x - x0) % kFlushBlocks == 0) {   // the next PV starts anew
                        wait_or_flag(&S.p_free[c][(x - 1) % kBufs], ((x - 1) / kBufs) & 1, A.err, kErrWaitMma, failed);
                        __syncwarp();
                        tc_fence_after();
                        add_o(o_sum);
                    }
                    if (any_move && x > x0) {
#pragma unroll
                        for (int e = 0; e < HD; ++e) o_sum[e] *= alpha;
                    }
                }
                if (any_move && x > x0 && (!F32 || (x - x0) % kFlushBlocks != 0)) {
                    if (F32) wait_uniform(&S.p_free[c][(x - 1) % kBufs], ((x - 1) / kBufs) & 1, A.err, kErrWaitMma, failed);
                    tc_fence_after();
#pragma unroll
                    for (int q = 0; q < HD / 16; ++q) {
                        float o[16];
                        tmem_ld16(tO + 16 * q, o);
                        tmem_wait_ld();
                        uint32_t ob[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) ob[e] = __float_as_uint(o[e] * alpha);
                        tmem_st16(tO + 16 * q, ob);
                    }
                }
                if constexpr (!F32) {
                    tc_fence_after();
                    tmem_st32(tP, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
                    tmem_st32(tP + 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[32]));
                } else {
#pragma unroll
                    for (int q = 0; q < kKeys / 32; ++q) {   // 32 keys: 16 columns of each term
#pragma unroll
                        for (int term = 0; term < kTerms; ++term) {
                            uint32_t t[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                float& x0 = s[32 * q + 2 * e];
                                float& x1 = s[32 * q + 2 * e + 1];
                                t[e] = top_pair(x0, x1);
                                if (term + 1 < kTerms) f2_split(rest_pair(x0, x1), x0, x1);
                            }
                            tmem_st16((term == kTerms - 1 ? tP : tS + 32 * term) + 16 * q, t);
                        }
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.p_full[c][h]);
                ++x;
            };
            for (int key = key0 + (dual ? 0 : c * kKeys); key < key_end; key += dual ? kKeys : 2 * kKeys) {
                if (key + kKeys - 1 > pos_min) block.template operator()<true>(key);
                else block.template operator()<false>(key);
            }
            // ---- the segment's result ----
            for (int y = max(x0, x - kBufs); y < x; ++y)
                wait_or_flag(&S.p_free[c][y % kBufs], (y / kBufs) & 1, A.err, kErrWaitMma, failed);
            wait_or_flag(&S.scanned[k & 1], (k >> 1) & 1, A.err, kErrWaitMma, failed);
            __syncwarp();
            tc_fence_after();
            if constexpr (F32) {
                if (x - x0 > kFlushBlocks) {   // O whole again, in its place
                    add_o(o_sum);
#pragma unroll
                    for (int q = 0; q < HD / 32; ++q) tmem_st32(tO + 32 * q, *reinterpret_cast<const uint32_t(*)[32]>(&o_sum[32 * q]));
                    tmem_wait_st();
                }
            }
            const bool mine = r < w.n_rows;
            // COLS columns from col0 on of every row of the warp, from one chain or two with
            // weights f0, f1 (a chain without weight may hold anything).  Through shared
            // memory, 16-byte chunk j of row r at j ^ (r & 7), so that the lanes of a store
            // write whole rows.
            uint4* stage = S.stage[4 * c + (warp & 3)];
            const int row_base = (dual ? kChunkRows * c : 0) + 32 * (warp & 3);   // the warp's rows in the item
            auto fetch = [&](float (&o)[32], int col, uint32_t t0, float f0, uint32_t t1, float f1, bool two) {
                tmem_ld32(t0 + col, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = f0 != 0.f ? o[e] * f0 : 0.f;
                if (two) {
                    float y[32];
                    tmem_ld32(t1 + col, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = f1 != 0.f ? fmaf(f1, y[e], o[e]) : o[e];
                }
            };
            // the staged rows, CHUNKS chunks each, to their places
            auto flush = [&]<int CHUNKS, class T>(T* base, int64_t stride) {   // stride 0: partial rows
                constexpr int kRowsPerStep = 32 / CHUNKS;
                __syncwarp();
                const int ch = lane % CHUNKS;
                int rr = lane / CHUNKS;
                RowWalk<T> at(A, base, stride, w.first, w.kvh, w.row0 + row_base + rr);
                if (stride == 0) {
                    at.p = base + static_cast<int64_t>(w.part + row_base + rr) * HD;
                    at.wrap = 0;
                }
#pragma unroll
                for (int q = 0; q < CHUNKS; ++q, rr += kRowsPerStep) {
                    if (row_base + rr < w.n_rows)
                        reinterpret_cast<uint4*>(at.p)[ch] = stage[rr * CHUNKS + (ch ^ (rr & (CHUNKS - 1)))];
                    at.template step<kRowsPerStep>(A);
                }
                __syncwarp();
            };
            auto put = [&]<int COLS>(int col0, uint32_t t0, float f0, uint32_t t1, float f1, bool two) {
                if (F32 || w.part >= 0) {
                    for (int col = col0; col < col0 + COLS; col += 32) {
                        float o[32];
                        fetch(o, col, t0, f0, t1, f1, two);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            stage[lane * 8 + (j ^ (lane & 7))] =
                                make_uint4(__float_as_uint(o[4 * j]), __float_as_uint(o[4 * j + 1]),
                                           __float_as_uint(o[4 * j + 2]), __float_as_uint(o[4 * j + 3]));
                        flush.template operator()<8>(w.part >= 0 ? A.part_o + col : static_cast<float*>(A.out) + col,
                                                     w.part >= 0 ? 0 : A.out_stride);
                    }
                } else {
                    constexpr int kChunks = COLS / 8;
#pragma unroll
                    for (int p = 0; p < COLS / 32; ++p) {
                        float o[32];
                        fetch(o, col0 + 32 * p, t0, f0, t1, f1, two);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            stage[lane * kChunks + ((4 * p + j) ^ (lane & (kChunks - 1)))] =
                                make_uint4(pack_bf16(o[8 * j], o[8 * j + 1]), pack_bf16(o[8 * j + 2], o[8 * j + 3]),
                                           pack_bf16(o[8 * j + 4], o[8 * j + 5]), pack_bf16(o[8 * j + 6], o[8 * j + 7]));
                    }
                    flush.template operator()<kChunks>(static_cast<Act*>(A.out) + col0, A.out_stride);
                }
            };
            float* lse = mine && w.part >= 0 ? A.part_lse + w.part + r : nullptr;
            // fp32: a NaN may come from a zero term of q against an infinity in K
            if (dual) {
                if (S.bad[k & 1] || (F32 && __any_sync(0xffffffffu, mine && l_run != l_run))) {
                    const Work cold = w;   // a copy, so that w itself stays in registers
                    if (mine) chunk_row_exact<Act>(A, cold, r, row_out<Act>(A, cold, r));
                    __syncwarp();
                } else {
                    const bool empty = m_ref == -INFINITY;
                    put.template operator()<HD>(0, tO, empty ? no_weight(w) : 1.0f / l_run, 0u, 0.f, false);
                    if (lse) *lse = empty ? -INFINITY : m_ref + log2f(l_run);
                }
                tc_fence_before();
            } else {
                tmem_st2(tL + col_p(c, 0), m_ref, l_run);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.joined);
                wait_or_flag(&S.joined, n_joins & 1, A.err, kErrWaitMma, failed);
                tc_fence_after();
                float m0, l0, m1, l1;   // the same in both chains
                tmem_ld2(tL + col_p(0, 0), m0, l0);
                tmem_ld2(tL + col_p(1, 0), m1, l1);
                tmem_wait_ld();
                const float m_all = fmaxf(m0, m1);
                const float w0 = m0 != -INFINITY ? exp2f(m0 - m_all) : 0.f, w1 = m1 != -INFINITY ? exp2f(m1 - m_all) : 0.f;
                const float l_all = (w0 != 0.f ? w0 * l0 : 0.f) + (w1 != 0.f ? w1 * l1 : 0.f);
                if (S.bad[k & 1] || (F32 && __any_sync(0xffffffffu, mine && l_all != l_all))) {
                    const Work cold = w;
                    if (mine && c == 0) chunk_row_exact<Act>(A, cold, r, row_out<Act>(A, cold, r));
                    __syncwarp();
                } else {
                    const bool empty = l_all == 0.f;
                    const float inv = empty ? no_weight(w) : 1.0f / l_all;
                    put.template operator()<HD / 2>(32 * c, tL + col_o(0), w0 * inv, tL + col_o(1), w1 * inv, true);
                    if (lse && c == 0) *lse = empty ? -INFINITY : m_all + log2f(l_all);
                }
                // both have read before either's O or P columns are written again
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.read);
                wait_or_flag(&S.read, n_joins & 1, A.err, kErrWaitMma, failed);
                ++n_joins;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.seg_end[k & 1]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- few rows --------------------------------------------------------------------
// Chunks of at most kChunkFewRows rows (decode steps, a few guessed tokens) are
// bound by the K/V bytes, and a 128-row tensor-core tile would be mostly empty:
// here eight warps with 16-row mma.sync tiles (m16n8k16) share a tile, as row
// groups of 16 rows times key groups of 128 / (16 groups) keys, each warp with its own running
// maximum, sum and output in registers; the key groups of a row are joined in
// shared memory at the segment's end.  K and V come through a ring of TMA
// tiles as above, kept full across segments by a producer warp.  Precision
// and the treatment of rows that not every token attends to as above.
// 64 decode steps of 32 query heads: behind 1024 to 2047 rows 25.3 us (fp32; 98.6 MB,
// 3.9 TB/s, of which launch, start and end are 8 us), behind 8000 rows 86.0 us (bf16;
// 525 MB, 6.1 TB/s).  Tiles that every row attends to have code of their own: 0.9 us
// less than with one code for both; two such tiles side by side per warp: 0.6 us more.
constexpr int FW_WARPS = 8;
constexpr int FW_THREADS = 32 * (FW_WARPS + 1);
constexpr int FW_STAGES = 4;       // 64 x 1 behind 2047 rows: 25.8 us, with 3 the same, with 5 28.4 us
constexpr int kFewFlush = 8;        // fp32: tiles (of one row group) whose MMAs are summed in a row
struct FewSmem {
    uint16_t k[FW_STAGES][kTileHalfs];
    uint16_t v[FW_STAGES][kTileHalfs];
    float o[FW_WARPS][16][HD + 4];      // a warp's result, and its rows' maximum and sum
    float2 ml[FW_WARPS][16];
    uint64_t full[FW_STAGES], empty[FW_STAGES], work_full;
    int bad[2];                         // the segment has a non-finite V row that not every row attends to
    Work work[kWorkCache];              // the CTA's first segments
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool F32>
__global__ void __launch_bounds__(FW_THREADS, 1)
    chunk_few_kernel(const __grid_constant__ ChunkArgs A, const __grid_constant__ ChunkTma M) {
    using Act = std::conditional_t<F32, float, __nv_bfloat16>;
    constexpr int kTerms = F32 ? 3 : 1;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    FewSmem& S = *reinterpret_cast<FewSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < FW_STAGES; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], FW_WARPS);
        }
        mbar_init(&S.work_full, 1);
        S.bad[0] = S.bad[1] = 0;
        fence_barrier_init();
        prefetch_tmap(&M.k);
        prefetch_tmap(&M.v);
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
    if (warp == FW_WARPS) {
        produce_tiles<FW_STAGES>(A, M, seg0, seg1, work_of, S.k, S.v, S.full, S.empty, failed);
        return;
    }
    const int gid = lane >> 2, tg = lane & 3;     // fragment row and column pair
    const int mi = lane >> 3, li = lane & 7;      // ldmatrix: matrix and row of this lane's address
    static_assert(kChunkFewRows <= 32, "two row groups at most");
    auto row_groups = [](int n_rows) { return n_rows <= 16 ? 1 : 2; };
    // This lane's rows gid and gid + 8 of the row group, two columns of each 8:
    // loaded ahead of the segment that needs them.
    using Raw = std::conditional_t<F32, float2, uint32_t>;
    Raw raw[2][HD / 8];
    auto load_q = [&](const Work& w) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = warp % row_groups(w.n_rows) * 16 + gid + 8 * e;
            const bool ok = r < w.n_rows;
            const int row = w.row0 + (ok ? r : 0), t = row_token(A, row), h = row - t * A.group;
            const Raw* src = reinterpret_cast<const Raw*>(static_cast<const Act*>(A.q) +
                                                          static_cast<int64_t>(w.first + t) * A.q_stride +
                                                          (w.kvh * A.group + h) * HD) + tg;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) raw[e][i] = ok ? src[4 * i] : Raw{};
        }
    };
    int ring = 0;
    // The tiles of one segment; leaves the warp's maxima, sums and outputs in S.
    // HALF (at most 8 rows): with fp32 the upper 8 rows of the A fragments hold the
    // second term of the same rows, so two MMAs do for three terms.
    auto segment = [&]<bool HALF>(const Work& w, int k) {
        constexpr int kRows = HALF ? 1 : 2;       // rows of a lane: gid (, gid + 8)
        constexpr int kFrags = !F32 ? 1 : HALF ? 2 : 3;
        const int rgroups = row_groups(w.n_rows);
        const int keys = 16 * rgroups;            // of a tile, per warp
        const int rg = warp % rgroups, kg = warp / rgroups;
        int pos_r[kRows];
        uint32_t qf[kFrags][HD / 16][4];          // A fragments of Q
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) qf[f][ks][0] = qf[f][ks][1] = qf[f][ks][2] = qf[f][ks][3] = 0u;
#pragma unroll
        for (int e = 0; e < kRows; ++e) {
            pos_r[e] = w.pos + row_token(A, w.row0 + min(rg * 16 + gid + 8 * e, w.n_rows - 1));
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                if constexpr (F32) {
                    float2 x = raw[e][i];
#pragma unroll
                    for (int term = 0; term < kTerms; ++term) {
                        if (HALF) qf[term >> 1][i >> 1][2 * (i & 1) + (term & 1)] = top_pair(x.x, x.y);
                        else qf[term][i >> 1][2 * (i & 1) + e] = top_pair(x.x, x.y);
                        f2_split(rest_pair(x.x, x.y), x.x, x.y);
                    }
                } else {
                    qf[0][i >> 1][2 * (i & 1) + e] = raw[e][i];
                }
            }
        }
        float m_ref[kRows], l_run[kRows];
#pragma unroll
        for (int e = 0; e < kRows; ++e) {
            m_ref[e] = -INFINITY;
            l_run[e] = 0.f;
        }
        float o[HD / 8][4];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        // fp32: o is summed by MMAs over kFewFlush tiles only and from there on in S
        // (the tensor cores cut their sums off)
        int since = 0;
        bool flushed = false;
        auto held = [&](int e, int i) -> float2& {
            return *reinterpret_cast<float2*>(&S.o[warp][gid + 8 * e][8 * i + 2 * tg]);
        };
        auto flush = [&]() {
#pragma unroll
            for (int e = 0; e < kRows; ++e)
#pragma unroll
                for (int i = 0; i < HD / 8; ++i) {
                    float2 y = HALF ? make_float2(o[i][0] + o[i][2], o[i][1] + o[i][3]) : make_float2(o[i][2 * e], o[i][2 * e + 1]);
                    if (flushed) y = make_float2(held(e, i).x + y.x, held(e, i).y + y.y);
                    held(e, i) = y;
                }
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            flushed = true;
            since = 0;
        };
        // Tile n; EDGE: some row does not attend to all of it.
        auto tile = [&]<bool EDGE>(int n) {
            if (F32 && ++since > kFewFlush / rgroups) flush();
            const int st = ring % FW_STAGES;
            wait_or_flag(&S.full[st], (ring / FW_STAGES) & 1, A.err, kErrWaitFull, failed);
            __syncwarp();
            const uint32_t kb = smem_u32(S.k[st]), vb = smem_u32(S.v[st]);
            for (int j0 = kg * keys; j0 < (kg + 1) * keys; j0 += 16) {   // 16 keys
                const int key0 = n * kTile + j0;
                if (EDGE && key0 >= w.kv_len) break;
                if constexpr (EDGE) {
                    // V rows behind the last one: zero; rows only some attend to: finite?
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int jl = 4 * e + (lane >> 3), key = key0 + jl;
                        uint4* p = reinterpret_cast<uint4*>(S.v[st] + (j0 + jl) * HD) + (lane & 7);
                        if (key >= w.kv_len) *p = make_uint4(0, 0, 0, 0);
                        else if (key > w.pos_min) bad |= not_finite(*p);
                    }
                    if (__any_sync(0xffffffffu, bad) && lane == 0) S.bad[k & 1] = 1;
                    __syncwarp();
                }
                // S: one accumulator per fragment and 8 keys, so that the MMAs of a
                // fragment only wait for each other
                float sf[kFrags][2][4];
#pragma unroll
                for (int f = 0; f < kFrags; ++f)
#pragma unroll
                    for (int b = 0; b < 2; ++b) sf[f][b][0] = sf[f][b][1] = sf[f][b][2] = sf[f][b][3] = 0.f;
                uint32_t kf[HD / 16][4];
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const int r = j0 + li + 8 * (mi >> 1), ch = 2 * ks + (mi & 1);
                    ldsm4(kb + r * (HD * 2) + ((ch ^ (r & 7)) << 4), kf[ks]);
                }
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                    for (int f = 0; f < kFrags; ++f) {
                        mma16816(sf[f][0], qf[f][ks], kf[ks][0], kf[ks][1]);
                        mma16816(sf[f][1], qf[f][ks], kf[ks][2], kf[ks][3]);
                    }
                uint32_t vf[HD / 16][4];
#pragma unroll
                for (int dp = 0; dp < HD / 16; ++dp) {
                    const int r = j0 + li + 8 * (mi & 1), ch = 2 * dp + (mi >> 1);
                    ldsm4_t(vb + r * (HD * 2) + ((ch ^ (r & 7)) << 4), vf[dp]);
                }
                float s[kRows][4];   // row, keys key0 + 2 tg (+1), key0 + 8 + 2 tg (+1)
                float mt[kRows];
                bool grow = false;   // m_ref is the same in the four lanes of a row
#pragma unroll
                for (int e = 0; e < kRows; ++e) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int b = q >> 1, i = 2 * e + (q & 1);
                        if (!F32) s[e][q] = sf[0][b][i];
                        else if (HALF) s[e][q] = sf[0][b][i] + (sf[0][b][i + 2] + sf[kFrags - 1][b][i]);
                        else s[e][q] = sf[0][b][i] + (sf[kFrags > 1 ? 1 : 0][b][i] + sf[kFrags - 1][b][i]);
                        if (EDGE && key0 + 8 * b + 2 * tg + (q & 1) > pos_r[e]) s[e][q] = -INFINITY;
                    }
                    mt[e] = fmax3(fmax3(s[e][0], s[e][1], s[e][2]), s[e][3], s[e][3]) * kExpScale;
                    grow |= m_ref[e] == m_ref[e] && !(mt[e] <= m_ref[e] + kMoveThreshold);
                }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int e = 0; e < kRows; ++e) {
                        float m = fmax3(mt[e], __shfl_xor_sync(0xffffffffu, mt[e], 1), -INFINITY);
                        m = fmax3(m, __shfl_xor_sync(0xffffffffu, m, 2), -INFINITY);
                        if (m_ref[e] == m_ref[e] && !(m <= m_ref[e] + kMoveThreshold)) {
                            const float alpha = ex2_sfu(m_ref[e] - m);   // 0 from -inf
                            m_ref[e] = m;
                            l_run[e] *= alpha;
#pragma unroll
                            for (int i = 0; i < HD / 8; ++i) {
                                o[i][2 * e] *= alpha;
                                o[i][2 * e + 1] *= alpha;
                                if (HALF) {
                                    o[i][2] *= alpha;
                                    o[i][3] *= alpha;
                                }
                                if (F32 && flushed) held(e, i) = make_float2(held(e, i).x * alpha, held(e, i).y * alpha);
                            }
                        }
                    }
                }
                uint32_t pf[kFrags][4];   // A fragments of P: keys 2 tg (+1), then + 8
#pragma unroll
                for (int f = 0; f < kFrags; ++f) pf[f][0] = pf[f][1] = pf[f][2] = pf[f][3] = 0u;
#pragma unroll
                for (int e = 0; e < kRows; ++e) {
                    const float m_use = m_ref[e] == -INFINITY ? 0.f : m_ref[e];
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[e][q] = ex2_sfu(fmaf(s[e][q], kExpScale, -m_use));
                    l_run[e] += (s[e][0] + s[e][1]) + (s[e][2] + s[e][3]);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        float x0 = s[e][2 * b], x1 = s[e][2 * b + 1];
                        if constexpr (F32) {
#pragma unroll
                            for (int term = 0; term < kTerms; ++term) {
                                if (HALF) pf[term >> 1][2 * b + (term & 1)] = top_pair(x0, x1);
                                else pf[term][2 * b + e] = top_pair(x0, x1);
                                f2_split(rest_pair(x0, x1), x0, x1);
                            }
                        } else {
                            pf[0][2 * b + e] = pack_bf16(x0, x1);
                        }
                    }
                }
#pragma unroll
                for (int f = kFrags - 1; f >= 0; --f)
#pragma unroll
                    for (int dp = 0; dp < HD / 16; ++dp) {
                        mma16816(o[2 * dp], pf[f], vf[dp][0], vf[dp][1]);
                        mma16816(o[2 * dp + 1], pf[f], vf[dp][2], vf[dp][3]);
                    }
            }
            if (EDGE) fence_proxy_async_smem();   // zeroed rows: before the stage's next TMA load
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.empty[st]);
        };
        for (int n = w.t0; n < w.t1; ++n, ++ring) {
            if (w.edge(n)) tile.template operator()<true>(n);
            else tile.template operator()<false>(n);
        }
#pragma unroll
        for (int e = 0; e < kRows; ++e) {
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
            if (tg == 0) S.ml[warp][gid + 8 * e] = make_float2(m_ref[e], l_run[e]);
            // fp32: a NaN may come from a zero term of q against an infinity in K
            if (F32 && rg * 16 + gid + 8 * e < w.n_rows && l_run[e] != l_run[e]) S.bad[k & 1] = 1;
        }
        flush();
    };
    if (seg0 < seg1) load_q(S.work[0]);
    if (warp == FW_WARPS - 1) fetch_work(A, seg0, seg1, S.work, &S.work_full);
    for (int sg = seg0; sg < seg1; ++sg) {
        const int k = sg - seg0;
        const Work w = work_of(sg);
        const int rgroups = row_groups(w.n_rows);
        if (w.n_rows <= 8) segment.template operator()<true>(w, k);
        else segment.template operator()<false>(w, k);
        // ---- join the key groups ----
        if (sg + 1 < seg1) load_q(work_of(sg + 1));
        named_bar_sync(1, 32 * FW_WARPS);
        if (tid == 0) S.bad[(k + 1) & 1] = 0;   // of the next segment: nobody is there before the barrier below
        if (S.bad[k & 1]) {
            const Work cold = w;
            if (tid < w.n_rows) chunk_row_exact<Act>(A, cold, tid, row_out<Act>(A, cold, tid));
        } else {
            // a row per warp, two columns per lane; lane q has the weight of key group q
            const int kgroups = FW_WARPS / rgroups;
            for (int r = warp; r < w.n_rows; r += FW_WARPS) {
                const int w0 = r >> 4, rr = r & 15;
                const float2 ml = lane < kgroups ? S.ml[w0 + lane * rgroups][rr] : make_float2(-INFINITY, 0.f);
                float m_all = ml.x;
#pragma unroll
                for (int d = 1; d < FW_WARPS; d *= 2) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, d));
                const float f = ml.x == -INFINITY ? 0.f : ex2_sfu(ml.x - m_all);
                float l_all = f == 0.f ? 0.f : f * ml.y;
#pragma unroll
                for (int d = 1; d < FW_WARPS; d *= 2) l_all += __shfl_xor_sync(0xffffffffu, l_all, d);
                float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < FW_WARPS; ++q) {
                    const float fq = __shfl_sync(0xffffffffu, f, q);
                    if (q < kgroups) {
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
        }
        named_bar_sync(1, 32 * FW_WARPS);
    }
}

// Items in several partial blocks: out = sum_b w_b o_b / sum_b w_b, w_b =
// 2^(lse_b - max), in block order.  A warp per row, lane = two columns.  About
// 2.5 us with its launch, which is why the plan cuts items only where that pays.
constexpr int kMergeThreads = 256;
template <class Act>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const __grid_constant__ ChunkArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    if (A.d.hdr->id != A.plan_id) {
        if (threadIdx.x == 0) record_error(A.err, kErrBadDesc);
        return;
    }
    const ChunkMerge m = A.d.merges[blockIdx.x];
    const int r = blockIdx.y * (kMergeThreads / 32) + (threadIdx.x >> 5);
    if (r >= m.n_rows) return;
    const float* lse = A.part_lse + m.part + r;
    const float* po = A.part_o + (static_cast<size_t>(m.part) + r) * HD + 2 * lane;
    // four blocks at a time, all of their loads in flight
    float2 acc = make_float2(0.f, 0.f);
    float mx = -INFINITY, sum = 0.f;
    for (int b0 = 0; b0 < m.n_parts; b0 += 4) {
        float l[4];
        float2 x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const bool in = b0 + b < m.n_parts;
            const size_t at = static_cast<size_t>(in ? b0 + b : b0) * m.n_rows;
            l[b] = in ? lse[at] : -INFINITY;
            x[b] = *reinterpret_cast<const float2*>(po + at * HD);
        }
        const float top = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), mx);
        const float keep = mx == -INFINITY ? 0.f : exp2f(mx - top);
        sum *= keep;
        acc.x *= keep;
        acc.y *= keep;
        mx = top;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float w = l[b] == -INFINITY ? 0.f : exp2f(l[b] - mx);
            sum += w;
            acc.x = fmaf(w, x[b].x, acc.x);
            acc.y = fmaf(w, x[b].y, acc.y);
        }
    }
    const ChunkSeq sq = A.d.seqs[m.seq];
    const int row = m.row0 + r, t = row_token(A, row), h = row - t * A.group;
    const float inv = 1.0f / sum;
    Act* out = static_cast<Act*>(A.out) + static_cast<int64_t>(sq.first + t) * A.out_stride +
               (m.kvh * A.group + h) * HD + 2 * lane;
    store_pair(out, make_float2(acc.x * inv, acc.y * inv));
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, bool act_bf16, bool pool_bf16, cudaStream_t stream) {
    // a warp per token, or parts of one where that leaves SMs without work: at
    // least kAppendPart pieces each (64 tokens of 40 fp32 heads: 3.2 us in five
    // parts, 3.7 us in two)
    const int per_piece = act_bf16 ? 4 : 2;   // heads
    const int pieces = (a.n_head + 2 * a.n_head_kv + per_piece - 1) / per_piece;
    const int most = (pieces + kAppendPart - 1) / kAppendPart;
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, kAppendWarps / a.n_tokens)));
    const int64_t warps = static_cast<int64_t>(a.n_tokens) * parts;
    const int64_t blocks = (warps * 32 + kAppendThreads - 1) / kAppendThreads;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    Launch L(dim3(static_cast<unsigned>(blocks)), kAppendThreads, 0, stream);
    if (act_bf16)
        return pool_bf16 ? cudaLaunchKernelEx(&L.cfg, append_kernel<__nv_bfloat16, __nv_bfloat16>, a, parts)
                         : cudaLaunchKernelEx(&L.cfg, append_kernel<__nv_bfloat16, float>, a, parts);
    return pool_bf16 ? cudaLaunchKernelEx(&L.cfg, append_kernel<float, __nv_bfloat16>, a, parts)
                     : cudaLaunchKernelEx(&L.cfg, append_kernel<float, float>, a, parts);
}

template <bool F32>
cudaError_t launch_chunk_attn(const ChunkArgs& a, const ChunkTma& m, cudaStream_t stream) {
    constexpr size_t smem = sizeof(ChunkSmem<F32>) + 1024;
    static_assert(smem <= 232448, "shared memory of one SM");
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        // setmaxnreg.inc draws on the registers of the launch: refuse instead
        // of waiting forever if the kernel was compiled with fewer
        cudaFuncAttributes fa{};
        cudaError_t r = cudaFuncGetAttributes(&fa, chunk_attn_kernel<F32>);
        if (r != cudaSuccess) return r;
        if (fa.numRegs < kRegsLaunch) return cudaErrorInvalidConfiguration;
        return cudaFuncSetAttribute(chunk_attn_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(smem));
    });
    if (e != cudaSuccess) return e;
    Launch L(dim3(a.n_ctas), CT_THREADS, smem, stream);
    return cudaLaunchKernelEx(&L.cfg, chunk_attn_kernel<F32>, a, m);
}

template <bool F32>
cudaError_t launch_chunk_few(const ChunkArgs& a, const ChunkTma& m, cudaStream_t stream) {
    constexpr size_t smem = sizeof(FewSmem) + 1024;
    static_assert(smem <= 232448, "shared memory of one SM");
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        return cudaFuncSetAttribute(chunk_few_kernel<F32>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    });
    if (e != cudaSuccess) return e;
    Launch L(dim3(a.n_few_ctas), FW_THREADS, smem, stream);
    return cudaLaunchKernelEx(&L.cfg, chunk_few_kernel<F32>, a, m);
}

static cudaError_t chunk_maps(const ChunkArgs& a, ChunkTma* m) {
    const uint64_t cols = static_cast<uint64_t>(a.n_head_kv) * HD, rows = static_cast<uint64_t>(a.pool_pages) << a.page_shift;
    cudaError_t e = make_tmap_16b(&m->k, const_cast<uint16_t*>(a.key_pool), cols, rows, kBox, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    if (e != cudaSuccess) return e;
    return make_tmap_16b(&m->v, const_cast<uint16_t*>(a.value_pool), cols, rows, kBox, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

cudaError_t launch_chunk_merge(const ChunkArgs& a, bool act_bf16, cudaStream_t stream) {
    if (a.n_merge == 0) return cudaSuccess;
    constexpr int warps = kMergeThreads / 32;
    Launch L(dim3(a.n_merge, (a.merge_rows + warps - 1) / warps), kMergeThreads, 0, stream);
    return act_bf16 ? cudaLaunchKernelEx(&L.cfg, chunk_merge_kernel<__nv_bfloat16>, a)
                    : cudaLaunchKernelEx(&L.cfg, chunk_merge_kernel<float>, a);
}

cudaError_t launch_chunk_many(const ChunkArgs& a, bool act_bf16, cudaStream_t stream) {
    ChunkTma m;
    cudaError_t e = chunk_maps(a, &m);
    if (e != cudaSuccess) return e;
    return act_bf16 ? launch_chunk_attn<false>(a, m, stream) : launch_chunk_attn<true>(a, m, stream);
}

cudaError_t launch_chunk_attention(const ChunkArgs& a, bool act_bf16, cudaStream_t stream) {
    ChunkTma m;
    cudaError_t e = chunk_maps(a, &m);
    if (e != cudaSuccess) return e;
    if (a.n_few_ctas > 0) {
        e = act_bf16 ? launch_chunk_few<false>(a, m, stream) : launch_chunk_few<true>(a, m, stream);
        if (e != cudaSuccess) return e;
    }
    if (a.n_ctas > 0) {
        e = act_bf16 ? launch_chunk_attn<false>(a, m, stream) : launch_chunk_attn<true>(a, m, stream);
        if (e != cudaSuccess) return e;
    }
    return launch_chunk_merge(a, act_bf16, stream);
}

}  // namespace tle
