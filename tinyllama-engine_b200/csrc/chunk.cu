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

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace tle {

namespace {

constexpr int HD = kHeadDim;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kScale = 0.125f;   // 1/sqrt(64)

__device__ __forceinline__ float2 load_pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load_pair(const __nv_bfloat16* p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
}
__device__ __forceinline__ void store_pair(float* p, float2 x) { *reinterpret_cast<float2*>(p) = x; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float2 x) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x.x, x.y);
}

// ---- append -----------------------------------------------------------------
// A warp takes kUnitsPerWarp of the n_head + 2 n_head_kv heads ("units") of a
// token, lane = rotation pair, so one sincosf serves them all; every load is
// issued before the first store.  HBM/latency-bound: each element is read
// once and written once.
constexpr int kAppendThreads = 256;
constexpr int kUnitsPerWarp = 8;

template <class Act, class Pool>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int units = A.n_head + 2 * A.n_head_kv;
    const int per_token = (units + kUnitsPerWarp - 1) / kUnitsPerWarp;
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int64_t tok = w / per_token;
    if (tok >= A.n_tokens) return;
    const int u0 = static_cast<int>(w - tok * per_token) * kUnitsPerWarp;
    const ChunkTok tk = A.d.toks[tok];
    const Act* q = static_cast<const Act*>(A.q) + tok * A.q_stride + 2 * lane;
    const Act* k = static_cast<const Act*>(A.k) + tok * A.k_stride + 2 * lane;
    const Act* v = static_cast<const Act*>(A.v) + tok * A.v_stride + 2 * lane;
    const int kv0 = A.n_head, v0 = A.n_head + A.n_head_kv;   // first k and v unit
    float2 x[kUnitsPerWarp];
#pragma unroll
    for (int j = 0; j < kUnitsPerWarp; ++j) {
        const int u = u0 + j;
        x[j] = make_float2(0.f, 0.f);
        if (u < kv0) x[j] = load_pair(q + u * HD);
        else if (u < v0) x[j] = load_pair(k + (u - kv0) * HD);
        else if (u < units) x[j] = load_pair(v + (u - v0) * HD);
    }
    // the token's row in the pools (only the warps with k or v units need it)
    Pool* kr = nullptr;
    Pool* vr = nullptr;
    if (u0 + kUnitsPerWarp > kv0) {
        const ChunkSeq s = A.d.seqs[tk.seq];
        const int id = s.pages[tk.pos >> A.page_shift];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages)) {
            const size_t row = (static_cast<size_t>(id) << A.page_shift) | (tk.pos & ((1 << A.page_shift) - 1));
            kr = static_cast<Pool*>(A.key_pool) + row * A.n_head_kv * HD + 2 * lane;
            vr = static_cast<Pool*>(A.value_pool) + row * A.n_head_kv * HD + 2 * lane;
        } else {
            record_error(A.err, kErrBadPage);
        }
    }
    float sn = 0.f, cs = 1.f;
    if (A.rotate) sincosf(static_cast<float>(tk.pos) * A.inv_freq[lane], &sn, &cs);
    Act* qo = static_cast<Act*>(A.q_out) + tok * A.n_head * HD + 2 * lane;
#pragma unroll
    for (int j = 0; j < kUnitsPerWarp; ++j) {
        const int u = u0 + j;
        const float2 y = A.rotate ? make_float2(x[j].x * cs - x[j].y * sn, x[j].x * sn + x[j].y * cs) : x[j];
        if (u < kv0) store_pair(qo + u * HD, y);
        else if (u < v0) {
            if (kr) store_pair(kr + (u - kv0) * HD, y);
        } else if (u < units) {
            if (vr) store_pair(vr + (u - v0) * HD, x[j]);
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
// contexts with few tokens and whole prompts all fill the GPU).  An item of
// more than 128 rows ("dual") has its two row tiles in the two softmax
// warpgroups, which share each K/V tile; a smaller one has the same rows in
// both, and they take the tiles alternately, so the tensor cores and the
// exponentials of two tiles are in flight either way.
//
// Per tile (M = 128 rows, N = 128 keys): S = Q K^T into TMEM, softmax by one
// thread per row with a lazily moved reference maximum, P back into TMEM as
// the A operand of O += P V.  K and V tiles come by TMA (two 64-row boxes,
// each inside a page, 128-byte swizzle): K is K-major, V is read MN-major, so
// nothing is transposed or copied beforehand.
//
// Precision: bf16 activations: P rounded to bf16 (its sum is not), fp32
// accumulation.  fp32 activations: q and P are cut into three bf16 numbers of
// 8 bits each whose sum is the 24-bit value exactly, so S and O are 32-bit
// sums of exact products; the cost is three times the MMAs.
//
// Rows beyond what a token attends to: a score is masked by selection, but
// P = 0 does not silence a NaN or infinity in V.  Tiles that hold such rows
// for any row of the item ("edge" tiles, the last one or two) therefore pass
// through warp 3 first: rows behind the last one are zeroed in shared memory,
// and if a row that only some of the item's tokens attend to is not finite,
// the segment's rows are computed again one by one from global memory
// (chunk_row_exact), which reads nothing but the attended rows.
constexpr int CT_THREADS = 512;
constexpr int CT_STAGES = 4;
constexpr int kTile = kChunkTile;            // 128
constexpr int kBox = 64;                     // rows per TMA box: the smallest bf16 page
constexpr int kTileHalfs = kTile * HD;       // elements of a K or V tile (16 KB)
constexpr int kRegsControl = 56, kRegsLoader = 56, kRegsSoftmax = 200, kRegsLaunch = 128;
static_assert(128 * (kRegsControl + kRegsLoader) + 256 * kRegsSoftmax <= CT_THREADS * kRegsLaunch,
              "setmaxnreg split exceeds the launch register budget");
constexpr float kExpScale = kScale * kLog2e;
// The reference maximum moves only when the row's maximum grows by more than
// 8 (log2 units), so O is rescaled rarely; P <= 2^8.
constexpr float kMoveThreshold = 8.0f;

// A segment as the kernel's roles see it.
struct Work {
    const int32_t* pages;
    int kvh, row0, n_rows, t0, t1, part;
    int pos, first;
    int pos_min, kv_len;   // position of the item's first token; rows of its last token
    bool dual;
    __device__ __forceinline__ bool edge(int n) const { return n * kTile + kTile - 1 > pos_min; }
};
__device__ __forceinline__ Work work_at(const ChunkArgs& A, int i) {
    const ChunkSeg sg = A.d.segs[i];
    const ChunkSeq sq = A.d.seqs[sg.seq];
    Work w;
    w.pages = sq.pages;
    w.kvh = sg.kvh;
    w.row0 = sg.row0;
    w.n_rows = sg.n_rows;
    w.t0 = sg.t0;
    w.t1 = sg.t1;
    w.part = sg.part;
    w.pos = sq.pos;
    w.first = sq.first;
    const int g = A.group;
    w.pos_min = sq.pos + sg.row0 / g;
    w.kv_len = sq.pos + (sg.row0 + sg.n_rows - 1) / g + 1;
    w.dual = sg.n_rows > kChunkRows;
    return w;
}

constexpr int kWorkCache = 20;

template <bool F32>
struct ChunkSmem {
    static constexpr int kTerms = F32 ? 3 : 1;      // bf16 terms of q and P
    static constexpr int kQBufs = F32 ? 1 : 2;      // Q buffers (segments in flight)
    uint16_t q[kQBufs][2][kTerms][kTileHalfs];      // 16 KB each, SW128 K-major
    uint16_t k[CT_STAGES][kTileHalfs];
    uint16_t v[CT_STAGES][kTileHalfs];
    uint64_t kv_full[CT_STAGES];
    uint64_t kv_empty[CT_STAGES];                   // both MMA warps and warp 3
    uint64_t v_ok[CT_STAGES];                       // edge tiles: V checked by warp 3
    uint64_t q_full[2];
    uint64_t q_free[2];                             // both MMA warps' last S and the 8 softmax warps
    uint64_t scanned[2];                            // warp 3 is done with a segment's edge tiles
    uint64_t s_full[2], s_free[2], p_full[2], p_free[2];
    int bad[2];                                     // the segment has a non-finite masked V row
    Work work[kWorkCache];                          // the CTA's first segments
    uint32_t tmem_base;
};

// TMEM columns (all 512).  bf16: S 128, P 64 and O 64 per warpgroup.  fp32:
// the first two terms of P lie on S (read before they are written, and the
// next S waits for the PV that reads them), the third beside it.
constexpr uint32_t col_s(int i) { return 128u * i; }
constexpr uint32_t col_p(int i) { return 256u + 64u * i; }
constexpr uint32_t col_o(int i) { return 384u + 64u * i; }

constexpr uint32_t kIdS = idesc_bf16_f32(kChunkRows, kTile);
constexpr uint32_t kIdO = idesc_bf16_f32(kChunkRows, HD) | (1u << 16);   // B (= V) MN-major

// Shared-memory descriptor of 16 rows of V as an MN-major B operand: rows of
// 128 bytes (the 64 columns of N), 8-row swizzle atoms 1024 bytes apart along K.
__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1024u >> 4) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
           (static_cast<uint64_t>(2u) << 61);
}

__device__ __forceinline__ float ex2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// Maxima that keep a NaN: a NaN score poisons its row's reference maximum
// and with it every weight of the row.
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x for a pair on the FMA and ALU pipes: x = n + f with n the nearest
// integer (the 1.5 2^23 shifter), 2^f by a cubic on [-1/2, 1/2] (relative
// error 7.5e-5, a fiftieth of the bf16 rounding of P), n added to the
// exponent field.  x is clamped at -126, so a masked score gives 1e-38.
__device__ __forceinline__ void ex2_poly2(float x0, float x1, float& r0, float& r1) {
    const uint64_t x2 = f2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
    const uint64_t sh = f2(12582912.0f, 12582912.0f);
    const uint64_t t = fadd2(x2, sh);
    const uint64_t n = fadd2(t, f2(-12582912.0f, -12582912.0f));
    const uint64_t f = ffma2(n, f2(-1.0f, -1.0f), x2);
    uint64_t p = ffma2(f2(0.0551716648f, 0.0551716648f), f, f2(0.2426111251f, 0.2426111251f));
    p = ffma2(p, f, f2(0.6932609677f, 0.6932609677f));
    p = ffma2(p, f, f2(0.9999280572f, 0.9999280572f));
    float t0, t1, p0, p1;
    f2_split(t, t0, t1);
    f2_split(p, p0, p1);
    const int kSh = __float_as_int(12582912.0f);
    r0 = __int_as_float(__float_as_int(p0) + ((__float_as_int(t0) - kSh) << 23));
    r1 = __int_as_float(__float_as_int(p1) + ((__float_as_int(t1) - kSh) << 23));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
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

// Bounded wait; after the first expiry in a thread its later waits return at
// once, so a broken pipeline unwinds in about one timeout.
__device__ __forceinline__ void wait_or_flag(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code, bool& failed) {
    if (failed) return;
    if (!mbar_wait(bar, parity)) {
        record_error(err, code);
        failed = true;
    }
}

struct ChunkTma {
    CUtensorMap k, v;   // the layer's pools as [pool rows][n_head_kv * 64] bf16, box {64, 64}
};

// Where a row's result goes: 64 values in the type of q, or a partial row.
template <class Act>
struct RowOut {
    Act* out;        // nullptr: partial
    float* part;
    float* lse;
};
// r: the row's index in the item; block: which of the item's partial blocks
// after the segment's first (0 or 1).
template <class Act>
__device__ __forceinline__ RowOut<Act> row_out(const ChunkArgs& A, const Work& w, int r, int block) {
    RowOut<Act> o{};
    if (w.part < 0) {
        const int row = w.row0 + r, t = row / A.group, h = row - t * A.group;
        o.out = static_cast<Act*>(A.out) + static_cast<int64_t>(w.first + t) * A.out_stride +
                (w.kvh * A.group + h) * HD;
    } else {
        const size_t at = static_cast<size_t>(w.part) + static_cast<size_t>(block) * w.n_rows + r;
        o.part = A.part_o + at * HD;
        o.lse = A.part_lse + at;
    }
    return o;
}
__device__ __forceinline__ void store8(float* p, const float* x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* x) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

__device__ __forceinline__ void bf16x8(const uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

// One row of a segment from global memory, attended rows only: the way taken
// when a masked row of V is not finite (see above); tiles t, t + step, ...
template <class Act>
__device__ __noinline__ void chunk_row_exact(const ChunkArgs& A, const Work& w, int r, int t, int step, RowOut<Act> dst) {
    const int row = w.row0 + r, tok = row / A.group, h = w.kvh * A.group + row - tok * A.group;
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
    for (; t < w.t1; t += step) {
        const int end = min((t + 1) * kTile, pos + 1);
        for (int j = t * kTile; j < end; ++j) {
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
    const float inv = m == -INFINITY ? 0.f : 1.0f / l;
    if (dst.lse) *dst.lse = m == -INFINITY ? -INFINITY : m + log2f(l);
    for (int d = 0; d < HD; d += 8) {
        float x[8];
        for (int e = 0; e < 8; ++e) x[e] = o[d + e] * inv;
        if (dst.out) store8(dst.out + d, x);
        else store8(dst.part + d, x);
    }
}

// Warp roles (512 threads, one CTA per SM):
//   warp 0      TMA producer of K/V tiles, all segments in order;
//   warps 1, 2  MMA issuers of softmax warpgroup 1 / 2;
//   warp 3      V of the edge tiles;
//   warps 4-11  softmax, one TMEM lane (= row) per thread;
//   warps 12-15 Q rows into shared memory (bf16 terms, swizzled).
template <bool F32>
__global__ void __launch_bounds__(CT_THREADS, 1)
    chunk_attn_kernel(const __grid_constant__ ChunkArgs A, const __grid_constant__ ChunkTma M) {
    using Smem = ChunkSmem<F32>;
    using Act = std::conditional_t<F32, float, __nv_bfloat16>;
    constexpr int kTerms = Smem::kTerms, kQBufs = Smem::kQBufs;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < CT_STAGES; ++i) {
            mbar_init(&S.kv_full[i], 1);
            mbar_init(&S.kv_empty[i], 3);
            mbar_init(&S.v_ok[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.q_full[i], 4);   // one arrival per loader warp
            mbar_init(&S.q_free[i], 2 + 8);
            mbar_init(&S.scanned[i], 1);
            mbar_init(&S.s_full[i], 1);
            mbar_init(&S.s_free[i], 4);
            mbar_init(&S.p_full[i], 4);
            mbar_init(&S.p_free[i], 1);
        }
        fence_barrier_init();
        prefetch_tmap(&M.k);
        prefetch_tmap(&M.v);
    }
    if (warp == 0) {
        tmem_alloc(&S.tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = S.tmem_base;
    // everything below reads what earlier kernels on the stream wrote
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int seg0 = A.d.cta_start[blockIdx.x], seg1 = A.d.cta_start[blockIdx.x + 1];
    if (tid < kWorkCache && seg0 + tid < seg1) S.work[tid] = work_at(A, seg0 + tid);
    __syncthreads();
    auto work_of = [&](int i) { return i - seg0 < kWorkCache ? S.work[i - seg0] : work_at(A, i); };
    bool failed = false;

    if (wg == 0) {
        regs_dealloc<kRegsControl>();
        if (warp == 0) {
            // ------------------------------ TMA producer ------------------------------
            int ring = 0;
            for (int i = seg0; i < seg1; ++i) {
                const Work w = work_of(i);
                const int pool_rows = A.pool_pages << A.page_shift;   // a box from here on is all zeros
                // lane l holds where box b0 + l starts
                int b0 = 2 * w.t0, y = 0;
                auto refill = [&]() {
                    const int r = (b0 + lane) * kBox;
                    y = pool_rows;
                    if (r < w.kv_len) {
                        const int id = w.pages[r >> A.page_shift];
                        if (static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages))
                            y = (id << A.page_shift) + (r & ((1 << A.page_shift) - 1));
                        else if (b0 + lane < 2 * w.t1)
                            record_error(A.err, kErrBadPage);
                    }
                };
                refill();
                for (int n = w.t0; n < w.t1; ++n, ++ring) {
                    if (2 * n - b0 >= 32) {
                        b0 = 2 * n;
                        refill();
                    }
                    const int st = ring % CT_STAGES;
                    const int y0 = __shfl_sync(0xffffffffu, y, 2 * n - b0);
                    const int y1 = __shfl_sync(0xffffffffu, y, 2 * n - b0 + 1);
                    wait_or_flag(&S.kv_empty[st], ((ring / CT_STAGES) & 1) ^ 1, A.err, kErrWaitEmpty, failed);
                    if (lane == 0 && !failed) {
                        mbar_arrive_expect_tx(&S.kv_full[st], 2 * kTileHalfs * 2);
                        tma_load_2d(S.k[st], &M.k, w.kvh * HD, y0, &S.kv_full[st]);
                        tma_load_2d(S.k[st] + kBox * HD, &M.k, w.kvh * HD, y1, &S.kv_full[st]);
                        tma_load_2d(S.v[st], &M.v, w.kvh * HD, y0, &S.kv_full[st]);
                        tma_load_2d(S.v[st] + kBox * HD, &M.v, w.kvh * HD, y1, &S.kv_full[st]);
                    }
                    __syncwarp();
                }
            }
            // no copy may still be in flight when the CTA leaves
            for (int u = ring > CT_STAGES ? ring - CT_STAGES : 0; u < ring && !failed; ++u)
                wait_or_flag(&S.kv_full[u % CT_STAGES], (u / CT_STAGES) & 1, A.err, kErrDrain, failed);
        } else if (warp == 3) {
            // -------------------------- V of the edge tiles ----------------------------
            int ring = 0;
            for (int i = seg0; i < seg1; ++i) {
                const int k = i - seg0;
                const Work w = work_of(i);
                // the Q of this segment is loaded only after the softmax is done with
                // the segment that used this flag before
                wait_or_flag(&S.q_full[k % kQBufs], (k / kQBufs) & 1, A.err, kErrWaitFull, failed);
                if (lane == 0) S.bad[k & 1] = 0;
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
                                const uint4 x = v[e];
                                auto full = [](uint32_t u) { return ((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
                                bad |= (full(x.x) | full(x.y) | full(x.z) | full(x.w)) != 0;   // exponent all ones
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
            // ------------------------------ MMA issuers --------------------------------
            // Warp 1 + i serves softmax warpgroup i.  It walks every tile: its
            // own ones get S = Q K^T (as soon as the softmax has read the last
            // S, ahead of the last tile's PV) and O += P V, the others are
            // released at once.
            const int i = warp - 1;
            const uint32_t tS = tmem + col_s(i), tP = tmem + col_p(i), tO = tmem + col_o(i);
            int ring = 0;          // the tile the walk stands on
            uint32_t v_par = 0;    // parity of the next v_ok of each stage
            int seg = seg0, k = 0, n = 0;
            Work w{};
            if (seg < seg1) {
                w = work_of(seg);
                n = w.t0;
            }
            struct Own {
                int ring, k;
                bool first, edge;
                uint32_t v_parity;
            };
            // The next own tile, the walk left behind it; false at the end.
            auto next_own = [&](Own& o) {
                while (seg < seg1) {
                    if (n == w.t1) {
                        const bool none = !w.dual && w.t0 + i >= w.t1;
                        if (none) {   // no tile of this segment is ours: q_full first, so that the
                                      // arrival belongs to this segment's phase
                            wait_or_flag(&S.q_full[k % kQBufs], (k / kQBufs) & 1, A.err, kErrWaitFull, failed);
                            if (lane == 0) mbar_arrive(&S.q_free[k % kQBufs]);
                        }
                        ++seg;
                        ++k;
                        if (seg == seg1) return false;
                        w = work_of(seg);
                        n = w.t0;
                        continue;
                    }
                    const int st = ring % CT_STAGES;
                    const bool edge = w.edge(n);
                    const bool mine = w.dual || ((n - w.t0) & 1) == i;
                    const uint32_t par = (v_par >> st) & 1;
                    if (edge) v_par ^= 1u << st;
                    if (mine) {
                        o = Own{ring, k, n - w.t0 < (w.dual ? 1 : 2), edge, par};
                        ++n;
                        ++ring;
                        return true;
                    }
                    wait_or_flag(&S.kv_full[st], (ring / CT_STAGES) & 1, A.err, kErrWaitFull, failed);
                    if (lane == 0) mbar_arrive(&S.kv_empty[st]);
                    __syncwarp();
                    ++n;
                    ++ring;
                }
                return false;
            };
            // Whether the own tile just returned is the segment's last own one.
            auto last_own = [&]() { return w.dual ? n == w.t1 : n + 1 >= w.t1; };
            auto issue_s = [&](const Own& o, int a, bool last) {   // a: own tiles before this one
                const int st = o.ring % CT_STAGES, b = o.k % kQBufs;
                if (o.first) wait_or_flag(&S.q_full[b], (o.k / kQBufs) & 1, A.err, kErrWaitFull, failed);
                wait_or_flag(&S.kv_full[st], (o.ring / CT_STAGES) & 1, A.err, kErrWaitFull, failed);
                if (a > 0) wait_or_flag(F32 ? &S.p_free[i] : &S.s_free[i], (a - 1) & 1, A.err, kErrWaitMma, failed);
                tc_fence_after();
                if (elect_one()) {
                    const int m = w.dual ? i : 0;
                    const uint64_t dk = sw128_desc(smem_u32(S.k[st]));
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) {   // the smallest first
                        const uint64_t dq = sw128_desc(smem_u32(S.q[b][m][term]));
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk)
                            umma_bf16(tS, dq + 2 * kk, dk + 2 * kk, kIdS, term < kTerms - 1 || kk > 0);
                    }
                    umma_commit(&S.s_full[i]);
                    if (last) umma_commit(&S.q_free[b]);
                }
                __syncwarp();
            };
            auto issue_pv = [&](const Own& o, int a) {
                const int st = o.ring % CT_STAGES;
                if (o.edge) wait_or_flag(&S.v_ok[st], o.v_parity, A.err, kErrWaitFull, failed);
                wait_or_flag(&S.p_full[i], a & 1, A.err, kErrWaitMma, failed);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t dv = v_desc(smem_u32(S.v[st]));
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) {
                        const uint32_t tp = term == kTerms - 1 ? tP : tS + 64 * term;
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; ++kk)
                            umma_bf16_tmem_a(tO, tp + 8 * kk, dv + (2048 >> 4) * kk, kIdO,
                                             (!o.first || term < kTerms - 1 || kk > 0) ? 1u : 0u);
                    }
                    umma_commit(&S.p_free[i]);
                    umma_commit(&S.kv_empty[st]);
                }
                __syncwarp();
            };
            Own cur{}, nxt{};
            int a = 0;
            bool have = next_own(cur);
            if (have) issue_s(cur, 0, last_own());
            while (have) {
                if constexpr (F32) {
                    issue_pv(cur, a);
                    have = next_own(nxt);
                    if (have) issue_s(nxt, a + 1, last_own());
                } else {
                    have = next_own(nxt);
                    if (have) issue_s(nxt, a + 1, last_own());
                    issue_pv(cur, a);
                }
                cur = nxt;
                ++a;
            }
            if (a > 0) wait_or_flag(&S.p_free[i], (a - 1) & 1, A.err, kErrDrain, failed);   // MMAs done before TMEM is freed
        }
    } else if (wg == 3) {
        // ------------------------------ Q loader -----------------------------------
        regs_dealloc<kRegsLoader>();
        const int lw = warp - 12;
        for (int i = seg0; i < seg1; ++i) {
            const int k = i - seg0, b = k % kQBufs;
            const Work w = work_of(i);
            if (k >= kQBufs) wait_or_flag(&S.q_free[b], ((k / kQBufs) - 1) & 1, A.err, kErrWaitEmpty, failed);
            // 8 lanes per row, 4 rows per step, a quarter of each row tile per warp
            const int ch = lane & 7;
            for (int m = 0; m < (w.dual ? 2 : 1); ++m) {
                auto source = [&](int r, bool& ok) {
                    const int row = w.row0 + m * kChunkRows + r, t = row / A.group, h = row - t * A.group;
                    ok = m * kChunkRows + r < w.n_rows;
                    return ok ? static_cast<const Act*>(A.q) + static_cast<int64_t>(w.first + t) * A.q_stride +
                                    (w.kvh * A.group + h) * HD + ch * 8
                              : static_cast<const Act*>(A.q);
                };
                if constexpr (!F32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int r = lw * 32 + 4 * j + (lane >> 3);
                        bool ok;
                        const Act* src = source(r, ok);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         smem_u32(&S.q[b][m][0][r * HD + ((ch ^ (r & 7)) << 3)])),
                                     "l"(src), "r"(ok ? 16 : 0)
                                     : "memory");
                    }
                } else {
#pragma unroll
                    for (int j0 = 0; j0 < 8; j0 += 4) {
                        float4 x[4][2];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            bool ok;
                            const float4* src = reinterpret_cast<const float4*>(source(lw * 32 + 4 * (j0 + j) + (lane >> 3), ok));
                            x[j][0] = x[j][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (ok) {
                                x[j][0] = src[0];
                                x[j][1] = src[1];
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int r = lw * 32 + 4 * (j0 + j) + (lane >> 3);
                            float* f = reinterpret_cast<float*>(x[j]);
#pragma unroll
                            for (int term = 0; term < kTerms; ++term) {
                                *reinterpret_cast<uint4*>(&S.q[b][m][term][r * HD + ((ch ^ (r & 7)) << 3)]) =
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
    } else {
        // ------------------------------ softmax ------------------------------------
        regs_alloc<kRegsSoftmax>();
        const int i = wg - 1;
        const int lr = tid - 128 * wg;                 // TMEM lane
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lanes + col_s(i), tP = tmem + lanes + col_p(i), tO = tmem + lanes + col_o(i);
        int a = 0;   // own tiles so far (barrier phases)
        for (int sgi = seg0; sgi < seg1; ++sgi) {
            const int k = sgi - seg0;
            const Work w = work_of(sgi);
            const int step = w.dual ? 1 : 2;
            const int n0 = w.dual ? w.t0 : w.t0 + i;
            if (n0 >= w.t1) {   // no tile of this segment is ours
                wait_or_flag(&S.q_full[k % kQBufs], (k / kQBufs) & 1, A.err, kErrWaitFull, failed);
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.q_free[k % kQBufs]);
                continue;
            }
            const int r = w.dual ? 128 * i + lr : lr;  // row of the item
            const int my_pos = w.pos + (w.row0 + min(r, w.n_rows - 1)) / A.group;
            float m_ref = -INFINITY;                   // reference maximum, log2 units
            float l_run = 0.f;
            for (int n = n0; n < w.t1; n += step, ++a) {
                wait_or_flag(&S.s_full[i], a & 1, A.err, kErrWaitMma, failed);
                tc_fence_after();
                float s[kTile];
#pragma unroll
                for (int c = 0; c < kTile / 32; ++c) {
                    float tmp[32];
                    tmem_ld32(tS + 32 * c, tmp);
#pragma unroll
                    for (int e = 0; e < 32; ++e) s[32 * c + e] = tmp[e];
                }
                tmem_wait_ld();
                if constexpr (!F32) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S.s_free[i]);   // the MMA may overwrite S
                }
                const int left = my_pos - n * kTile;   // the last attended key of this tile
                if (left < kTile - 1) {
#pragma unroll
                    for (int e = 0; e < kTile; ++e)
                        if (e > left) s[e] = -INFINITY;
                }
                float mc[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    float m = fmax3(s[8 * c], s[8 * c + 1], s[8 * c + 2]);
                    m = fmax3(m, s[8 * c + 3], s[8 * c + 4]);
                    m = fmax3(m, s[8 * c + 5], s[8 * c + 6]);
                    mc[c] = fmax3(m, s[8 * c + 7], m);
                }
#pragma unroll
                for (int c = 0; c < 5; ++c) mc[c] = fmax3(mc[3 * c], mc[3 * c + 1], mc[3 * c + 2]);
                const float mt = fmax3(fmax3(mc[0], mc[1], mc[2]), fmax3(mc[3], mc[4], mc[15]), -INFINITY) * kExpScale;
                float alpha = 1.f;
                const bool move = m_ref == m_ref && !(mt <= m_ref + kMoveThreshold);   // to a NaN too, never from one
                if (move) {
                    alpha = (m_ref == -INFINITY) ? 0.f : exp2f(m_ref - mt);
                    m_ref = mt;
                }
                const float m_use = m_ref == -INFINITY ? 0.f : m_ref;   // nothing attended so far: weights 0
                const uint64_t sc2 = f2(kExpScale, kExpScale), negm2 = f2(-m_use, -m_use);
                // P and O may be touched once the previous PV is done
                auto settle = [&]() {
                    if (n > n0) {
                        wait_or_flag(&S.p_free[i], (a - 1) & 1, A.err, kErrWaitMma, failed);
                        tc_fence_after();
                        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                            for (int c = 0; c < HD / 32; ++c) {
                                float o[32];
                                tmem_ld32(tO + 32 * c, o);
                                tmem_wait_ld();
                                uint32_t ob[32];
#pragma unroll
                                for (int e = 0; e < 32; ++e) ob[e] = __float_as_uint(o[e] * alpha);
                                tmem_st32(tO + 32 * c, ob);
                            }
                        }
                    }
                };
                uint64_t lsum2[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
                if constexpr (!F32) {
                    uint32_t pk[kTile / 2];
#pragma unroll
                    for (int e = 0; e < kTile / 2; ++e)
                        f2_split(ffma2(f2(s[2 * e], s[2 * e + 1]), sc2, negm2), s[2 * e], s[2 * e + 1]);
#pragma unroll
                    for (int e = 0; e < kTile / 2; ++e) {   // 5 pairs in 16 on the FMA pipe, the rest on the SFU
                        float p0, p1;
                        if ((e & 15) == 2 || (e & 15) == 5 || (e & 15) == 7 || (e & 15) == 10 || (e & 15) == 13) {
                            ex2_poly2(s[2 * e], s[2 * e + 1], p0, p1);
                        } else {
                            p0 = ex2_sfu(s[2 * e]);
                            p1 = ex2_sfu(s[2 * e + 1]);
                        }
                        s[2 * e] = p0;
                        s[2 * e + 1] = p1;
                    }
                    if (left < kTile - 1) {   // the cubic leaves 1e-38 at masked keys
#pragma unroll
                        for (int e = 0; e < kTile; ++e)
                            if (e > left) s[e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < kTile / 2; ++e) {
                        lsum2[e & 3] = fadd2(lsum2[e & 3], f2(s[2 * e], s[2 * e + 1]));
                        pk[e] = pack_bf16(s[2 * e], s[2 * e + 1]);
                    }
                    settle();
                    tmem_st32(tP, *reinterpret_cast<const uint32_t(*)[32]>(&pk[0]));
                    tmem_st32(tP + 32, *reinterpret_cast<const uint32_t(*)[32]>(&pk[32]));
                } else {
                    settle();
#pragma unroll
                    for (int c = 0; c < kTile / 32; ++c) {   // 32 keys: 16 columns of each term
                        uint32_t t0[16], t1[16], t2[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float x0, x1;
                            f2_split(ffma2(f2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), sc2, negm2), x0, x1);
                            x0 = ex2_sfu(x0);
                            x1 = ex2_sfu(x1);
                            lsum2[e & 3] = fadd2(lsum2[e & 3], f2(x0, x1));
                            t0[e] = top_pair(x0, x1);
                            f2_split(rest_pair(x0, x1), x0, x1);
                            t1[e] = top_pair(x0, x1);
                            f2_split(rest_pair(x0, x1), x0, x1);
                            t2[e] = top_pair(x0, x1);
                        }
                        tmem_st16(tS + 16 * c, t0);
                        tmem_st16(tS + 64 + 16 * c, t1);
                        tmem_st16(tP + 16 * c, t2);
                    }
                }
                float lsum0, lsum1;
                f2_split(fadd2(fadd2(lsum2[0], lsum2[1]), fadd2(lsum2[2], lsum2[3])), lsum0, lsum1);
                l_run = l_run * alpha + (lsum0 + lsum1);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.p_full[i]);
            }
            // ---- epilogue ----
            wait_or_flag(&S.p_free[i], (a - 1) & 1, A.err, kErrWaitMma, failed);
            wait_or_flag(&S.scanned[k & 1], (k >> 1) & 1, A.err, kErrWaitMma, failed);
            tc_fence_after();
            const bool mine = r < w.n_rows;
            const RowOut<Act> dst = row_out<Act>(A, w, mine ? r : 0, w.dual ? 0 : i);
            if (S.bad[k & 1]) {
                if (mine) chunk_row_exact<Act>(A, w, r, n0, step, dst);
                __syncwarp();
            } else {
                const bool empty = m_ref == -INFINITY;
                const float inv = empty ? 0.f : 1.0f / l_run;
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    float o[32];
                    tmem_ld32(tO + 32 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = empty ? 0.f : o[e] * inv;
                    if (mine) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (dst.out) store8(dst.out + 32 * c + e, o + e);
                            else store8(dst.part + 32 * c + e, o + e);
                        }
                    }
                }
                if (mine && dst.lse) *dst.lse = empty ? -INFINITY : m_ref + log2f(l_run);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.q_free[k % kQBufs]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Items in several partial blocks: out = sum_b w_b o_b / sum_b w_b, w_b =
// 2^(lse_b - max), in block order.  A warp per row, lane = two columns.
constexpr int kMergeThreads = 256;
template <class Act>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const __grid_constant__ ChunkArgs A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const ChunkMerge m = A.d.merges[blockIdx.x];
    const int r = blockIdx.y * (kMergeThreads / 32) + (threadIdx.x >> 5);
    if (r >= m.n_rows) return;
    const float* lse = A.part_lse + m.part + r;
    const float* po = A.part_o + (static_cast<size_t>(m.part) + r) * HD + 2 * lane;
    float mx = -INFINITY;
    for (int b = lane; b < m.n_parts; b += 32) mx = fmaxf(mx, lse[static_cast<size_t>(b) * m.n_rows]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float2 acc = make_float2(0.f, 0.f);
    float sum = 0.f;
    for (int b0 = 0; b0 < m.n_parts; b0 += 32) {
        const int nb = min(32, m.n_parts - b0);
        float w = lane < nb ? exp2f(lse[static_cast<size_t>(b0 + lane) * m.n_rows] - mx) : 0.f;
#pragma unroll 8
        for (int b = 0; b < nb; ++b) {
            const float wb = __shfl_sync(0xffffffffu, w, b);
            const float2 x = *reinterpret_cast<const float2*>(po + static_cast<size_t>(b0 + b) * m.n_rows * HD);
            sum += wb;
            acc.x = fmaf(wb, x.x, acc.x);
            acc.y = fmaf(wb, x.y, acc.y);
        }
    }
    const ChunkSeq sq = A.d.seqs[m.seq];
    const int row = m.row0 + r, t = row / A.group, h = row - t * A.group;
    const float inv = 1.0f / sum;
    Act* out = static_cast<Act*>(A.out) + static_cast<int64_t>(sq.first + t) * A.out_stride +
               (m.kvh * A.group + h) * HD + 2 * lane;
    store_pair(out, make_float2(acc.x * inv, acc.y * inv));
}

// Launch configuration of a programmatic dependent of the kernel before it.
struct Launch {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg{};
    Launch(dim3 grid, int threads, size_t smem, cudaStream_t stream) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
};

}  // namespace

cudaError_t launch_append(const AppendArgs& a, bool act_bf16, bool pool_bf16, cudaStream_t stream) {
    const int units = a.n_head + 2 * a.n_head_kv;
    const int64_t warps = static_cast<int64_t>(a.n_tokens) * ((units + kUnitsPerWarp - 1) / kUnitsPerWarp);
    const int64_t blocks = (warps * 32 + kAppendThreads - 1) / kAppendThreads;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    Launch L(dim3(static_cast<unsigned>(blocks)), kAppendThreads, 0, stream);
    if (act_bf16)
        return pool_bf16 ? cudaLaunchKernelEx(&L.cfg, append_kernel<__nv_bfloat16, __nv_bfloat16>, a)
                         : cudaLaunchKernelEx(&L.cfg, append_kernel<__nv_bfloat16, float>, a);
    return pool_bf16 ? cudaLaunchKernelEx(&L.cfg, append_kernel<float, __nv_bfloat16>, a)
                     : cudaLaunchKernelEx(&L.cfg, append_kernel<float, float>, a);
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

cudaError_t launch_chunk_attention(const ChunkArgs& a, bool act_bf16, cudaStream_t stream) {
    ChunkTma m;
    const uint64_t cols = static_cast<uint64_t>(a.n_head_kv) * HD, rows = static_cast<uint64_t>(a.pool_pages) << a.page_shift;
    cudaError_t e = make_tmap_16b(&m.k, const_cast<uint16_t*>(a.key_pool), cols, rows, kBox, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    if (e != cudaSuccess) return e;
    e = make_tmap_16b(&m.v, const_cast<uint16_t*>(a.value_pool), cols, rows, kBox, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
    if (e != cudaSuccess) return e;
    e = act_bf16 ? launch_chunk_attn<false>(a, m, stream) : launch_chunk_attn<true>(a, m, stream);
    if (e != cudaSuccess || a.n_merge == 0) return e;
    constexpr int warps = kMergeThreads / 32;
    Launch L(dim3(a.n_merge, (a.merge_rows + warps - 1) / warps), kMergeThreads, 0, stream);
    return act_bf16 ? cudaLaunchKernelEx(&L.cfg, chunk_merge_kernel<__nv_bfloat16>, a)
                    : cudaLaunchKernelEx(&L.cfg, chunk_merge_kernel<float>, a);
}

}  // namespace tle
