// chunk.cuh -- what the kernels on a chunk descriptor share: rows and their
// places, a CTA's pieces of work, bounded waits, conversions, launches.
#pragma once

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

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

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void bf16x8(const uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ void store8(float* p, const float* x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* x) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void store4(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}
template <int N, class T>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N]) {
    if constexpr (N == 8) store8(p, x);
    else store4(p, x);
}

constexpr float kExpScale = kScale * kLog2e;
// The reference maximum moves only when the row's maximum grows by more than
// 8 (log2 units), so O is rescaled rarely; P <= 2^8.
constexpr float kMoveThreshold = 8.0f;

// The token of row `row` of a (chunk, KV head): row / group by a multiplication
// (group_mul = ceil(2^(31 + L) / group) with L = ceil(log2 group), exact for rows
// below 2^31; 0 for a group of one).
__device__ __forceinline__ int row_token(const ChunkArgs& A, int row) {
    return A.group_mul ? static_cast<int>(__umulhi(static_cast<uint32_t>(row), A.group_mul) >> A.group_shift) : row;
}
constexpr int kTile = kChunkTile;   // 128
// A segment as the kernel's roles see it.
struct Work : ChunkSeg {
    __device__ __forceinline__ bool dual() const { return n_rows > kChunkRows; }
    __device__ __forceinline__ bool edge(int n) const { return n * kTile + kTile - 1 > pos_min; }
};
// The CTA's record `cta` (its first segment, and the range of all) into shared
// memory, by one thread; an empty range if the descriptor is not the launch's,
// of which nothing but the number is read then: it may end before this record.
__device__ __forceinline__ void fetch_first(const ChunkArgs& A, int cta, Work* to) {
    if (A.d.hdr->id == A.plan_id) {
        *to = *static_cast<const Work*>(A.d.cta + cta);
    } else {
        to->seg0 = to->seg1 = 0;
        record_error(A.err, kErrBadDesc);
    }
}
constexpr int kWorkCache = 20;   // segments of a CTA that are held in shared memory
// Those behind the first, by a warp that has nothing to do yet.
__device__ __forceinline__ void fetch_work(const ChunkArgs& A, int seg0, int seg1, Work* to, uint64_t* full) {
    const int lane = threadIdx.x & 31;
    for (int i = 4 + lane; i < 4 * kWorkCache; i += 32)
        if (seg0 + i / 4 < seg1) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(A.d.segs + seg0)[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
}

// Four 8 x 8 matrices of 16-bit elements (ldmatrix), as they lie and transposed.
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ float ex2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Maxima that keep a NaN: a NaN score poisons its row's reference maximum
// and with it every weight of the row.
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Bounded wait; after the first expiry in a thread its later waits return at
// once, so a broken pipeline unwinds in about one timeout.  The timer is read
// only after 256 probes: a wait here is short.
__device__ __forceinline__ void wait_or_flag(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code, bool& failed) {
    if (failed || mbar_test_wait(bar, parity)) return;
    uint64_t t0 = 0;
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 256; ++i)
            if (mbar_try_wait(bar, parity)) return;
        const uint64_t t = globaltimer();
        if (t0 == 0) t0 = t;
        if (t - t0 > kWaitTimeoutNs) break;
    }
    record_error(err, code);
    failed = true;
}

// Where a row's result goes: 64 values in the type of q, or a partial row.
template <class Act>
struct RowOut {
    Act* out;        // nullptr: partial
    float* part;
    float* lse;
};
// r: the row's index in the item.
template <class Act>
__device__ __forceinline__ RowOut<Act> row_out(const ChunkArgs& A, const Work& w, int r) {
    RowOut<Act> o{};
    if (w.part < 0) {
        const int row = w.row0 + r, t = row_token(A, row), h = row - t * A.group;
        o.out = static_cast<Act*>(A.out) + static_cast<int64_t>(w.first + t) * A.out_stride +
                (w.kvh * A.group + h) * HD;
    } else {
        const size_t at = static_cast<size_t>(w.part) + r;
        o.part = A.part_o + at * HD;
        o.lse = A.part_lse + at;
    }
    return o;
}
// Factor of the results of rows without any weight: a piece of an item counts
// for nothing when the pieces are joined; a whole row with scores of -inf only
// is 0/0.
__device__ __forceinline__ float no_weight(const Work& w) { return w.part < 0 ? NAN : 0.f; }

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

}  // namespace tle
