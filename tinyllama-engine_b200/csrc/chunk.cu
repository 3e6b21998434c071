// chunk.cu -- chunks of new tokens over a paged KV cache: append (rope + store)
// and causal attention.
//
// Reference semantics per token: rope() src/ops.cpp:1223-1281, then
// attention() src/ops.cpp:1317-1515 at its position, for a batch of chunks
// (generate.cpp:52-59 feeds a prompt one token at a time).  With f_i the
// frequency of pair i and p the token's position,
//   (x'_2i, x'_2i+1) = (x_2i cos a - x_2i+1 sin a, x_2i sin a + x_2i+1 cos a),  a = fl32(p f_i)
//   out_h(t) = sum_{j <= p} softmax_j(q'_h(t) . k_{h/g}(j) / 8) v_{h/g}(j).
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

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
// Simple form: one thread per (token, head), all keys in order.
constexpr int kRowThreads = 128;

__device__ __forceinline__ void bf16x8(const uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

template <class Act>
__global__ void __launch_bounds__(kRowThreads) chunk_rows_kernel(const __grid_constant__ ChunkArgs A, int n_tokens) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x;
    if (i >= static_cast<int64_t>(n_tokens) * A.n_head) return;
    const int g = A.n_head / A.n_head_kv;
    const int64_t tok = i / A.n_head;
    const int h = static_cast<int>(i - tok * A.n_head);
    const ChunkTok tk = A.d.toks[tok];
    const ChunkSeq sq = A.d.seqs[tk.seq];
    const int kvh = h / g;
    const Act* qp = static_cast<const Act*>(A.q) + tok * A.q_stride + h * HD;
    float q[HD], o[HD];
#pragma unroll
    for (int d = 0; d < HD; d += 2) {
        const float2 x = load_pair(qp + d);
        q[d] = x.x * (kScale * kLog2e);
        q[d + 1] = x.y * (kScale * kLog2e);
        o[d] = o[d + 1] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const size_t rs = static_cast<size_t>(A.n_head_kv) * HD;
    for (int j = 0; j <= tk.pos; ++j) {
        const int id = sq.pages[j >> A.page_shift];
        const bool ok = static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages);
        if (!ok) record_error(A.err, kErrBadPage);
        const size_t row = ok ? (static_cast<size_t>(id) << A.page_shift) | (j & ((1 << A.page_shift) - 1)) : 0;
        const uint4* kp = reinterpret_cast<const uint4*>(A.key_pool + row * rs + kvh * HD);
        const uint4* vp = reinterpret_cast<const uint4*>(A.value_pool + row * rs + kvh * HD);
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
            float f[8];
            bf16x8(ok ? kp[c] : make_uint4(0, 0, 0, 0), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(q[8 * c + e], f[e], s);
        }
        const float mn = fmaxf(m, s);
        const float al = (m == mn) ? 1.f : exp2f(m - mn);
        const float p = exp2f(s - mn);
        m = mn;
        l = l * al + p;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
            float f[8];
            bf16x8(ok ? vp[c] : make_uint4(0, 0, 0, 0), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[8 * c + e] = fmaf(o[8 * c + e], al, p * f[e]);
        }
    }
    const float inv = 1.0f / l;
    Act* op = static_cast<Act*>(A.out) + tok * A.out_stride + h * HD;
#pragma unroll
    for (int d = 0; d < HD; d += 2) store_pair(op + d, make_float2(o[d] * inv, o[d + 1] * inv));
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

cudaError_t launch_chunk_attention(const ChunkArgs& a, bool act_bf16, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.n_tokens) * a.n_head;
    Launch L(dim3(static_cast<unsigned>((rows + kRowThreads - 1) / kRowThreads)), kRowThreads, 0, stream);
    return act_bf16 ? cudaLaunchKernelEx(&L.cfg, chunk_rows_kernel<__nv_bfloat16>, a, a.n_tokens)
                    : cudaLaunchKernelEx(&L.cfg, chunk_rows_kernel<float>, a, a.n_tokens);
}

}  // namespace tle
