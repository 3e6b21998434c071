// logits.cu -- the rules applied to a batch of logits before a token is
// sampled: repetition, frequency and presence penalties, biases and the mask
// of allowed tokens, in one launch.
//
// No reference counterpart (sample_temperature / sample_top_p,
// src/ops.h:262-278, take the raw logits).  For row r and token t, with c the
// times t was made and seen = t was given or made:
//   x  = seen ? (x > 0 ? x / rep_r : x rep_r) : x
//   x -= freq_r c;  x -= pres_r [c > 0];  x += sum of r's biases for t
//   out = allowed(r, t) ? x : -inf
//
// HBM-bound: 8 bytes per logit, read once and written once.  CTA (c, r) takes
// a slice of kSlice tokens of row r and holds what the lists say about them
// in shared memory (a count and a bias per token), so no list entry is
// written to global memory and none is lost or counted twice; it reads the
// whole lists of its row, which stay in L2.  Counts are integers, so their
// order does not matter; a token's biases are added in the list's order by
// one warp.
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace tle {

namespace {

constexpr int kSlice = 4096;        // tokens per CTA (32 KB of shared memory)
constexpr int kThreads = 256;
constexpr uint32_t kGiven = 0x80000000u;   // bit of a count: the token is in the prompt

template <bool PEN, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitArgs A) {
    __shared__ uint32_t count[PEN ? kSlice : 1];
    __shared__ float bias[BIAS ? kSlice : 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = blockIdx.y;
    const int v0 = blockIdx.x * kSlice;
    const int n = min(kSlice, A.n_vocab - v0);
    if constexpr (PEN)
        for (int i = tid; i < kSlice; i += kThreads) count[i] = 0;
    if constexpr (BIAS)
        for (int i = tid; i < kSlice; i += kThreads) bias[i] = 0.f;
    if constexpr (PEN || BIAS) __syncthreads();
    if constexpr (PEN) {
        const int lo = max(A.token_start[r], 0), hi = min(A.token_start[r + 1], A.n_list_tokens);
        const int given = A.n_prompt ? A.n_prompt[r] : 0;
        bool bad = false;
        for (int i = lo + tid; i < hi; i += kThreads) {
            const int t = A.tokens[i];
            if (static_cast<unsigned>(t) >= static_cast<unsigned>(A.n_vocab)) bad = true;
            else if (static_cast<unsigned>(t - v0) < static_cast<unsigned>(n)) {
                if (i - lo < given) atomicOr(&count[t - v0], kGiven);
                else atomicAdd(&count[t - v0], 1u);
            }
        }
        if (bad && blockIdx.x == 0) record_error(A.err, kErrBadToken);
    }
    if constexpr (BIAS) {
        if (warp == 0) {
            const int lo = max(A.bias_start[r], 0), hi = min(A.bias_start[r + 1], A.n_list_biases);
            for (int i0 = lo; i0 < hi; i0 += 32) {
                const int i = i0 + lane;
                const int t = i < hi ? A.bias_tokens[i] : -1;
                const float b = i < hi ? A.bias_values[i] : 0.f;
                if (i < hi && static_cast<unsigned>(t) >= static_cast<unsigned>(A.n_vocab) && blockIdx.x == 0)
                    record_error(A.err, kErrBadToken);
                const bool mine = t >= 0 && static_cast<unsigned>(t - v0) < static_cast<unsigned>(n);
                const uint32_t same = __match_any_sync(0xffffffffu, mine ? t : -1 - lane);
                // the first lane of a token adds the values of all its lanes, in order
                float sum = mine ? bias[t - v0] : 0.f;
                for (int l = 0; l < 32; ++l) {
                    const float x = __shfl_sync(0xffffffffu, b, l);
                    if ((same >> l) & 1u) sum += x;
                }
                if (mine && __ffs(same) - 1 == lane) bias[t - v0] = sum;
                __syncwarp();
            }
        }
    }
    if constexpr (PEN || BIAS) __syncthreads();
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if constexpr (PEN) {
        if (A.repetition) rep = A.repetition[r];
        if (A.frequency) freq = A.frequency[r];
        if (A.presence) pres = A.presence[r];
    }
    const float* src = A.logits + r * A.logits_stride + v0;
    float* dst = A.out + r * A.out_stride + v0;
    const uint32_t* words = MASK ? A.allowed + r * A.allowed_stride + v0 / 32 : nullptr;
    auto rule = [&](int i, float x) {
        if constexpr (PEN) {
            const uint32_t c = count[i];
            if (c) {
                x = x > 0.f ? x / rep : x * rep;
                const uint32_t made = c & ~kGiven;
                if (made) x = x - freq * static_cast<float>(made) - pres;
            }
        }
        if constexpr (BIAS) x += bias[i];
        return x;
    };
    for (int i = tid; i < n; i += kThreads) {
        float x = rule(i, src[i]);
        if constexpr (MASK)
            if (!((words[i >> 5] >> (i & 31)) & 1u)) x = -INFINITY;
        dst[i] = x;
    }
}

}  // namespace

cudaError_t launch_logits_adjust(const LogitArgs& a, int n_rows, cudaStream_t stream) {
    using Fn = void (*)(LogitArgs);
    static const Fn fns[8] = {logits_kernel<false, false, false>, logits_kernel<true, false, false>,
                              logits_kernel<false, true, false>,  logits_kernel<true, true, false>,
                              logits_kernel<false, false, true>,  logits_kernel<true, false, true>,
                              logits_kernel<false, true, true>,   logits_kernel<true, true, true>};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.n_vocab + kSlice - 1) / kSlice, n_rows);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fns[(a.tokens ? 1 : 0) + (a.bias_tokens ? 2 : 0) + (a.allowed ? 4 : 0)], a);
}

}  // namespace tle
