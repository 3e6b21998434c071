// logits.cu -- the rules applied to a batch of logits before a token is
// sampled: repetition, frequency and presence penalties, biases and the mask
// of allowed tokens, in one launch.
//
// No reference counterpart (sample_temperature / sample_top_p,
// src/ops.h:262-278, take the raw logits).  For row r and token t, with c the
// times t was made and seen = t was given or made:
//   x  = seen ? (x > 0 ? x / rep_r : x rep_r) : x
//   x -= freq_r c;  x -= pres_r [c > 0];  x += r's biases for t, in order
//   out = allowed(r, t) ? x : -inf
//
// HBM-bound: 8 bytes per logit, read once and written once.  CTA (c, r) takes
// a slice of SLICE tokens of row r and counts in shared memory what the list of
// tokens so far says about them, so no list entry is written to global memory
// and none is lost or counted twice; it reads the whole lists of its row, which
// stay in L2, 16 bytes a lane.  Counts are integers, so their order does not
// matter.  The logits go through in 16-byte pieces wherever both rows are
// aligned alike, loaded before the lists are gone through.  Biases are few:
// the slice's own are gathered in the list's order, and after the logits are
// stored the thread of a token's first entry adds its entries, in order, to the
// token's result.
//
// The slice: 8192 tokens, so that a row's lists are read few times (256 rows of
// 100003 with lists of 4000 tokens: 63 us, with 4096 tokens 71 us), or 2048 where
// that would leave SMs idle (one row of 32000: 3.3 us against 5.0 us).  Of the 63 us
// the 205 MB of logits are 31 us at the copy rate; the rest is the chain of row
// scalars, lists, counts and results, with three CTAs per SM (74 registers) to hide
// it.  Held to 64 or 48 registers it spills (67, 92 us); 512 threads a CTA: 71 us.
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace tle {

namespace {

constexpr int kThreads = 256;
constexpr int kBiasList = 512;      // biases of a slice that are gathered at a time
constexpr int kManySlices = 2 * 148;   // slices of 8192 from which on they are taken
constexpr uint32_t kGiven = 0x80000000u;   // bit of a count: the token is in the prompt

template <int SLICE, bool PEN, bool BIAS, bool MASK>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ LogitArgs A) {
    constexpr int kSlice = SLICE;
    constexpr int kPieces = kSlice / 4 / kThreads;   // 16-byte pieces per thread
    extern __shared__ __align__(16) unsigned char tables[];
    uint32_t* count = reinterpret_cast<uint32_t*>(tables);   // PEN: [kSlice + 4]
    __shared__ int bias_token[BIAS ? kBiasList : 1];
    __shared__ float bias_value[BIAS ? kBiasList : 1];
    __shared__ int bias_n, bias_next;   // entries gathered; where the list goes on
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r = blockIdx.y;
    const int v0 = blockIdx.x * kSlice;
    const int n = min(kSlice, A.n_vocab - v0);
    const float* src = A.logits + r * A.logits_stride + v0;
    float* dst = A.out + r * A.out_stride + v0;
    // elements before the first 16-byte boundary of the slice, and where its
    // token 0 lies in the tables, so that their pieces are aligned with it
    const int head = static_cast<int>((-(reinterpret_cast<uintptr_t>(src) >> 2)) & 3u);
    const int pad = (4 - head) & 3;
    if constexpr (PEN)
        for (int i = tid; i < (kSlice + 4) / 4; i += kThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // everything whose place is known is on its way at once: the row's scalars, the
    // slice's mask and logits (needed only after the lists are gone through)
    int lo = 0, hi = 0, given = 0, bias_lo = 0, bias_hi = 0;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if constexpr (PEN) {
        lo = A.token_start[r];
        hi = A.token_start[r + 1];
        if (A.n_prompt) given = A.n_prompt[r];
        if (A.repetition) rep = A.repetition[r];
        if (A.frequency) freq = A.frequency[r];
        if (A.presence) pres = A.presence[r];
    }
    if constexpr (BIAS) {
        bias_lo = A.bias_start[r];
        bias_hi = A.bias_start[r + 1];
    }
    static_assert(kSlice / 32 <= kThreads, "a mask word per thread");
    __shared__ uint32_t words[MASK ? kSlice / 32 + 1 : 1];
    uint32_t word = 0;
    if (MASK && tid < (n + 31) / 32) word = A.allowed[r * A.allowed_stride + v0 / 32 + tid];
    const bool alike = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15u) == 0;
    const int body = alike && n > head ? (n - head) / 4 : 0;   // pieces
    float4 x[kPieces];
#pragma unroll
    for (int q = 0; q < kPieces; ++q)
        if (tid + q * kThreads < body) x[q] = *reinterpret_cast<const float4*>(src + head + 4 * (tid + q * kThreads));
    if constexpr (PEN) __syncthreads();
    // cut to the lists, which end at 2^30, so that no sum below overflows
    hi = max(min(hi, A.n_list_tokens), 0);
    lo = min(max(lo, 0), hi);
    bias_hi = max(min(bias_hi, A.n_list_biases), 0);
    bias_lo = min(max(bias_lo, 0), bias_hi);
    // The last warp gathers the slice's biases from entry i0 of the list on, until
    // the list ends or kBiasList are there.
    auto gather = [&](int i0) {
        constexpr int kAhead = 8;   // times 32 entries in flight
        int have = 0;
        for (; i0 < bias_hi && have + 32 * kAhead <= kBiasList; i0 += 32 * kAhead) {
            int t[kAhead];
            float b[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int i = i0 + 32 * q + lane;
                t[q] = i < bias_hi ? A.bias_tokens[i] : -1;
                b[q] = i < bias_hi ? A.bias_values[i] : 0.f;
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int i = i0 + 32 * q + lane;
                if (i < bias_hi && static_cast<unsigned>(t[q]) >= static_cast<unsigned>(A.n_vocab) && blockIdx.x == 0)
                    record_error(A.err, kErrBadToken);
                const bool mine = i < bias_hi && static_cast<unsigned>(t[q] - v0) < static_cast<unsigned>(n);
                const uint32_t set = __ballot_sync(0xffffffffu, mine);
                if (mine) {
                    const int at = have + __popc(set & ((1u << lane) - 1));
                    bias_token[at] = t[q] - v0;
                    bias_value[at] = b[q];
                }
                have += __popc(set);
            }
        }
        if (lane == 0) {
            bias_n = have;
            bias_next = i0;
        }
    };
    // With biases the last warp goes through their list and the others through the
    // tokens.  Up to 32 biases that are the whole list's stay in its lanes, with
    // their tokens' logits.
    const bool lister = BIAS && warp == kThreads / 32 - 1;
    constexpr int kCounters = BIAS ? kThreads - 32 : kThreads;
    bool in_lanes = false;
    int my_t = -1 - lane;
    float my_b = 0.f, my_x = 0.f;
    if (lister) {
        gather(bias_lo);
        __syncwarp();
        const int nb = bias_n;
        in_lanes = nb <= 32 && bias_next >= bias_hi;
        if (in_lanes && lane < nb) {
            my_t = bias_token[lane];
            my_b = bias_value[lane];
            my_x = src[my_t];
        }
    }
    if (PEN && !lister) {
        bool bad = false;
        auto take = [&](int i, int t) {
            if (static_cast<unsigned>(t) >= static_cast<unsigned>(A.n_vocab)) bad = true;
            else if (static_cast<unsigned>(t - v0) < static_cast<unsigned>(n)) {
                if (i - lo < given) atomicOr(&count[pad + t - v0], kGiven);
                else atomicAdd(&count[pad + t - v0], 1u);
            }
        };
        // 4 tokens a lane from the first 16-byte boundary on, the ends one by one
        const int a0 = min(hi, lo + static_cast<int>((-(reinterpret_cast<uintptr_t>(A.tokens + lo) >> 2)) & 3u));
        const int a1 = hi > a0 ? a0 + (hi - a0) / 4 * 4 : a0;
        for (int i0 = a0 + 4 * tid; i0 < a1; i0 += 16 * kCounters) {   // four loads in flight
            int4 t[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (i0 + 4 * q * kCounters < a1) t[q] = *reinterpret_cast<const int4*>(A.tokens + i0 + 4 * q * kCounters);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = i0 + 4 * q * kCounters;
                if (i >= a1) break;
                take(i, t[q].x);
                take(i + 1, t[q].y);
                take(i + 2, t[q].z);
                take(i + 3, t[q].w);
            }
        }
        if (lo + tid < a0) take(lo + tid, A.tokens[lo + tid]);
        if (a1 + tid < hi && tid < 4) take(a1 + tid, A.tokens[a1 + tid]);
        if (bad && blockIdx.x == 0) record_error(A.err, kErrBadToken);
    }
    if (MASK && tid < kSlice / 32) words[tid] = word;
    if constexpr (PEN || MASK) __syncthreads();
    auto rule = [&](float x, uint32_t c, uint32_t allowed) {
        if constexpr (PEN) {
            if (c) {
                x = x > 0.f ? x / rep : x * rep;
                const uint32_t made = c & ~kGiven;
                if (made) x = x - freq * static_cast<float>(made) - pres;
            }
        }
        if constexpr (MASK) x = (allowed & 1u) ? x : -INFINITY;
        return x;
    };
    auto one = [&](int i) {
        dst[i] = rule(src[i], PEN ? count[pad + i] : 0u, MASK ? words[i >> 5] >> (i & 31) : 0u);
    };
    if (!alike) {
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads) one(i);
    } else {
        if (tid < min(head, n)) one(tid);
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
            const int i = head + 4 * (tid + q * kThreads);
            if (tid + q * kThreads >= body) break;
            uint4 c = make_uint4(0, 0, 0, 0);
            if constexpr (PEN) c = *reinterpret_cast<const uint4*>(&count[pad + i]);
            uint32_t m = 0;
            if constexpr (MASK) m = __funnelshift_r(words[i >> 5], words[(i + 3) >> 5], i & 31);
            float4 y;
            y.x = rule(x[q].x, c.x, m);
            y.y = rule(x[q].y, c.y, m >> 1);
            y.z = rule(x[q].z, c.z, m >> 2);
            y.w = rule(x[q].w, c.w, m >> 3);
            *reinterpret_cast<float4*>(dst + i) = y;
        }
        if (head + 4 * body + tid < n && tid < 4) one(head + 4 * body + tid);
    }
    if constexpr (BIAS) {
        __syncthreads();   // the results and the gathered biases are there
        if (bias_n <= 32 && bias_next >= bias_hi) {
            if (!in_lanes) return;
            const uint32_t same = __match_any_sync(0xffffffffu, my_t);   // the lanes with this token
            // a token that is not allowed keeps its -inf, whatever its bias
            const bool have = my_t >= 0 && (!MASK || ((words[my_t >> 5] >> (my_t & 31)) & 1u));
            float y = have ? rule(my_x, PEN ? count[pad + my_t] : 0u, 1u) : 0.f;
            if (!__any_sync(0xffffffffu, have && (same & (same - 1)) != 0)) {
                y += my_b;
            } else {
                for (int l = 0; l < 32; ++l) {
                    const float b = __shfl_sync(0xffffffffu, my_b, l);
                    if ((same >> l) & 1u) y += b;
                }
            }
            if (have && __ffs(same) - 1 == lane) dst[my_t] = y;
            return;
        }
        for (;;) {
            const int nb = bias_n, next = bias_next;
            for (int i = tid; i < nb; i += kThreads) {
                const int t = bias_token[i];
                bool first = true;
                for (int j = 0; j < i; ++j) first &= bias_token[j] != t;
                if (!first || (MASK && !((words[t >> 5] >> (t & 31)) & 1u))) continue;
                float y = dst[t] + bias_value[i];
                for (int j = i + 1; j < nb; ++j)
                    if (bias_token[j] == t) y += bias_value[j];
                dst[t] = y;
            }
            if (next >= bias_hi) break;
            __syncthreads();   // read by all: the next ones
            if (warp == kThreads / 32 - 1) gather(next);
            __syncthreads();
        }
    }
}

template <int SLICE>
cudaError_t launch_slices(const LogitArgs& a, int n_rows, cudaStream_t stream) {
    using Fn = void (*)(LogitArgs);
    static const Fn fns[8] = {logits_kernel<SLICE, false, false, false>, logits_kernel<SLICE, true, false, false>,
                              logits_kernel<SLICE, false, true, false>,  logits_kernel<SLICE, true, true, false>,
                              logits_kernel<SLICE, false, false, true>,  logits_kernel<SLICE, true, false, true>,
                              logits_kernel<SLICE, false, true, true>,   logits_kernel<SLICE, true, true, true>};
    constexpr int kTable = (SLICE + 4) * 4;
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        for (Fn f : fns) {
            cudaError_t r = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kTable);
            if (r != cudaSuccess) return r;
        }
        return cudaSuccess;
    });
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((a.n_vocab + SLICE - 1) / SLICE, n_rows);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = a.tokens ? kTable : 0;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fns[(a.tokens ? 1 : 0) + (a.bias_tokens ? 2 : 0) + (a.allowed ? 4 : 0)], a);
}

}  // namespace

cudaError_t launch_logits_adjust(const LogitArgs& a, int n_rows, cudaStream_t stream) {
    const int64_t large = static_cast<int64_t>(n_rows) * ((a.n_vocab + 8191) / 8192);
    return large < kManySlices ? launch_slices<2048>(a, n_rows, stream) : launch_slices<8192>(a, n_rows, stream);
}

}  // namespace tle
