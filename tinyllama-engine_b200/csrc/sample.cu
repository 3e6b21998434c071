// sample.cu -- temperature, top-k, top-p and min-p on a batch of logits, and
// the token that a given uniform number draws, in one launch.
//
// The reference samples one row, from numbers of its own (sample_temperature,
// sample_top_p, src/ops.h:262-278).  Here row r with logits x, temperature T:
//   rank     tokens by x, largest first, equal ones by index
//   weight   w_i = exp((x_i - max x) / T)
//   top-k    the first k of the ranking
//   min-p    of these the ones with w_i >= min_p
//   top-p    of these the first ones until their weights reach p times the sum
//   token    the first kept one, by index, whose running sum of kept weights
//            exceeds u times their sum
// T <= 0: the first of the ranking.
//
// A kept set is a beginning of the ranking: all tokens of a key (logit) above some
// key and the first few, by index, of that key.  Both cuts are found by counting
// in bins of falling logits and going on inside the bin in which the count (top-k)
// or the sum of weights (top-p) is reached, so nothing is sorted.
//
// Weights are whole numbers of 2^-40 of the largest one, from an exponential in
// 64 bits: every sum is exact, whatever its order, so the same row gives the same
// token in any launch, and sums of 100000 tokens decide as 64-bit numbers do.
// A token below 2^-41 of the likeliest one is never drawn.
//
// A row is a cluster's: its logits are read once, into the shared memory of C
// CTAs, C slices of the vocabulary; what they find out about a slice is
// exchanged through distributed shared memory.
#include <cooperative_groups.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace tle {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kRowCtas = 8;
constexpr uint64_t kOne = 1ull << 40;      // the largest weight
constexpr float kReach = 28.6f;            // exp(-kReach) < 2^-41: weights beyond it are 0
// A weight in three limbs of 14, 13 and 13 bits, so that a bin's sums of 32 bits
// hold any slice (2^15.6 tokens).
constexpr uint32_t kLimb0 = 14, kLimb1 = 13;

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// exp(z) 2^40 for -kReach - 1 < z <= 0: z = n ln 2 + r, |r| <= ln 2 / 2, and 12 terms
// of r's power series (the next one is below 2^-47).
__device__ __forceinline__ double exp_scaled(double z) {
    const double n = rint(z * 1.4426950408889634);
    double r = fma(n, -0.693147182464599609375, z);      // ln 2 in 24 bits: n times it is exact
    r = fma(n, 1.904654299957768e-9, r);                 // and the rest
    double p = 1.0 / 39916800;
    p = fma(p, r, 1.0 / 3628800);
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return p * __longlong_as_double((static_cast<long long>(static_cast<int>(n) + 40 + 1023)) << 52);
}

struct RowRules {
    float mx;          // the largest logit
    float reach;       // logits at least so far below it weigh nothing
    double inv_t;
    double least;      // min_p 2^40
    __device__ __forceinline__ uint64_t weight(float x) const {
        if (x == mx) return kOne;
        if (!(mx - x < reach)) return 0;
        const double w = exp_scaled((static_cast<double>(x) - static_cast<double>(mx)) * inv_t);
        return w < least ? 0 : __double2ull_rn(w);
    }
};

struct Shared {
    uint32_t hist[3][kBins];
    uint64_t slot[2][3][kRowCtas];   // what the CTAs of the cluster told each other, by turns
    uint64_t warp_sum[kWarps];
    uint64_t found[2];
    uint32_t warp_u32[kWarps];
    int warp_arg[kWarps];
};

// The CTA's part of the exchanges: three numbers from each CTA to all.
struct Cluster {
    cg::cluster_group g;
    Shared& S;
    int rank, n, turn;
    __device__ __forceinline__ Cluster(Shared& s) : g(cg::this_cluster()), S(s), turn(0) {
        rank = static_cast<int>(g.block_rank());
        n = static_cast<int>(g.num_blocks());
    }
    // a, b, c of one thread (`by`) of every CTA, in slot[...] of all; a barrier of the cluster
    __device__ __forceinline__ const uint64_t (*tell(bool by, uint64_t a, uint64_t b = 0, uint64_t c = 0))[kRowCtas] {
        auto& s = S.slot[turn & 1];
        ++turn;
        if (by)
            for (int i = 0; i < n; ++i) {
                *g.map_shared_rank(&s[0][rank], i) = a;
                *g.map_shared_rank(&s[1][rank], i) = b;
                *g.map_shared_rank(&s[2][rank], i) = c;
            }
        g.sync();
        return s;
    }
};

// Inclusive scan over the block; returns the thread's sum, total the block's.
__device__ __forceinline__ uint64_t block_scan(Shared& S, uint64_t x, uint64_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) S.warp_sum[warp] = x;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += S.warp_sum[w];
        all += S.warp_sum[w];
    }
    total = all;
    return x + before;
}

// A cut of the ranking: the tokens with a key above `key`, and the first `ties` of those with it.
struct Cut {
    uint32_t key;
    uint64_t ties;
};

__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleRowsArgs A) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Shared& S = *reinterpret_cast<Shared*>(smem_raw);
    float* xs = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // the CTAs of the cluster run: their shared memory may be written to behind the wait below
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Cluster cl(S);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / cl.n;
    const int v0 = cl.rank * A.slice, n = max(0, min(A.slice, A.n_vocab - v0));
    // ---- the slice into shared memory, its largest logit ----
    float mx = -INFINITY;
    int arg = INT32_MAX;
    const float* src = A.logits + row * A.stride + v0;
    for (int i = tid; i < n; i += kThreads) {
        float x = src[i] + 0.0f;               // -0 is 0
        if (x != x) x = -INFINITY;
        xs[i] = x;
        if (x > mx) {
            mx = x;
            arg = v0 + i;
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        const float y = __shfl_xor_sync(0xffffffffu, mx, d);
        const int b = __shfl_xor_sync(0xffffffffu, arg, d);
        if (y > mx || (y == mx && b < arg)) {
            mx = y;
            arg = b;
        }
    }
    if (lane == 0) {
        S.warp_u32[warp] = __float_as_uint(mx);
        S.warp_arg[warp] = arg;
    }
    __syncthreads();
    if (tid == 0)
        for (int w = 1; w < kWarps; ++w) {
            const float y = __uint_as_float(S.warp_u32[w]);
            if (y > mx || (y == mx && S.warp_arg[w] < arg)) {
                mx = y;
                arg = S.warp_arg[w];
            }
        }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    {
        const auto s = cl.tell(tid == 0, __float_as_uint(mx), static_cast<uint64_t>(static_cast<uint32_t>(arg)));
        mx = __uint_as_float(static_cast<uint32_t>(s[0][0]));
        arg = static_cast<int>(s[1][0]);
        for (int i = 1; i < cl.n; ++i) {
            const float y = __uint_as_float(static_cast<uint32_t>(s[0][i]));
            if (y > mx) {                      // equal: the earlier slice has the lower index
                mx = y;
                arg = static_cast<int>(s[1][i]);
            }
        }
    }
    const float T = A.temperature ? A.temperature[row] : 1.0f;
    if (mx == -INFINITY || !(T > 0.f)) {       // the same in all CTAs; nobody's memory is read from here on
        if (cl.rank == 0 && tid == 0) A.tokens[row] = mx == -INFINITY ? -1 : arg;
        cl.g.sync();
        return;
    }
    int k = A.top_k ? A.top_k[row] : 0;
    if (k < 0 || k >= A.n_vocab) k = 0;
    const float top_p = A.top_p ? A.top_p[row] : 1.0f;
    float min_p = A.min_p ? A.min_p[row] : 0.0f;
    min_p = min_p > 0.f ? fminf(min_p, 1.0f) : 0.f;
    RowRules R;
    R.mx = mx;
    R.inv_t = 1.0 / static_cast<double>(T);
    R.least = static_cast<double>(min_p) * static_cast<double>(kOne);
    R.reach = (min_p > 0.f ? fminf(kReach, -logf(min_p) + 0.01f) : kReach) * T;
    const int L = A.per_thread, i0 = min(n, tid * L), i1 = min(n, i0 + L);   // this thread's tokens
    // The cut at which the ranking's count (WEIGHT: sum of weights, without the
    // tokens at or below `from`) first reaches `want`, which it does.
    auto search = [&]<bool WEIGHT>(uint64_t want, uint32_t from) -> Cut {
        constexpr int kLimbs = WEIGHT ? 3 : 1;
        uint32_t lo = from + 1, hi = key_of(mx);   // the keys in question
        const float per = R.reach > 0.f ? (kBins - 1) / R.reach : 0.f;
        bool by_logit = true;                      // bins of equal width in logits, then in keys
        int shift = 0;
        auto bin_of = [&](uint32_t key) {
            if (!by_logit) return static_cast<int>((hi - key) >> shift);
            const float d = (mx - of_key(key)) * per;   // falls with the key; inf * 0 and inf - inf: the last, the first
            return d < kBins - 1 ? static_cast<int>(d) : key == key_of(mx) ? 0 : kBins - 1;
        };
        for (;;) {
            for (int i = tid; i < kLimbs * kBins; i += kThreads) (&S.hist[0][0])[i] = 0;
            __syncthreads();
            for (int i = i0; i < i1; ++i) {
                const float x = xs[i];
                const uint32_t key = key_of(x);
                if (key < lo || key > hi) continue;
                if constexpr (WEIGHT) {
                    const uint64_t w = R.weight(x);
                    if (w == 0) continue;
                    const int b = bin_of(key);
                    atomicAdd(&S.hist[0][b], static_cast<uint32_t>(w) & ((1u << kLimb0) - 1));
                    atomicAdd(&S.hist[1][b], static_cast<uint32_t>(w >> kLimb0) & ((1u << kLimb1) - 1));
                    atomicAdd(&S.hist[2][b], static_cast<uint32_t>(w >> (kLimb0 + kLimb1)));
                } else {
                    atomicAdd(&S.hist[0][bin_of(key)], 1u);
                }
            }
            cl.g.sync();
            // this CTA's bins, of all CTAs
            const int per_cta = kBins / cl.n, per_t = (per_cta + kThreads - 1) / kThreads;
            uint64_t mine[kBins / kThreads], sum = 0;
#pragma unroll
            for (int q = 0; q < kBins / kThreads; ++q) {
                mine[q] = 0;
                const int at = tid * per_t + q;
                if (q < per_t && at < per_cta) {
                    const int b = cl.rank * per_cta + at;
                    for (int c = 0; c < cl.n; ++c) {
                        mine[q] += *cl.g.map_shared_rank(&S.hist[0][b], c);
                        if constexpr (WEIGHT) {
                            mine[q] += static_cast<uint64_t>(*cl.g.map_shared_rank(&S.hist[1][b], c)) << kLimb0;
                            mine[q] += static_cast<uint64_t>(*cl.g.map_shared_rank(&S.hist[2][b], c)) << (kLimb0 + kLimb1);
                        }
                    }
                    sum += mine[q];
                }
            }
            uint64_t total;
            uint64_t before = block_scan(S, sum, total) - sum;
            const auto s = cl.tell(tid == 0, total);
            uint64_t base = 0;
            for (int i = 0; i < cl.rank; ++i) base += s[0][i];
            before += base;
            // one thread of one CTA has the bin
            if (tid == 0) S.found[0] = ~0ull;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kBins / kThreads; ++q) {
                if (q < per_t && before < want && before + mine[q] >= want) {
                    S.found[0] = cl.rank * per_cta + tid * per_t + q;
                    S.found[1] = before;
                }
                before += mine[q];
            }
            __syncthreads();
            const auto f = cl.tell(tid == 0, S.found[0], S.found[1]);
            int bin = 0;
            uint64_t so_far = 0;
            for (int i = 0; i < cl.n; ++i)
                if (f[0][i] != ~0ull) {
                    bin = static_cast<int>(f[0][i]);
                    so_far = f[1][i];
                }
            want -= so_far;
            if (by_logit) {
                // the keys of that bin: the largest one, and the smallest, by 32 probes at a time
                auto last_with = [&](auto&& holds, uint32_t a, uint32_t b) {   // holds(a), holds falls: the largest key in [a, b]
                    while (a < b) {
                        const uint64_t range = static_cast<uint64_t>(b) - a;
                        const uint32_t probe = a + static_cast<uint32_t>((range * (lane + 1) + 31) / 32);
                        const uint32_t yes = __popc(__ballot_sync(0xffffffffu, holds(probe)));
                        const uint32_t na = yes == 0 ? a : a + static_cast<uint32_t>((range * yes + 31) / 32);
                        if (yes < 32) b = a + static_cast<uint32_t>((range * (yes + 1) + 31) / 32) - 1;
                        a = na;
                    }
                    return a;
                };
                const uint32_t top = last_with([&](uint32_t key) { return bin_of(key) >= bin; }, lo, hi);
                uint32_t bottom = lo;
                if (bin < kBins - 1 && bin_of(lo) > bin) bottom = last_with([&](uint32_t key) { return bin_of(key) > bin; }, lo, top) + 1;
                lo = bottom;
                hi = top;
                by_logit = false;
            } else {
                const uint32_t h = hi - (static_cast<uint32_t>(bin) << shift);
                lo = max(lo, h - ((1u << shift) - 1));
                hi = h;
            }
            cl.g.sync();                            // all have read the others' bins
            if (lo == hi) return Cut{hi, want};
            shift = max(0, 32 - __clz(hi - lo) - 11);   // (hi - lo) >> shift < kBins
        }
    };
    Cut cut{0, 0};
    const bool ranked = k > 0;
    if (ranked) cut = search.template operator()<false>(static_cast<uint64_t>(k), 0);
    uint64_t tie_w = 0, ties_before = 0;            // weight of a tie; ties before this thread's tokens
    // sum of this thread's kept weights
    auto kept_sum = [&]() {
        uint64_t sum = 0, ties = 0;
        for (int i = i0; i < i1; ++i) {
            const uint32_t key = key_of(xs[i]);
            if (key > cut.key) sum += R.weight(xs[i]);
            else if (key == cut.key) ++ties;
        }
        tie_w = cut.ties ? R.weight(of_key(cut.key)) : 0;
        if (tie_w) {
            uint64_t total;
            ties_before = block_scan(S, ties, total) - ties;
            const auto s = cl.tell(tid == 0, total);
            for (int i = 0; i < cl.rank; ++i) ties_before += s[0][i];
            if (ties_before < cut.ties) sum += min(ties, cut.ties - ties_before) * tie_w;
        }
        return sum;
    };
    uint64_t sum = kept_sum(), in_cta, upto = block_scan(S, sum, in_cta), base = 0, all = 0;
    auto prefix = [&]() {
        const auto s = cl.tell(tid == 0, in_cta);
        base = all = 0;
        for (int i = 0; i < cl.n; ++i) {
            if (i < cl.rank) base += s[0][i];
            all += s[0][i];
        }
    };
    prefix();
    if (top_p < 1.0f) {
        const double t = ceil(static_cast<double>(fmaxf(top_p, 0.f)) * static_cast<double>(all));
        const uint64_t want = min(max(static_cast<uint64_t>(t), static_cast<uint64_t>(1)), all);
        // above the ties of the cut so far, or among them
        const uint64_t tied = cut.ties * tie_w;     // all tied and kept tokens' weight, if k was reached
        const uint64_t above = all - tied;
        if (want <= above) {
            cut = search.template operator()<true>(want, cut.key);
            const uint64_t w = R.weight(of_key(cut.key));
            cut.ties = (cut.ties + w - 1) / w;      // so many of them reach what was left
        } else {
            cut.ties = (want - above + tie_w - 1) / tie_w;
        }
        sum = kept_sum();
        upto = block_scan(S, sum, in_cta);
        prefix();
    }
    const float u = A.uniform[row];
    const uint64_t at = min(static_cast<uint64_t>(static_cast<double>(u > 0.f ? fminf(u, 1.0f) : 0.f) * static_cast<double>(all)), all - 1);
    uint64_t run = base + upto - sum;
    if (run <= at && at < run + sum) {
        uint64_t ties = ties_before;
        int i = i0;
        for (; i < i1; ++i) {
            const uint32_t key = key_of(xs[i]);
            if (key > cut.key) run += R.weight(xs[i]);
            else if (key == cut.key && ties++ < cut.ties) run += tie_w;
            if (run > at) break;
        }
        A.tokens[row] = v0 + i;
    }
    cl.g.sync();                                    // the others may still read this CTA's memory
}

}  // namespace

cudaError_t launch_sample_rows(SampleRowsArgs a, int n_rows, cudaStream_t stream) {
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(sizeof(Shared) + kSampleSlice * sizeof(float)));
    });
    if (e != cudaSuccess) return e;
    int ctas = 1;
    while (ctas < kRowCtas && (n_rows * ctas < 148 || (a.n_vocab + ctas - 1) / ctas > 12800)) ctas *= 2;
    a.slice = (a.n_vocab + ctas - 1) / ctas;
    a.per_thread = ((a.slice + kThreads - 1) / kThreads) | 1;   // odd: no bank conflicts
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(n_rows) * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared) + a.slice * sizeof(float);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel, a);
}

}  // namespace tle
