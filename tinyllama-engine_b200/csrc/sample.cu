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
// exchanged through distributed shared memory.  With slices of at most 12800
// logits two CTAs fit on an SM, and one waits while the other counts; small batches are
// spread over 8 CTAs a row for latency.
//
// Bound by latency: the load, three to six barriers of the cluster, and passes
// over shared memory between them.  256 x 100003, mixed rules, 122 us, 0.8 TB/s of logits (issue 41 %, DRAM
// 13 % busy; no filters 108, without the exponentials 71); 1 x 32000 11.5 us (no filters 7.0).
// Weights in bins by three additions of a third each, 124 and 11.7 us.
// Tried: rereading logits from global memory instead of holding a row 279 us,
// three CTAs an SM (42 registers a thread) 148, 4 CTAs a row 127; lists pulled by rank 0 instead of pushed to it, 130.
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
constexpr int kBins = 2048;                // of a level of a search; in kGroups groups of 32
constexpr int kGroups = kBins / 32;
constexpr int kRowCtas = 8;
constexpr int kList = kThreads;            // tokens of a bin that are ranked one by one
constexpr uint64_t kFew = 128;             // so many tokens in all are ranked without bins
constexpr uint64_t kOne = 1ull << 40;      // the largest weight
constexpr float kReach = 28.6f;            // exp(-kReach) < 2^-41: weights beyond it are 0
static_assert(kGroups * kRowCtas == kThreads && kBins == 4 * kThreads, "a group of a CTA, and 4 bins, per thread");

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^(j / 64) 2^40, j < 64, by the power series of exp.
struct Powers {
    double v[64];
    constexpr Powers() : v{} {
        for (int j = 0; j < 64; ++j) {
            double term = 1.0, sum = 0.0;
            for (int k = 1; k < 24; ++k) {
                sum += term;
                term *= j * (0.69314718055994530942 / 64) / k;
            }
            v[j] = sum * 1099511627776.0;
        }
    }
};
__constant__ const Powers kPowers = Powers();

struct RowRules {
    float mx;              // the largest logit
    float reach;           // logits further below it weigh nothing
    double c;              // 64 log2(e) / T
    uint64_t least;        // min_p 2^40
    const double* powers;  // Powers, in shared memory
    // exp((x - mx) / T) 2^40 = 2^(n / 64) 2^40 e^s with a whole number n and |s| <= ln 2 / 128: four terms of e^s
    // beyond 1 (the next is below 2^-44), the rounding to whole numbers by adding 1.5 * 2^52 and 2^52.
    __device__ __forceinline__ bool in_reach(float x) const { return x - mx >= -reach; }
    __device__ __forceinline__ uint64_t weight(float x) const {
        constexpr double kRound = 6755399441055744.0, kWhole = 4503599627370496.0, kUnit = 0.69314718055994530942 / 64;
        const double d = static_cast<double>(x) - static_cast<double>(mx);
        const double t = fma(d, c, kRound);
        const int n = __double2loint(t);
        const double s = fma(d, c, -(t - kRound));
        double p = fma(s, kUnit * kUnit * kUnit * kUnit / 24, kUnit * kUnit * kUnit / 6);
        p = fma(p, s, kUnit * kUnit / 2);
        p = fma(p, s, kUnit);
        p = fma(p, s, 1.0);
        const double q = powers[n & 63];
        const double w = fma(p, __hiloint2double(__double2hiint(q) + ((n >> 6) << 20), __double2loint(q)), kWhole);
        const uint64_t whole = static_cast<uint64_t>(__double_as_longlong(w)) & 0xfffffffffffffull;
        return in_reach(x) && whole >= least ? whole : 0;   // what is out of reach has come out as anything
    }
};

struct alignas(16) Shared {                // the slice lies behind it
    union {
        uint32_t hist[2][kBins];           // a bin's count; or its sum of weights, low and high 32 bits
        struct {                           // once nobody reads the bins any more:
            uint64_t weight[kList];        // the weights and keys of the bin's tokens, of all CTAs
            uint32_t key[kList];
        };
    };
    union {
        uint64_t group[kRowCtas][kGroups]; // sums of 32 bins, of each CTA of the cluster
        uint32_t fine[2 * kRowCtas][32];   // then the bins of one group
    };
    uint32_t list[2][kList];               // of two searches in turn: this CTA's keys of the bin in question
    uint32_t count[2][kRowCtas];           // how many each CTA has
    uint32_t mine;
    uint32_t n_last[2], last_key[kFew], last_at[kFew];   // rank 0: what is left of the row, if that is few
    uint64_t slot[2][2][kRowCtas];         // what the CTAs of the cluster told each other, by turns
    double powers[64];
    uint64_t warp_sum[kWarps];
    uint32_t warp_ties[kWarps];
    uint64_t found;
    uint32_t found_key;
    float warp_max[kWarps];
};

// The CTA's part of the exchanges.
struct Cluster {
    cg::cluster_group g;
    Shared& S;
    int rank, n, turn;
    __device__ __forceinline__ Cluster(Shared& s) : g(cg::this_cluster()), S(s), turn(0) {
        rank = static_cast<int>(g.block_rank());
        n = static_cast<int>(g.num_blocks());
    }
    // a, b, the same in all threads of a CTA, to slot[..][this rank] of all CTAs; a barrier of the cluster
    __device__ __forceinline__ const uint64_t (*tell(uint64_t a, uint64_t b = 0))[kRowCtas] {
        auto& s = S.slot[turn & 1];
        ++turn;
        if (static_cast<int>(threadIdx.x) < n) {
            *g.map_shared_rank(&s[0][rank], threadIdx.x) = a;
            *g.map_shared_rank(&s[1][rank], threadIdx.x) = b;
        }
        g.sync();
        return s;
    }
};

__device__ __forceinline__ uint64_t warp_scan(uint64_t x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    return x;
}
// A cut of the ranking: the tokens with a key above `key`, and the first `ties` of those with it.
struct Cut {
    uint32_t key;
    uint64_t ties;
};

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleRowsArgs A) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Shared& S = *reinterpret_cast<Shared*>(smem_raw);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // the CTAs of the cluster run: their shared memory may be written to behind the wait below
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Cluster cl(S);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / cl.n;
    if (tid < 64) S.powers[tid] = kPowers.v[tid];
    if (tid < 2) S.n_last[tid] = 0;
    for (int i = tid; i < 2 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(S.hist)[i] = make_uint4(0, 0, 0, 0);
    const int v0 = cl.rank * A.slice, n = max(0, min(A.slice, A.n_vocab - v0));
    // ---- the slice into shared memory, its largest logit ----
    const float* src = A.logits + row * A.stride + v0;
    const int head = min(n, static_cast<int>((-(reinterpret_cast<uintptr_t>(src) >> 2)) & 3u));   // before the first 16-byte boundary
    float* xs = reinterpret_cast<float*>(smem_raw + sizeof(Shared)) + ((4 - head) & 3);              // aligned as the row is
    float mx = -INFINITY;
    auto take = [&](float x) {
        x = fminf(fmaxf(x + 0.0f, -INFINITY), 3.4028234e38f);   // -0 is 0, NaN -inf, +inf the largest number
        mx = fmaxf(mx, x);
        return x;
    };
    {
        const int body = (n - head) / 4;
        const float4* from = reinterpret_cast<const float4*>(src + head);
        float4* to = reinterpret_cast<float4*>(xs + head);
        constexpr int kAhead = 8;
        for (int i0 = tid; i0 < body; i0 += kAhead * kThreads) {
            float4 x[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
                if (i0 + q * kThreads < body) x[q] = from[i0 + q * kThreads];
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
                if (i0 + q * kThreads < body) to[i0 + q * kThreads] = make_float4(take(x[q].x), take(x[q].y), take(x[q].z), take(x[q].w));
        }
        if (tid < head) xs[tid] = take(src[tid]);
        const int tail = head + 4 * body;
        if (tail + tid < n && tid < 4) xs[tail + tid] = take(src[tail + tid]);
    }
    float T = A.temperature ? A.temperature[row] : 1.0f;
    T = T > 1e30f ? 1e30f : T;                 // so that differences of logits stay within reach or below it
    int k = A.top_k ? A.top_k[row] : 0;
    if (k >= A.n_vocab) k = 0;
    const float top_p = A.top_p ? A.top_p[row] : 1.0f;
    float min_p = A.min_p ? A.min_p[row] : 0.0f;
    min_p = min_p > 0.f ? fminf(min_p, 1.0f) : 0.f;
    const float u = A.uniform[row];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if (lane == 0) S.warp_max[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, S.warp_max[w]);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    {
        const auto s = cl.tell(__float_as_uint(mx));
        for (int i = 0; i < cl.n; ++i) mx = fmaxf(mx, __uint_as_float(static_cast<uint32_t>(s[0][i])));
    }
    if (mx == -INFINITY) {                     // the same in all CTAs
        if (cl.rank == 0 && tid == 0) A.tokens[row] = -1;
        return;
    }
    // the weight that top-p asks for of a sum, and the place of the drawn number in one
    auto want_of_p = [&](uint64_t all) {
        const double t = ceil(static_cast<double>(fmaxf(top_p, 0.f)) * static_cast<double>(all));
        return min(max(static_cast<uint64_t>(t), static_cast<uint64_t>(1)), all);
    };
    auto number_of = [&](uint64_t all) {
        return min(static_cast<uint64_t>(static_cast<double>(u > 0.f ? fminf(u, 1.0f) : 0.f) * static_cast<double>(all)), all - 1);
    };
    // a part of the slice for each warp, in order; `have` of its tokens are left in x and id
    const int part = (A.slice + kWarps - 1) / kWarps, p0 = min(n, warp * part);
    int have = min(n - p0, part);
    float* x_of = xs + p0;
    if (!(T > 0.f)) {                          // the first of the largest
        int at = INT32_MAX;
        for (int i = lane; i < have; i += 32)
            if (x_of[i] == mx) at = min(at, v0 + p0 + i);
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) S.warp_sum[warp] = at;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) at = min(at, static_cast<int>(S.warp_sum[w]));
        const auto s = cl.tell(at);
        for (int i = 0; i < cl.n; ++i) at = min(at, static_cast<int>(s[0][i]));
        if (cl.rank == 0 && tid == 0) A.tokens[row] = at;
        return;
    }
    RowRules R;
    R.mx = mx;
    R.c = 64 * 1.4426950408889634 / static_cast<double>(T);
    R.least = static_cast<uint64_t>(ceil(static_cast<double>(min_p) * static_cast<double>(kOne)));
    R.powers = S.powers;
    R.reach = (min_p > 0.f ? fminf(kReach, -logf(min_p) + 0.01f) : kReach) * T;
    // Drops tokens of the warp, the others stay in place and in order; id is a token's place in the warp's part.
    // stays(logit, whether there is one); four at a time: a row of 32000 with top-k 11.7 us, one at a time 12.0 us.
    uint16_t* id_of = reinterpret_cast<uint16_t*>(smem_raw + sizeof(Shared) + 16 + A.slice * sizeof(float)) + p0;
    bool whole = true;                         // nothing has been dropped: ids are not written yet
    auto keep = [&](auto&& stays) {
        constexpr int kAhead = 4;
        int out = 0;
        for (int i0 = 0; i0 < have; i0 += 32 * kAhead) {
            float x[kAhead];
            int id[kAhead];
            uint32_t set[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int i = i0 + 32 * q + lane;
                x[q] = i < have ? x_of[i] : 0.f;
                id[q] = whole ? i : i < have ? id_of[i] : 0;
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) set[q] = __ballot_sync(0xffffffffu, stays(x[q], i0 + 32 * q + lane < have));
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                if (set[q] >> lane & 1) {
                    const int to = out + __popc(set[q] & ((1u << lane) - 1));
                    x_of[to] = x[q];
                    id_of[to] = static_cast<uint16_t>(id[q]);
                }
                out += __popc(set[q]);
            }
            __syncwarp();
        }
        have = out;
        whole = false;
    };
    uint64_t left = ~0ull;                     // tokens left in all CTAs at most, once something was dropped
    // The tokens left to rank 0, as far as there is room (try 0 or 1), before a barrier of the cluster.
    auto hand_over = [&](int turn) {
        if (have == 0) return;
        uint32_t to = 0;
        if (lane == 0) to = atomicAdd(cl.g.map_shared_rank(&S.n_last[turn], 0), static_cast<uint32_t>(have));
        to = __shfl_sync(0xffffffffu, to, 0);
        for (int i = lane; i < have && to + i < kFew; i += 32) {
            *cl.g.map_shared_rank(&S.last_key[to + i], 0) = key_of(x_of[i]);
            *cl.g.map_shared_rank(&S.last_at[to + i], 0) = static_cast<uint32_t>(v0 + p0 + id_of[i]);
        }
    };
    // The row's token from its last n <= kFew tokens, by rank 0: everything by comparing all pairs, four threads a token.
    auto finish = [&](uint32_t n) {
        static_assert(4 * kFew == kThreads, "four threads a token");
        uint64_t* kept = S.weight;             // weights of the tokens that pass the filters so far
        uint64_t* kept2 = S.weight + kFew;
        const uint32_t i = tid >> 2, key = i < n ? S.last_key[i] : 0, at = i < n ? S.last_at[i] : 0;
        const uint64_t w = i < n ? R.weight(of_key(key)) : 0;
        auto sum4 = [](auto x) {
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            return x + __shfl_xor_sync(0xffffffffu, x, 2);
        };
        auto before = [&](uint32_t j) { return S.last_key[j] > key || (S.last_key[j] == key && S.last_at[j] < at); };
        uint32_t rank = 0;
        for (uint32_t j = tid & 3; j < n; j += 4) rank += before(j);
        rank = sum4(rank);
        __syncthreads();                       // the weights' place may have held something else
        if ((tid & 3) == 0) kept[i] = k == 0 || rank < static_cast<uint32_t>(k) ? w : 0;
        __syncthreads();
        uint64_t above = 0, all = 0;
        for (uint32_t j = tid & 3; j < n; j += 4) {
            above += before(j) ? kept[j] : 0;
            all += kept[j];
        }
        above = sum4(above);
        all = sum4(all);
        if ((tid & 3) == 0) kept2[i] = top_p < 1.0f && above >= want_of_p(all) ? 0 : kept[i];
        __syncthreads();
        uint64_t run = 0, sum = 0;
        for (uint32_t j = tid & 3; j < n; j += 4) {
            run += S.last_at[j] < at ? kept2[j] : 0;
            sum += kept2[j];
        }
        run = sum4(run);
        sum = sum4(sum);
        const uint64_t drawn = number_of(sum);
        if ((tid & 3) == 0 && i < n && run <= drawn && drawn < run + kept2[i]) A.tokens[row] = static_cast<int32_t>(at);
    };
    int searches = 0;
    bool clean = true;                         // the bins are zeros
    // The cut at which the ranking's count (WEIGHT: sum of weights) within reach (the others weigh nothing) with a
    // key above `from` first reaches want_of(its sum over all of them).  A want of 0, or of more than there is: no cut.  Cut::ties is then
    // what is to be reached among the tokens of Cut::key.  Tokens below the cut may be dropped.
    auto search = [&]<bool WEIGHT>(uint32_t from, auto&& want_of, Cut& cut) -> bool {
        constexpr int kLimbs = WEIGHT ? 2 : 1;
        const int turn = searches++ & 1;
        uint32_t lo = from + 1, hi = key_of(mx);   // the keys in question
        const float per = R.reach > 0.f ? fminf(kBins / R.reach, 3e38f) : 0.f;   // finite: the largest logit's bin is 0
        uint64_t want = 0;
        int shift = 0;
        // level 0: bins of equal width in logits; then of keys.  Falls with the key.
        auto by_logit = [&](float x) {
            const float d = (mx - x) * per;
            return d < kBins ? static_cast<int>(d) : kBins - 1;
        };
        auto in = [&](float x, uint32_t key) { return key >= lo && key <= hi && R.in_reach(x); };
        // this CTA's keys to list one by one: to all CTAs' knowledge, then those of all with their weights
        // in S.key and S.weight; returns how many there are (more than kList: no list)
        auto gather = [&]() {
            __syncthreads();
            if (tid < cl.n) *cl.g.map_shared_rank(&S.count[turn][cl.rank], tid) = S.mine;
            cl.g.sync();
            const uint32_t me = tid;
            uint32_t all = 0, key = 0;
            for (int c = 0; c < cl.n; ++c) {
                const uint32_t m = S.count[turn][c];
                if (me >= all && me - all < min(m, static_cast<uint32_t>(kList))) key = *cl.g.map_shared_rank(&S.list[turn][me - all], c);
                all += m;
            }
            if (all <= kList) {
                S.key[tid] = key;
                S.weight[tid] = me >= all ? 0 : WEIGHT ? R.weight(of_key(key)) : 1;
            }
            __syncthreads();
            return all;
        };
        // the listed key at which `want` is reached, by as many threads a key as there are
        auto rank = [&](uint32_t all) {
            const int bits = all <= 32 ? 4 : all <= 64 ? 3 : all <= 128 ? 2 : all <= 256 ? 1 : 0;
            const uint32_t me = tid >> bits, key = me < all ? S.key[me] : 0;
            uint64_t above = 0, with = 0;
            for (uint32_t q = tid & ((1 << bits) - 1); q < all; q += 1 << bits) {
                const uint32_t kq = S.key[q];
                const uint64_t w = S.weight[q];
                above += kq > key ? w : 0;
                with += kq >= key ? w : 0;
            }
            for (int d = 1; d < 1 << bits; d *= 2) {
                above += __shfl_xor_sync(0xffffffffu, above, d);
                with += __shfl_xor_sync(0xffffffffu, with, d);
            }
            if (me < all && above < want && with >= want) {   // tokens of one key: they write the same
                S.found = want - above;
                S.found_key = key;
            }
            __syncthreads();
            cut = Cut{S.found_key, S.found};
        };
        auto list_key = [&](uint32_t key) {
            const uint32_t to = atomicAdd(&S.mine, 1u);
            if (to < kList) S.list[turn][to] = key;
        };
        for (int level = 0;; ++level) {
            auto bin_of = [&](float x, uint32_t key) { return level == 0 ? by_logit(x) : static_cast<int>((hi - key) >> shift); };
            __syncthreads();
            if (!clean)
                for (int i = tid; i < kLimbs * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(S.hist)[i] = make_uint4(0, 0, 0, 0);
            clean = false;
            if (tid == 0) S.mine = 0;
            __syncthreads();
            for (int i = lane; i < have; i += 32) {
                const float x = x_of[i];
                const uint32_t key = key_of(x);
                if (!in(x, key)) continue;
                const int b = bin_of(x, key);
                if constexpr (WEIGHT) {
                    const uint64_t w = R.weight(x);
                    if (w == 0) continue;
                    // most weights are below 2^32, 1 / 256 of the largest: one addition
                    const uint32_t low = static_cast<uint32_t>(w), was = atomicAdd(&S.hist[0][b], low);
                    const uint32_t high = static_cast<uint32_t>(w >> 32) + (was + low < low);
                    if (high) atomicAdd(&S.hist[1][b], high);
                } else {
                    atomicAdd(&S.hist[0][b], 1u);
                }
            }
            __syncthreads();
            auto both = [](uint32_t low, uint32_t high) { return low + (static_cast<uint64_t>(high) << 32); };
            // groups of 32 bins: 8 threads each, to all CTAs
            uint64_t sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int b = tid / 8 * 32 + tid % 8 + 8 * q;
                sum += WEIGHT ? both(S.hist[0][b], S.hist[1][b]) : S.hist[0][b];
            }
#pragma unroll
            for (int d = 1; d < 8; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane % 8 < cl.n) *cl.g.map_shared_rank(&S.group[cl.rank][tid / 8], lane % 8) = sum;
            cl.g.sync();
            // the group in which want is reached, by every warp for itself
            uint64_t g0 = 0, g1 = 0;
            for (int c = 0; c < cl.n; ++c) {
                g0 += S.group[c][2 * lane];
                g1 += S.group[c][2 * lane + 1];
            }
            const uint64_t upto = warp_scan(g0 + g1);
            __syncthreads();                   // read by all: its place is the group's bins'
            if (level == 0) {
                const uint64_t all = __shfl_sync(0xffffffffu, upto, 31);
                want = want_of(all);
                if (want == 0 || want > all) {
                    cl.g.sync();               // all have read the groups
                    return false;
                }
            }
            const int first = __ffs(__ballot_sync(0xffffffffu, upto >= want)) - 1;
            const uint64_t before2 = __shfl_sync(0xffffffffu, upto - g0 - g1, first), half = __shfl_sync(0xffffffffu, g0, first);
            const bool second = before2 + half < want;
            const int group = 2 * first + second;
            uint64_t before = before2 + (second ? half : 0);
            for (int e = warp; e < kLimbs * cl.n; e += kWarps)
                S.fine[e][lane] = *cl.g.map_shared_rank(&S.hist[e % kLimbs][32 * group + lane], e / kLimbs);
            __syncthreads();
            uint64_t f = 0;
            for (int c = 0; c < cl.n; ++c)
                f += WEIGHT ? both(S.fine[2 * c][lane], S.fine[2 * c + 1][lane]) : S.fine[c][lane];
            const uint64_t fine_upto = before + warp_scan(f);
            const int at = __ffs(__ballot_sync(0xffffffffu, fine_upto >= want)) - 1;
            want -= __shfl_sync(0xffffffffu, fine_upto - f, at);
            const int bin = 32 * group + at;
            if (!WEIGHT && level == 0) left = __shfl_sync(0xffffffffu, fine_upto, at);   // up to and with the bin
            if (level > 0) {
                const uint32_t h = hi - (static_cast<uint32_t>(bin) << shift);
                lo = max(lo, h - ((1u << shift) - 1));
                hi = h;
                if (lo == hi) {
                    cl.g.sync();               // all have read the bins
                    cut = Cut{hi, want};
                    return true;
                }
            }
            if (!WEIGHT && level == 0 && left <= kFew) {   // what the row's token will be one of
                keep([&](float x, bool there) { return there && R.in_reach(x) && by_logit(x) <= bin; });
                hand_over(1);
                cl.g.sync();
                return true;
            }
            // ---- the bin's tokens, if they are few, ranked one by one; those behind it dropped ----
            if (level == 0) {
                keep([&](float x, bool there) {
                    const int b = by_logit(x);
                    const bool stays = there && b <= bin && R.in_reach(x);
                    if (stays && b == bin) {
                        const uint32_t key = key_of(x);
                        if (in(x, key)) list_key(key);
                    }
                    return stays;
                });
            } else {
                for (int i = lane; i < have; i += 32) {
                    const float x = x_of[i];
                    const uint32_t key = key_of(x);
                    if (in(x, key)) list_key(key);
                }
            }
            const uint32_t all = gather();
            if (all <= kList) {
                rank(all);
                return true;
            }
            if (level == 0) {
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
                const uint32_t top = last_with([&](uint32_t q) { return by_logit(of_key(q)) >= bin; }, lo, hi);
                if (by_logit(of_key(lo)) > bin) lo = last_with([&](uint32_t q) { return by_logit(of_key(q)) > bin; }, lo, top) + 1;
                hi = top;
            }
            shift = max(0, 32 - __clz(hi - lo) - 11);   // (hi - lo) >> shift < kBins
        }
    };
    // where min-p leaves a narrow range, what is outside goes first
    if (min_p > 0.f) {
        keep([&](float x, bool there) { return there && R.in_reach(x); });
        hand_over(0);
        __syncthreads();
        if (lane == 0) S.warp_sum[warp] = have;
        __syncthreads();
        uint64_t mine = 0;
        for (int w = 0; w < kWarps; ++w) mine += S.warp_sum[w];
        const auto s = cl.tell(mine);
        left = 0;
        for (int i = 0; i < cl.n; ++i) left += s[0][i];
        if (left <= kFew) {
            if (cl.rank == 0) finish(static_cast<uint32_t>(left));
            return;
        }
    }
    Cut cut{0, 0};
    if (k > 0 && static_cast<uint64_t>(k) < left) {
        left = ~0ull;
        search.template operator()<false>(0, [&](uint64_t) { return static_cast<uint64_t>(k); }, cut);
        if (left <= kFew) {
            if (cl.rank == 0) finish(static_cast<uint32_t>(left));
            return;
        }
    }
    if (top_p < 1.0f) {
        const uint64_t tie_w = cut.ties ? R.weight(of_key(cut.key)) : 0, tied = cut.ties * tie_w;
        uint64_t in_ties = 0;                       // what is left to be reached among the ties of the cut so far
        Cut c2{0, 0};
        const bool above = search.template operator()<true>(
            cut.key,
            [&](uint64_t above) -> uint64_t {
                const uint64_t all = above + tied;
                const uint64_t want = want_of_p(all);
                in_ties = want > above ? want - above : 0;
                return want > above ? 0 : want;
            },
            c2);
        if (above) {
            const uint64_t w = R.weight(of_key(c2.key));
            cut = Cut{c2.key, (c2.ties + w - 1) / w};   // so many of them reach what was left
        } else {
            cut.ties = (in_ties + tie_w - 1) / tie_w;
        }
    }
    // ---- the running sum of kept weights, by index: warps' sums, then the warp's in which the number lies ----
    const uint64_t tie_w = cut.ties ? R.weight(of_key(cut.key)) : 0;
    uint64_t sum = 0;
    uint32_t ties = 0;
    if (cut.key == 0) {
#pragma unroll 4
        for (int i = lane; i < have; i += 32) sum += R.weight(x_of[i]);
    } else {
        for (int i = lane; i < have; i += 32) {
            const float x = x_of[i];
            const uint32_t key = key_of(x);
            if (key > cut.key) sum += R.weight(x);
            else if (key == cut.key) ++ties;
        }
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    ties = __reduce_add_sync(0xffffffffu, ties);
    __syncthreads();
    if (lane == 0) {
        S.warp_sum[warp] = sum;
        S.warp_ties[warp] = ties;
    }
    __syncthreads();
    uint64_t cta_sum = 0, cta_ties = 0, run = 0, tie = 0;   // run, tie: before this warp's tokens
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) {
            run = cta_sum;
            tie = cta_ties;
        }
        cta_sum += S.warp_sum[w];
        cta_ties += S.warp_ties[w];
    }
    const auto s = cl.tell(cta_sum, cta_ties);
    uint64_t all = 0, ties_all = 0;
    for (int i = 0; i < cl.n; ++i) {
        if (i < cl.rank) {
            run += s[0][i];
            tie += s[1][i];
        }
        all += s[0][i];
        ties_all += s[1][i];
    }
    all += min(ties_all, cut.ties) * tie_w;
    const uint64_t at = number_of(all);
    const uint64_t end = run + sum + min(tie + ties, cut.ties) * tie_w;
    run += min(tie, cut.ties) * tie_w;
    if (run > at || at >= end) return;
    for (int i = 0; i < have; i += 32) {
        const float x = i + lane < have ? x_of[i + lane] : -INFINITY;
        const uint32_t key = key_of(x);
        const bool is_tie = i + lane < have && key == cut.key;
        const uint32_t set = __ballot_sync(0xffffffffu, is_tie);
        uint64_t w = 0;
        if (i + lane < have && key > cut.key) w = R.weight(x);
        if (is_tie && tie + __popc(set & ((1u << lane) - 1)) < cut.ties) w = tie_w;
        tie += __popc(set);
        const uint64_t upto = run + warp_scan(w);
        const uint32_t over = __ballot_sync(0xffffffffu, upto > at);
        if (over) {
            if (lane == __ffs(over) - 1) A.tokens[row] = v0 + p0 + (whole ? i + lane : id_of[i + lane]);
            return;
        }
        run = __shfl_sync(0xffffffffu, upto, 31);
    }
}

}  // namespace

cudaError_t launch_sample_rows(SampleRowsArgs a, int n_rows, cudaStream_t stream) {
    constexpr int kExtra = sizeof(Shared) + 16;     // and the alignment of a slice
    constexpr int kToken = sizeof(float) + sizeof(uint16_t);
    static_assert(sizeof(Shared) % 16 == 0, "16-byte pieces of the slice");
    static_assert(kExtra + kSampleSlice * kToken <= 232448, "shared memory of one SM");
    static PerDeviceOnce once;
    cudaError_t e = once.run([&](int) {
        return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kExtra + kSampleSlice * kToken);
    });
    if (e != cudaSuccess) return e;
    // Several CTAs a row while SMs are idle, as long as a slice is worth a barrier (1 x 32000 8 CTAs 11.5 us, 4 13.7, 1
    // 27; 16 x 10000 4 CTAs 14.0 us, 8 15.9, 2 15.3), and so that two CTAs fit on an SM (256 x 100003 without filters
    // 108 us, with slices of 25001 129; top-p alone 254 and 240).
    int ctas = 1;
    for (; ctas < kRowCtas; ctas *= 2) {
        const int slice = (a.n_vocab + ctas - 1) / ctas;
        if (slice <= 12800 && (slice <= 3000 || n_rows * ctas >= 148)) break;
    }
    a.slice = (a.n_vocab + ctas - 1) / ctas;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(n_rows) * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kExtra + a.slice * kToken;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sample_kernel, a);
}

}  // namespace tle
