// cache8.cu -- append by rules (RMS norm of q and k heads, rope layouts) into
// fp32, bf16 and 8-bit pages, and 8-bit pages read back.
//
// For a head x[0..63] of token position p:
//   y = x / sqrt(mean(x^2) + eps) * w                              (norm, if given)
//   (y'_a, y'_b) = (y_a c - y_b s, y_a s + y_b c),  c, s = factor (cos, sin)(fl32(p f_i))
// for the pairs i < rotary_dim / 2, (a, b) = (2i, 2i + 1) or (i, i + rotary_dim / 2).
//
// 8-bit pages.  A head's row is 64 whole numbers n in -127..127 and a byte b:
// the values n 2^(b - 127), with 2^(b - 127) the smallest power of two for
// which max|y| <= 127 2^(b - 127) (1 <= b <= 248, so that n 2^(b - 127) is finite:
// numbers above 127 2^121 become that) and n the nearest whole number, ties to even.  A power of two, because n 2^(b - 127) is then a bf16 number
// exactly (8 bits): products with it are exact on the tensor cores, and rows
// read back as bf16 or fp32 are the stored ones.  A scale of more bits would be
// up to twice as fine (max|y| / 127 against 2^ceil(log2(max|y| / 127))), but every reader would
// round its product.  Rows with an infinity or NaN: b = 255 and n = 0, which
// is 0 * inf = NaN for every reader.
#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "chunk.cuh"
#include "common.cuh"
#include "kernels.h"

namespace tle {

namespace {

// ---- append -----------------------------------------------------------------
// A warp takes a token, or an equal part of its pieces where there are few
// tokens.  A piece is one load of a warp: four q heads, k heads or v heads, 8 lanes
// a head, each with two groups of 4 elements
// -- with the half layout the two that its pairs lie in, otherwise one of each
// half of the head, so that a load is of whole sectors -- so that a pair's elements meet in a lane, and the norm's sum and the largest
// value of a head are reductions over its lanes.  Sines and cosines are found once a token.
// HBM-bound: kBatch pieces are in flight, the first ones while the token's place is looked up.  Measured: 4096 tokens of 32 + 4 + 4
// heads, bf16, into bf16 pages 9.9 us, 4.2 TB/s; 16 x 1501 of 16 + 8 + 8 heads, bf16, normed, into 8-bit pages 34.7 us,
// 3.8 TB/s (a third of the instructions are the shuffles and roundings of norms and scales); 32 x 1 3.5 us, a launch.
// Blocks of 32 threads, all of a token's pieces in flight, or parts of two pieces were slower.
constexpr int kThreads = 64;
// Below so many tokens their heads are spread over several warps: 1 x 600 5.4 us (one warp a token 8.2), 1 x 2000 fp32
// 10.6 us (15.2); twice as many, 1 x 4096 bf16 10.7 us (9.8).
constexpr int kWarps = 148 * 32;

template <int LANES>
__device__ __forceinline__ float sum_over(float x) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}
template <int LANES>
__device__ __forceinline__ float max_over(float x) {   // keeps a NaN
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) x = fmax3(x, __shfl_xor_sync(0xffffffffu, x, d), 0.f);
    return x;
}

// The byte b of a row whose largest magnitude is `most`: 127 = 1.984375 * 2^6.
__device__ __forceinline__ int scale_byte(float most) {
    const uint32_t u = __float_as_uint(most);
    const int b = static_cast<int>(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return (u >> 23) == 255u ? 255 : min(max(b, 1), 248);
}

// A group of 4 activations as numbers.
constexpr int GE = 4;
template <class Act>
using Group = std::conditional_t<sizeof(Act) == 4, uint4, uint2>;
__device__ __forceinline__ void group_of(uint4 u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void group_of(uint2 u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x << 16);
    f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16);
    f[3] = __uint_as_float(u.y & 0xffff0000u);
}
// (4-byte aligned)
__device__ __forceinline__ void load_norm(const float* p, float (&f)[4]) {
    if ((reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        f[0] = x.x;
        f[1] = x.y;
        f[2] = x.z;
        f[3] = x.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = p[e];
    }
}
// Codes of a group, |f| inv <= 127: adding 1.5 * 2^23 rounds to whole numbers, whose low bytes are the codes.
__device__ __forceinline__ uint32_t code_bits(float y, float inv) { return __float_as_uint(fmaf(y, inv, 12582912.0f)); }
__device__ __forceinline__ void store_codes(int8_t* p, const float (&f)[4], float inv) {
    *reinterpret_cast<uint32_t*>(p) =
        __byte_perm(__byte_perm(code_bits(f[0], inv), code_bits(f[1], inv), 0x0040),
                    __byte_perm(code_bits(f[2], inv), code_bits(f[3], inv), 0x0040), 0x5410);
}

template <class Act, class Pool, bool HALF, bool NORM, int kBatch>
__global__ void __launch_bounds__(kThreads) append_rules_kernel(const __grid_constant__ AppendRulesArgs R, int parts) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr bool kBits8 = sizeof(Pool) == 1;
    constexpr int LPH = HD / (2 * GE);
    constexpr int HPW = 32 / LPH;
    const AppendArgs& A = R.a;
    const int lane = threadIdx.x & 31, hl = lane % LPH, sub = lane / LPH;
    // the warp's token, in a form that the compiler knows to be the same in all lanes
    const unsigned w = __reduce_max_sync(0xffffffffu, blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5));
    const int64_t tok = parts == 1 ? w : w / parts;
    if (tok >= A.n_tokens) return;
    const int part = parts == 1 ? 0 : static_cast<int>(w % parts);
    // this lane's two groups of a head: elements e1 .., e2 ..
    const int hg = R.half / GE;
    // those that are not turned: a head's rest in halves, or, of bf16, two in a row, which takes 8 registers less (16 x 1501
    // normed into 8 bits and read back 46.1 and 49.1 us)
    constexpr bool kNext = HALF && sizeof(Act) == 2;
    const int g1 = HALF && hl >= hg ? (kNext ? 2 * hl : hl + hg) : hl, g2 = HALF && hl < hg ? hl + hg : kNext ? g1 + 1 : hl + LPH;
    const int e1 = g1 * GE, e2 = g2 * GE;
    const bool turned = A.rotate && (HALF ? hl < hg : e1 < 2 * R.half);   // the first group; the second one:
    const bool turned2 = HALF ? turned : A.rotate && e2 < 2 * R.half;
    const int nq = (A.n_head + HPW - 1) / HPW, nk = (A.n_head_kv + HPW - 1) / HPW, pieces = nq + 2 * nk;
    const int j_first = parts == 1 ? 0 : part * pieces / parts, j_end = parts == 1 ? pieces : (part + 1) * pieces / parts;
    const Act* q = static_cast<const Act*>(A.q) + tok * A.q_stride;
    const Act* k = static_cast<const Act*>(A.k) + tok * A.k_stride;
    const Act* v = static_cast<const Act*>(A.v) + tok * A.v_stride;
    Group<Act> x[kBatch][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int j = j0 + b, base = j < nq ? 0 : j < nq + nk ? nq : nq + nk;
            const int h = (j - base) * HPW + sub;
            const Act* src = (j < nq ? q : j < nq + nk ? k : v) + h * HD;
            const bool in = j < j_end && h < (j < nq ? A.n_head : A.n_head_kv);
            x[b][0] = in ? *reinterpret_cast<const Group<Act>*>(src + e1) : Group<Act>{};
            x[b][1] = in ? *reinterpret_cast<const Group<Act>*>(src + e2) : Group<Act>{};
        }
    };
    load(j_first);
    // before its records: another plan's descriptor may end before this one's do
    if (A.d.hdr->id != A.plan_id) {
        if (lane == 0) record_error(A.err, kErrBadDesc);
        return;
    }
    const ChunkTok tk = A.d.toks[tok];
    // the token's row in the pools: its first head there, and from head to head
    const int page_rows = 1 << A.page_shift, r_in = tk.pos & (page_rows - 1);
    const size_t step = kBits8 ? static_cast<size_t>(page_rows) * HD : HD;
    size_t row = 0;
    bool have = false;
    const int id = A.d.seqs[tk.seq].pages[tk.pos >> A.page_shift];
    if (static_cast<unsigned>(id) < static_cast<unsigned>(A.pool_pages)) {
        have = true;
        row = kBits8 ? ((static_cast<size_t>(id) * A.n_head_kv) << A.page_shift) + r_in
                     : ((static_cast<size_t>(id) << A.page_shift) + r_in) * A.n_head_kv;
    } else if (lane == 0) {
        record_error(A.err, kErrBadPage);
    }
    float cs[GE], sn[GE];   // of this lane's pairs
    if (A.rotate) {
        float s1 = 0.f, c1 = 1.f;
        if (lane < R.half) sincosf(static_cast<float>(tk.pos) * A.inv_freq[lane], &s1, &c1);
        s1 *= R.factor;
        c1 *= R.factor;
#pragma unroll
        for (int e = 0; e < GE; ++e) {
            const int i = HALF ? e1 + e : e < GE / 2 ? e1 / 2 + e : e2 / 2 + e - GE / 2;
            cs[e] = __shfl_sync(0xffffffffu, c1, i & 31);
            sn[e] = __shfl_sync(0xffffffffu, s1, i & 31);
        }
    }
    for (int j0 = j_first;;) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int j = j0 + b;
            if (j >= j_end) break;   // the same in all lanes, as what kind of heads it is
            const bool is_q = j < nq, is_v = j >= nq + nk;
            const int h = (j - (is_q ? 0 : is_v ? nq + nk : nq)) * HPW + sub;
            const bool there = h < (is_q ? A.n_head : A.n_head_kv);
            float y[GE], z[GE];
            group_of(x[b][0], y);
            group_of(x[b][1], z);
            if (!is_v) {
                if constexpr (NORM) {
                    const float* norm = is_q ? R.q_norm : R.k_norm;
                    if (norm) {
                        float ss = 0.f;
#pragma unroll
                        for (int e = 0; e < GE; ++e) ss = fmaf(y[e], y[e], fmaf(z[e], z[e], ss));
                        const float f = rsqrtf(sum_over<LPH>(ss) * (1.0f / HD) + R.eps);
                        float ny[GE], nz[GE];
                        load_norm(norm + e1, ny);
                        load_norm(norm + e2, nz);
#pragma unroll
                        for (int e = 0; e < GE; ++e) {
                            y[e] = y[e] * f * ny[e];
                            z[e] = z[e] * f * nz[e];
                        }
                    }
                }
                if (turned) {
#pragma unroll
                    for (int e = 0; e < GE; ++e) {
                        if (!HALF && e >= GE / 2 && !turned2) break;
                        float& a = HALF ? y[e] : e < GE / 2 ? y[2 * e] : z[2 * e - GE];
                        float& c = HALF ? z[e] : e < GE / 2 ? y[2 * e + 1] : z[2 * e - GE + 1];
                        const float a0 = a, c0 = c;
                        a = a0 * cs[e] - c0 * sn[e];
                        c = a0 * sn[e] + c0 * cs[e];
                    }
                }
            }
            if (is_q) {
                if (there) {
                    Act* qo = static_cast<Act*>(A.q_out) + (tok * A.n_head + h) * HD;
                    store4(qo + e1, y);
                    store4(qo + e2, z);
                }
                continue;
            }
            Pool* to = static_cast<Pool*>(is_v ? A.value_pool : A.key_pool) + row * HD + h * step;
            if constexpr (kBits8) {
                float most = 0.f;
#pragma unroll
                for (int e = 0; e < GE; ++e) most = fmax3(most, fabsf(y[e]), fabsf(z[e]));
                const int sb = scale_byte(max_over<LPH>(most));
                if (there && have) {
                    const float inv = __uint_as_float(static_cast<uint32_t>(254 - min(sb, 248)) << 23);
                    if (sb >= 248) {   // no numbers, or some that may be too large for the largest power of two
#pragma unroll
                        for (int e = 0; e < GE; ++e) {
                            y[e] = sb == 255 ? 0.f : fminf(fmaxf(y[e], -127 * 0x1p121f), 127 * 0x1p121f);
                            z[e] = sb == 255 ? 0.f : fminf(fmaxf(z[e], -127 * 0x1p121f), 127 * 0x1p121f);
                        }
                    }
                    store_codes(to + e1, y, inv);
                    store_codes(to + e2, z, inv);
                    if (hl == 0) (is_v ? R.value_scale : R.key_scale)[row + (static_cast<size_t>(h) << A.page_shift)] = static_cast<uint8_t>(sb);
                }
            } else if (there && have) {
                store4(to + e1, y);
                store4(to + e2, z);
            }
        }
        j0 += kBatch;
        if (j0 >= j_end) break;
        load(j0);
    }
}

// ---- read -------------------------------------------------------------------
// Codes and their row's byte to 16 bytes of numbers: 4 (fp32) or 8 (bf16).
template <class Out>
constexpr int kPer = 16 / sizeof(Out);
// code i of u (codes with their signs flipped) times scale: 2^23 + (n + 128) has the code as its low byte, and
// both products of the fma are exact (zero: -8388736 scale)
__device__ __forceinline__ float number(uint32_t u, int i, float scale, float zero) {
    return fmaf(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650 | i)), scale, zero);
}
__device__ __forceinline__ void store_numbers(float* p, uint32_t c, uint8_t b) {
    // 255: infinity, and every number NaN.  The scale in two factors, so that `zero` stays in range.
    const float s = __uint_as_float(static_cast<uint32_t>(b) << 23), t = b > 200 ? 0x1p-64f : 1.0f, z = -8388736.0f * (s * t);
    const uint32_t u = c ^ 0x80808080u;
    float4 y = make_float4(number(u, 0, s * t, z), number(u, 1, s * t, z), number(u, 2, s * t, z), number(u, 3, s * t, z));
    if (b > 200) y = make_float4(y.x * 0x1p64f, y.y * 0x1p64f, y.z * 0x1p64f, y.w * 0x1p64f);
    *reinterpret_cast<float4*>(p) = y;
}
__device__ __forceinline__ void store_numbers(__nv_bfloat16* p, uint2 c, uint8_t b) {
    const float s = __uint_as_float(static_cast<uint32_t>(b) << 23), t = b > 200 ? 0x1p-64f : 1.0f, z = -8388736.0f * (s * t);
    const uint32_t u = c.x ^ 0x80808080u, w = c.y ^ 0x80808080u;
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = number(u, i, s * t, z);
        y[4 + i] = number(w, i, s * t, z);
    }
    if (b > 200) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= 0x1p64f;
    }
    store8(p, y);
}
template <class Out>
using Codes = std::conditional_t<sizeof(Out) == 4, uint32_t, uint2>;

// Rows [r0, r0 + n) of one page of the 8-bit pools to rows of k and v (either
// may be null): whole rows are stored by consecutive lanes, K and V and several turns at once.
template <class Out>
__device__ __forceinline__ void read_rows(const Pool8& P, int n_head_kv, int id, int r0, int n, Out* k, int64_t k_stride, Out* v,
                                          int64_t v_stride) {
    constexpr int kTurns = 2, kHead = HD / kPer<Out>;   // pieces of a head
    const int per_row = n_head_kv * kHead, threads = blockDim.x;
    const bool ok = static_cast<unsigned>(id) < static_cast<unsigned>(P.n_pages);
    const size_t first = ((static_cast<size_t>(ok ? id : 0) * n_head_kv) << P.page_shift) + r0;
    const int dr = threads / per_row, dc = threads - dr * per_row;
    int r = threadIdx.x / per_row, c = threadIdx.x - r * per_row;
    if (dc == 0 && k && v) {   // the same piece of every row: places go up by steps
        const size_t row = first + (static_cast<size_t>(c / kHead) << P.page_shift) + r;
        const size_t at = row * HD + c % kHead * kPer<Out>;
        const int8_t* kp = P.key_codes + at;
        const int8_t* vp = P.value_codes + at;
        const uint8_t* ksp = P.key_scale + row;
        const uint8_t* vsp = P.value_scale + row;
        Out* ko = k + r * k_stride + c * kPer<Out>;
        Out* vo = v + r * v_stride + c * kPer<Out>;
        const int64_t k_step = dr * k_stride, v_step = dr * v_stride;
        for (; r < n; r += kTurns * dr) {
            Codes<Out> kc[kTurns], vc[kTurns];
            uint8_t ks[kTurns], vs[kTurns];
#pragma unroll
            for (int q = 0; q < kTurns; ++q) {
                kc[q] = vc[q] = Codes<Out>{};
                ks[q] = vs[q] = 0;
                if (r + q * dr < n && ok) {
                    kc[q] = *reinterpret_cast<const Codes<Out>*>(kp + q * dr * HD);
                    vc[q] = *reinterpret_cast<const Codes<Out>*>(vp + q * dr * HD);
                    ks[q] = ksp[q * dr];
                    vs[q] = vsp[q * dr];
                }
            }
#pragma unroll
            for (int q = 0; q < kTurns; ++q)
                if (r + q * dr < n) {
                    store_numbers(ko + q * k_step, kc[q], ks[q]);
                    store_numbers(vo + q * v_step, vc[q], vs[q]);
                }
            kp += kTurns * dr * HD;
            vp += kTurns * dr * HD;
            ksp += kTurns * dr;
            vsp += kTurns * dr;
            ko += kTurns * k_step;
            vo += kTurns * v_step;
        }
        return;
    }
    while (r < n) {
        Codes<Out> kc[kTurns], vc[kTurns];
        uint8_t ks[kTurns], vs[kTurns];
        int rr[kTurns], cc[kTurns];
#pragma unroll
        for (int q = 0; q < kTurns; ++q) {
            rr[q] = r;
            cc[q] = c;
            kc[q] = vc[q] = Codes<Out>{};
            ks[q] = vs[q] = 0;
            if (r < n && ok) {
                const size_t row = first + (static_cast<size_t>(c / kHead) << P.page_shift) + r;
                if (k) {
                    kc[q] = reinterpret_cast<const Codes<Out>*>(P.key_codes + row * HD)[c % kHead];
                    ks[q] = P.key_scale[row];
                }
                if (v) {
                    vc[q] = reinterpret_cast<const Codes<Out>*>(P.value_codes + row * HD)[c % kHead];
                    vs[q] = P.value_scale[row];
                }
            }
            r += dr;
            c += dc;
            if (c >= per_row) {
                c -= per_row;
                ++r;
            }
        }
#pragma unroll
        for (int q = 0; q < kTurns; ++q) {
            if (rr[q] >= n) continue;
            if (k) store_numbers(k + rr[q] * k_stride + cc[q] * kPer<Out>, kc[q], ks[q]);
            if (v) store_numbers(v + rr[q] * v_stride + cc[q] * kPer<Out>, vc[q], vs[q]);
        }
    }
}

constexpr int kReadThreads = 256;
// The sequences in groups of kReadThreads: thread i of the group has the rows
// and blocks of rows of its sequence, the shared arrays where they start.
// f(sequence's ChunkSeq, block in the sequence, part of it, block in all, first row in all) for every
// part p (block * PARTS + part of it) with p % gridDim.x == blockIdx.x; then g(first sequence of
// the group, starts of its blocks).  Returns the blocks in all.
struct WalkSmem {
    int64_t block0[kReadThreads + 1], row0[kReadThreads + 1];
    int64_t warp_sum[2][kReadThreads / 32];
};
template <int PARTS, class Rows, class F, class G>
__device__ __forceinline__ int64_t walk(WalkSmem& S, const ChunkDesc& d, int n_seqs, int block_rows, Rows&& rows_of, F&& f, G&& g) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t blocks_so_far = 0, rows_so_far = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += kReadThreads) {
        const int n = min(kReadThreads, n_seqs - s0);
        int64_t x[2] = {0, 0};
        if (tid < n) {
            const int64_t rows = rows_of(d.seqs[s0 + tid]);
            x[0] = (rows + block_rows - 1) / block_rows;
            x[1] = rows;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int64_t y = __shfl_up_sync(0xffffffffu, x[q], o);
                if (lane >= o) x[q] += y;
            }
            if (lane == 31) S.warp_sum[q][warp] = x[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 2; ++q)
            for (int w = 0; w < warp; ++w) x[q] += S.warp_sum[q][w];
        S.block0[tid + 1] = blocks_so_far + x[0];
        S.row0[tid + 1] = rows_so_far + x[1];
        if (tid == 0) {
            S.block0[0] = blocks_so_far;
            S.row0[0] = rows_so_far;
        }
        __syncthreads();
        const int64_t end = S.block0[n], p0 = blocks_so_far * PARTS;
        int64_t p = p0 + (gridDim.x + blockIdx.x - p0 % gridDim.x) % gridDim.x;
        for (int lo = 0; p < end * PARTS; p += gridDim.x) {
            const int64_t b = p / PARTS;
            int hi = n;   // the sequence with block0[lo] <= b < block0[lo + 1]
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (S.block0[mid] <= b) lo = mid;
                else hi = mid;
            }
            f(d.seqs[s0 + lo], static_cast<int>(b - S.block0[lo]), static_cast<int>(p % PARTS), b, S.row0[lo]);
        }
        g(s0, n, S.block0);
        blocks_so_far = end;
        rows_so_far = S.row0[n];
        __syncthreads();
    }
    return blocks_so_far;
}

// All rows of all sequences, one sequence after another.  HBM-bound: 24 x 8000 rows to bf16 44 us, 5.2 TB/s; 700 rows 3.8 us.
constexpr int kReadBlock = 64;       // the smallest page
// Rows of a part of a block, the unit of a CTA's work: 16, so that small reads reach all SMs (700 rows 3.8 us, with 32
// 4.9, with 64 7.6; 4 x 4000 12.5, with 32 13.8), or 32 where every CTA has a part (16 x 4000 to bf16 22.0 us, with 16
// 25.1; 60 x 8000 131, with 64 146).
constexpr int kReadFew = 16, kReadMany = 32;
constexpr int kReadCtas = 148 * 6;
// go(rows of a part) for a read of so many rows
template <class F>
cudaError_t by_part(int64_t rows, F&& go) {
    return rows > int64_t{1} * kReadCtas * kReadMany ? go(std::integral_constant<int, kReadMany>{})
                                                     : go(std::integral_constant<int, kReadFew>{});
}
template <class Out, int ROWS>
__global__ void __launch_bounds__(kReadThreads, 6) read8_kernel(const __grid_constant__ Read8Args A) {
    __shared__ WalkSmem S;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (A.d.hdr->id != A.plan_id) {
        if (threadIdx.x == 0) record_error(A.err, kErrBadDesc);
        return;
    }
    walk<kReadBlock / ROWS>(
        S, A.d, A.n_seqs, kReadBlock, [](const ChunkSeq& s) { return s.n_tokens > 0 ? static_cast<int64_t>(s.pos) + s.n_tokens : 0; },
        [&](const ChunkSeq& s, int block, int part, int64_t, int64_t row0) {
            const int r = block * kReadBlock + part * ROWS;
            const int64_t at = row0 + r;
            const int there = min(ROWS, s.pos + s.n_tokens - r);
            const int n = static_cast<int>(min(static_cast<int64_t>(there), A.n_rows - at));
            if (n < there && threadIdx.x == 0) record_error(A.err, kErrRoom);
            if (n <= 0) return;
            const int id = s.pages[r >> A.pool.page_shift];
            if (threadIdx.x == 0 && static_cast<unsigned>(id) >= static_cast<unsigned>(A.pool.n_pages)) record_error(A.err, kErrBadPage);
            read_rows(A.pool, A.n_head_kv, id, r & ((1 << A.pool.page_shift) - 1), n,
                      A.k ? static_cast<Out*>(A.k) + at * A.k_stride : nullptr, A.k_stride,
                      A.v ? static_cast<Out*>(A.v) + at * A.v_stride : nullptr, A.v_stride);
        },
        [](int, int, const int64_t*) {});
}

// The rows of the batch's new tokens, 16 bytes of numbers a thread: 16 x 1501 of 8 KV heads to bf16, just stored, 14.3 us,
// 48 x 1 2.6 us, a launch.
constexpr int kNewTurns = 2;
template <class Out>
__global__ void __launch_bounds__(kReadThreads) read8_new_kernel(const __grid_constant__ Read8Args A) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (A.d.hdr->id != A.plan_id) {
        if (threadIdx.x == 0) record_error(A.err, kErrBadDesc);
        return;
    }
    constexpr int kHead = HD / kPer<Out>;
    const uint32_t per_row = A.n_head_kv * kHead;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (kNewTurns * kReadThreads), tok0 = i0 / per_row;
    // kNewTurns pieces a thread, so that their ways from token to page overlap
    int64_t tok[kNewTurns];
    uint32_t c[kNewTurns];
    ChunkTok tk[kNewTurns];
    int id[kNewTurns];
#pragma unroll
    for (int q = 0; q < kNewTurns; ++q) {
        const uint32_t in = static_cast<uint32_t>(i0 - tok0 * per_row) + q * kReadThreads + threadIdx.x, more = in / per_row;
        tok[q] = tok0 + more;
        c[q] = in - more * per_row;
        tk[q] = tok[q] < A.n_tokens ? A.d.toks[tok[q]] : ChunkTok{};
    }
#pragma unroll
    for (int q = 0; q < kNewTurns; ++q) id[q] = tok[q] < A.n_tokens ? A.d.seqs[tk[q].seq].pages[tk[q].pos >> A.pool.page_shift] : 0;
    Codes<Out> kc[kNewTurns], vc[kNewTurns];
    uint8_t ks[kNewTurns], vs[kNewTurns];
#pragma unroll
    for (int q = 0; q < kNewTurns; ++q) {
        kc[q] = vc[q] = Codes<Out>{};
        ks[q] = vs[q] = 0;
        if (tok[q] >= A.n_tokens) continue;
        if (static_cast<unsigned>(id[q]) >= static_cast<unsigned>(A.pool.n_pages)) {
            record_error(A.err, kErrBadPage);
            continue;
        }
        const size_t row = ((static_cast<size_t>(id[q]) * A.n_head_kv + c[q] / kHead) << A.pool.page_shift) +
                           (tk[q].pos & ((1 << A.pool.page_shift) - 1));
        if (A.k) {
            kc[q] = reinterpret_cast<const Codes<Out>*>(A.pool.key_codes + row * HD)[c[q] % kHead];
            ks[q] = A.pool.key_scale[row];
        }
        if (A.v) {
            vc[q] = reinterpret_cast<const Codes<Out>*>(A.pool.value_codes + row * HD)[c[q] % kHead];
            vs[q] = A.pool.value_scale[row];
        }
    }
#pragma unroll
    for (int q = 0; q < kNewTurns; ++q) {
        if (tok[q] >= A.n_tokens) continue;
        if (A.k) store_numbers(static_cast<Out*>(A.k) + tok[q] * A.k_stride + c[q] * kPer<Out>, kc[q], ks[q]);
        if (A.v) store_numbers(static_cast<Out*>(A.v) + tok[q] * A.v_stride + c[q] * kPer<Out>, vc[q], vs[q]);
    }
}

// The rows of the sequences of many rows (those that chunk_few8_kernel does
// not take) as bf16 pages of kStageRows rows, and a copy of the descriptor's
// first records with page tables that lead to them, for the attention over
// bf16 pages.  Nothing is rounded: the stored values are bf16 numbers.  4 x 601
// behind up to 2999 rows, 11 us of the call's 84 (over bf16 pages 73.5); 32 x 6 behind 2000, 48 rows a KV head, 27 of 50 (bf16 pages 23).
template <int ROWS>
__global__ void __launch_bounds__(kReadThreads, 6) stage8_kernel(const __grid_constant__ Stage8Args A) {
    __shared__ WalkSmem S;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool mine = A.d.hdr->id == A.plan_id;
    if (!mine) {   // the attention will find the number of no plan
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            record_error(A.err, kErrBadDesc);
            A.hdr->id = 0;
        }
        return;
    }
    const size_t row_halfs = static_cast<size_t>(A.n_head_kv) * HD;
    const int64_t total = walk<kStageRows / ROWS>(
        S, A.d, A.n_seqs, kStageRows,
        [&](const ChunkSeq& s) {
            return static_cast<int64_t>(s.n_tokens) * A.group > kChunkFewRows ? static_cast<int64_t>(s.pos) + s.n_tokens : 0;
        },
        [&](const ChunkSeq& s, int block, int part, int64_t at, int64_t) {
            if (at >= A.n_pages) return;
            if (part == 0 && threadIdx.x == 0) A.table[at] = static_cast<int32_t>(at);
            const int r = block * kStageRows + part * ROWS, n = min(ROWS, s.pos + s.n_tokens - r);
            if (n <= 0) return;
            const int id = s.pages[r >> A.pool.page_shift];
            if (threadIdx.x == 0 && static_cast<unsigned>(id) >= static_cast<unsigned>(A.pool.n_pages)) record_error(A.err, kErrBadPage);
            const size_t to = (static_cast<size_t>(at) * kStageRows + part * ROWS) * row_halfs;
            read_rows(A.pool, A.n_head_kv, id, r & ((1 << A.pool.page_shift) - 1), n, A.k + to, row_halfs, A.v + to, row_halfs);
        },
        [&](int s0, int n, const int64_t* block0) {
            const int n_rec = A.n_ctas + A.n_segs;   // cta records and segments are one array
            for (int i = blockIdx.x * kReadThreads + threadIdx.x; i < n_rec; i += gridDim.x * kReadThreads) {
                ChunkSeg sg = A.d.cta[i];
                if (sg.seq < s0 || sg.seq >= s0 + n) continue;
                sg.pages = A.table + block0[sg.seq - s0];
                A.cta[i] = sg;
            }
        });
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        ChunkHeader h = *A.d.hdr;
        if (total > A.n_pages) {
            record_error(A.err, kErrRoom);
            h.id = 0;
        }
        *A.hdr = h;
    }
}

}  // namespace

template <class Act, class Pool, int BATCH>
static cudaError_t launch_append(const AppendRulesArgs& a, int parts, int64_t blocks, cudaStream_t stream) {
    Launch L(dim3(static_cast<unsigned>(blocks)), kThreads, 0, stream);
    if (a.q_norm || a.k_norm)
        return a.halves ? cudaLaunchKernelEx(&L.cfg, append_rules_kernel<Act, Pool, true, true, BATCH>, a, parts)
                        : cudaLaunchKernelEx(&L.cfg, append_rules_kernel<Act, Pool, false, true, BATCH>, a, parts);
    return a.halves ? cudaLaunchKernelEx(&L.cfg, append_rules_kernel<Act, Pool, true, false, BATCH>, a, parts)
                    : cudaLaunchKernelEx(&L.cfg, append_rules_kernel<Act, Pool, false, false, BATCH>, a, parts);
}
template <class Act, class Pool>
static cudaError_t launch_append(const AppendRulesArgs& a, cudaStream_t stream) {
    constexpr int heads = 32 * 2 * GE / HD;   // of a piece
    const int pieces = (a.a.n_head + heads - 1) / heads + 2 * ((a.a.n_head_kv + heads - 1) / heads);
    constexpr int part = sizeof(Act) == 4 ? 3 : 4;   // pieces of the smallest part of a token: one turn
    const int most = (pieces + part - 1) / part;
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, kWarps / a.a.n_tokens)));
    const int64_t blocks = (static_cast<int64_t>(a.a.n_tokens) * parts * 32 + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffLL / (kThreads / 32)) return cudaErrorInvalidConfiguration;
    if constexpr (sizeof(Act) == 4) {
        // three pieces in flight: 1 x 4096 with norms 18.2 us, with two 18.7, with four or five 20.3
        return launch_append<Act, Pool, 3>(a, parts, blocks, stream);
    } else {
        // four pieces in flight, or five where that saves a turn (8 pieces of 18 k tokens: 34.7 us with four, 39.5 with
        // five, for registers; 10 pieces of 4096: 11.0 and 9.8 us)
        const int mine = (pieces + parts - 1) / parts;
        return (mine + 4) / 5 < (mine + 3) / 4 ? launch_append<Act, Pool, 5>(a, parts, blocks, stream)
                                               : launch_append<Act, Pool, 4>(a, parts, blocks, stream);
    }
}

cudaError_t launch_append_rules(const AppendRulesArgs& a, bool act_bf16, int pool_bytes, cudaStream_t stream) {
    if (act_bf16)
        return pool_bytes == 1   ? launch_append<__nv_bfloat16, int8_t>(a, stream)
               : pool_bytes == 2 ? launch_append<__nv_bfloat16, __nv_bfloat16>(a, stream)
                                 : launch_append<__nv_bfloat16, float>(a, stream);
    return pool_bytes == 1   ? launch_append<float, int8_t>(a, stream)
           : pool_bytes == 2 ? launch_append<float, __nv_bfloat16>(a, stream)
                             : launch_append<float, float>(a, stream);
}

cudaError_t launch_read8(const Read8Args& a, bool out_bf16, bool new_only, cudaStream_t stream) {
    if (new_only) {
        const int64_t blocks = (static_cast<int64_t>(a.n_tokens) * a.n_head_kv * (HD / (out_bf16 ? 8 : 4)) + kNewTurns * kReadThreads - 1) /
                               (kNewTurns * kReadThreads);
        if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
        Launch L(dim3(static_cast<unsigned>(blocks)), kReadThreads, 0, stream);
        return out_bf16 ? cudaLaunchKernelEx(&L.cfg, read8_new_kernel<__nv_bfloat16>, a)
                        : cudaLaunchKernelEx(&L.cfg, read8_new_kernel<float>, a);
    }
    return by_part(a.n_rows, [&](auto part) {
        const int64_t blocks = std::min<int64_t>(kReadCtas, a.n_rows / part + a.n_seqs);
        Launch L(dim3(static_cast<unsigned>(blocks)), kReadThreads, 0, stream);
        return out_bf16 ? cudaLaunchKernelEx(&L.cfg, read8_kernel<__nv_bfloat16, decltype(part)::value>, a)
                        : cudaLaunchKernelEx(&L.cfg, read8_kernel<float, decltype(part)::value>, a);
    });
}

cudaError_t launch_stage8(const Stage8Args& a, cudaStream_t stream) {
    const int64_t rows = a.n_pages * kStageRows;   // at most: what the workspace has room for
    return by_part(rows, [&](auto part) {
        Launch L(dim3(static_cast<unsigned>(std::min<int64_t>(kReadCtas, std::max<int64_t>(rows / part, 1)))), kReadThreads, 0, stream);
        return cudaLaunchKernelEx(&L.cfg, stage8_kernel<decltype(part)::value>, a);
    });
}

}  // namespace tle
