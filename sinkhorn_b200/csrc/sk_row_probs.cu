// sk_row_probs.cu -- log probabilities of the rows of a cost (or of logits):
// log-sum-exp, log probability of a given column, entropy and the best k
// columns of each row from one read, and the gradients of all of them.
//
// With x_j = g_j - C_ij (or the logit itself) and z = x / eps, a row's
// distribution is p = softmax(z): the conditional P_ij / sum_j P_ij of the
// transport plan. One pass carries, relative to the running maximum m of x,
//     y = (x - m) log2(e) / eps,   s = sum 2^y,   u = sum y 2^y
// and moves them to a new maximum M with t = (m - M) log2(e) / eps:
//     s <- 2^t s,   u <- 2^t (u + t s),
// so that lse = m/eps + log s, log p_j = (x_j - m)/eps - log s and the entropy
// is log s - ln 2 u / s. Differences are taken before the scaling: the
// statistics (m, log s) lose nothing where |z| is large, and the backward gets
// them as that pair instead of as their rounded sum.
//
// The best k (k <= 32), ordered by (x descending, column ascending), cost the
// pass one maximum a lane: if k lanes each hold a value at or above t, nothing
// below t counts, and with t the k-th largest of the lanes' maxima hardly more
// than k lanes hold anything at or above it. Only those lanes' columns (1/256 of
// the row each) are read again, out of L2, by whole warps, and the few values
// that pass are ranked by counting how many beat each.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cooperative_groups.h>
#include <limits.h>

#include <algorithm>
#include <cmath>

#include "sk_common.cuh"
#include "sk_internal.h"

namespace sk {
namespace {

namespace cg = cooperative_groups;

constexpr float kNegInf = -INFINITY;
// An exponent (base 2, or e) that stands for all lower ones, -inf among them,
// where it is a factor of its own power: that power is 0 far above it, and
// 0 * -inf would be NaN.
constexpr float kFarBelow = -1e4f;

struct RowProbArgs {
    const void* X;
    int64_t N, M, sXb, sXn;
    int64_t rows;           // B * N
    const float* g;         // (B,M) or NULL; -inf where mask_b leaves a column out
    const uint8_t* mask_a;  // (B,N) or NULL
    float sign;             // x = g + sign * X
    float k;                // 1 / eps
    const int64_t* targets;  // (B,N) or NULL
    int top_k;
    float *lse, *logprob, *entropy, *top_lp;
    int64_t* top_idx;
    float2* stats;  // (m, log s) of each row
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

// 16 bytes of elements, streaming: each is read once.
template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
};

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// How a value becomes x. kPlain: the element itself. kAffine: g_j + sign * X.
// kMasked: the same, and -inf where g_j is -inf whatever X holds. A column mask
// is folded into g once a call (k_masked_g): in the rows' loop a byte mask cost
// as much as all the rest (16 x 2048 x 2048 fp32 on a B200: 154 us against 93 us
// with g alone and 53 us with neither).
enum Shape { kPlain = 0, kAffine = 1, kMasked = 2 };

struct RowShape {
    const float* g;  // this item's, or NULL
    float sign;
    bool g16;  // g is 16-byte aligned at the row's vectors
};

template <int SHAPE>
__device__ __forceinline__ float shaped1(float v, float g, float sign) {
    const float x = fmaf(v, sign, g);  // exact product: one rounding
    return SHAPE == kMasked && g == kNegInf ? kNegInf : x;
}

template <int SHAPE>
__device__ __forceinline__ float shaped(float v, const RowShape& rs, int64_t j) {
    if (SHAPE == kPlain) return v;
    return shaped1<SHAPE>(v, rs.g ? __ldg(rs.g + j) : 0.f, rs.sign);
}

// 2 * V2 consecutive values from column j on.
template <int SHAPE, int V2>
__device__ __forceinline__ void shape_pairs(float2* x, const RowShape& rs, int64_t j) {
    if (SHAPE == kPlain) return;
    float2 g[V2];
    if (!rs.g) {
#pragma unroll
        for (int e = 0; e < V2; ++e) g[e] = make_float2(0.f, 0.f);
    } else if (rs.g16) {
#pragma unroll
        for (int e = 0; e < V2; e += 2) {
            const float4 v = ld_vec4(rs.g + j + 2 * e);
            g[e] = make_float2(v.x, v.y);
            g[e + 1] = make_float2(v.z, v.w);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V2; ++e)
            g[e] = make_float2(__ldg(rs.g + j + 2 * e), __ldg(rs.g + j + 2 * e + 1));
    }
    const float2 sg = make_float2(rs.sign, rs.sign);
#pragma unroll
    for (int e = 0; e < V2; ++e) {
        x[e] = __ffma2_rn(x[e], sg, g[e]);
        if (SHAPE == kMasked) {
            if (g[e].x == kNegInf) x[e].x = kNegInf;
            if (g[e].y == kNegInf) x[e].y = kNegInf;
        }
    }
}

__device__ __forceinline__ RowShape row_shape(const float* g, float sign, int64_t b, int64_t M,
                                              int64_t lead) {
    RowShape rs;
    rs.g = g ? g + b * M : nullptr;
    rs.sign = sign;
    rs.g16 = (reinterpret_cast<uintptr_t>(rs.g + lead) & 15) == 0;
    return rs;
}

// g with -inf at the columns that mask_b leaves out.
__global__ void __launch_bounds__(256) k_masked_g(const float* g, const uint8_t* mask, float* out,
                                                  int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n;
         i += (int64_t)gridDim.x * 256)
        out[i] = mask[i] ? (g ? g[i] : 0.f) : kNegInf;
}

// Elements before the first 16-byte boundary of a row (at most the row).
template <typename T>
__device__ __forceinline__ int64_t row_lead(const T* row, int64_t M) {
    const int64_t lead = ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T);
    return lead < M ? lead : M;
}

// Running (m, s, u) of a row's distribution; empty: (-inf, 0, 0).
struct Moments {
    float m = kNegInf, s = 0.f, u = 0.f;

    __device__ __forceinline__ void move_to(float mn, float k2) {
        if (m != kNegInf) {
            const float t = fmaxf((m - mn) * k2, kFarBelow), r = ex2(t);
            u = r * fmaf(t, s, u);
            s *= r;
        }
        m = mn;
    }
    // A NaN shows in s; m passes over it. s of an empty set is 0, or NaN where
    // it held nothing but NaN.
    __device__ __forceinline__ void merge(float m2, float s2, float u2, float k2) {
        const float mn = fmaxf(m, m2);
        if (mn != kNegInf) {
            Moments o;
            o.m = m2;
            o.s = s2;
            o.u = u2;
            move_to(mn, k2);
            o.move_to(mn, k2);
            u += o.u;
            s2 = o.s;
        }
        s += s2;
    }
    // The warp's from its lanes': the maximum first, then plain sums.
    __device__ __forceinline__ void join(float k2) {
        move_to(warp_max(m), k2);
        s = warp_sum(s);
        u = warp_sum(u);
    }
    // Fold values with maximum cm in, two at a time on the packed fp32 pipe.
    // BOUND: exponents of -inf are expected (masks), else they are looked for.
    template <bool BOUND, int V2>
    __device__ __forceinline__ void fold(const float2 (&x)[V2], float cm, float k2) {
        const float mn = fmaxf(m, cm);
        if (mn == kNegInf) {
#pragma unroll
            for (int e = 0; e < V2; ++e)
                if (isnan(x[e].x + x[e].y)) s = NAN;
            return;
        }
        if (mn != m) move_to(mn, k2);
        const float2 nm = make_float2(-mn, -mn), kk = make_float2(k2, k2);
        float2 ss = make_float2(0.f, 0.f), uu = ss;
#pragma unroll
        for (int e = 0; e < V2; ++e) {
            const float2 y = __fmul2_rn(__fadd2_rn(x[e], nm), kk);
            const float2 t = make_float2(ex2(y.x), ex2(y.y));
            ss = __fadd2_rn(ss, t);
            uu = __ffma2_rn(
                t, BOUND ? make_float2(fmaxf(y.x, kFarBelow), fmaxf(y.y, kFarBelow)) : y, uu);
        }
        float du = uu.x + uu.y;
        if (!BOUND && isnan(du)) {
            // 0 * -inf (or a NaN value): once more with the exponents bounded
            du = 0.f;
#pragma unroll
            for (int e = 0; e < V2; ++e) {
                const float2 y = __fmul2_rn(__fadd2_rn(x[e], nm), kk);
                du = fmaf(ex2(y.x), fmaxf(y.x, kFarBelow), du);
                du = fmaf(ex2(y.y), fmaxf(y.y, kFarBelow), du);
            }
        }
        s += ss.x + ss.y;
        u += du;
    }
};

// Floats as unsigned integers of the same order (never NaN here).
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The r-th largest of the lanes' values (1 <= r <= 32).
__device__ __forceinline__ float warp_rth_largest(float v, int r, int lane) {
    if (r > 6) {
        int rank = 0;
#pragma unroll
        for (int l = 0; l < 32; ++l) {
            const float o = __shfl_sync(0xffffffffu, v, l);
            rank += o > v || (o == v && l < lane);
        }
        return __shfl_sync(0xffffffffu, v,
                           __ffs(__ballot_sync(0xffffffffu, rank == r - 1)) - 1);
    }
    unsigned o = ordered(v), top = 0;
    for (;;) {
        top = __reduce_max_sync(0xffffffffu, o);
        if (--r == 0) return unordered(top);
        if (lane == __ffs(__ballot_sync(0xffffffffu, o == top)) - 1) o = 0;
    }
}

__device__ __forceinline__ bool beats(float v, int i, float w, int j) {
    return v > w || (v == w && i < j);
}

constexpr int kListCap = 128;  // entries of a warp's list, four to a lane

// A warp's candidates for the best k, in shared memory, in any order.
struct TopList {
    float* v;
    int* i;
    int n = 0;
    float kth = kNegInf;  // the k-th when the list was last sorted
    int kth_i = INT_MAX;

    // Sort, keep the best k.
    __device__ __forceinline__ void keep(int k, int lane) {
        if (n <= 32) {
            __syncwarp();
            const float ev = lane < n ? v[lane] : kNegInf;
            const int ei = lane < n ? i[lane] : INT_MAX;
            int rank = lane < n ? 0 : 32;
            for (int l = 0; l < n; ++l)
                rank += beats(__shfl_sync(0xffffffffu, ev, l), __shfl_sync(0xffffffffu, ei, l),
                              ev, ei);
            if (rank < k) {
                v[rank] = ev;
                i[rank] = ei;
            }
            __syncwarp();
            n = min(n, k);
            return;  // (kth serves a list that ran full)
        }
        constexpr int P = kListCap / 32;
        float ev[P];
        int ei[P], rank[P];
        __syncwarp();
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const bool in = q * 32 + lane < n;
            ev[q] = in ? v[q * 32 + lane] : kNegInf;
            ei[q] = in ? i[q * 32 + lane] : INT_MAX;
            rank[q] = in ? 0 : kListCap;
        }
        for (int j = 0; j < n; ++j) {
            const float w = v[j];
            const int wi = i[j];
#pragma unroll
            for (int q = 0; q < P; ++q)
                if (q * 32 < n) rank[q] += beats(w, wi, ev[q], ei[q]);
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < P; ++q)
            if (rank[q] < k) {
                v[rank[q]] = ev[q];
                i[rank[q]] = ei[q];
            }
        __syncwarp();
        n = min(n, k);
        if (n == k) {
            kth = v[k - 1];
            kth_i = i[k - 1];
        }
    }
    // One candidate a lane; -inf, NaN, what is below `floor` and what does not
    // beat the k-th entry are passed over.
    __device__ __forceinline__ void offer(float cv, int ci, int k, float floor, int lane) {
        bool in = cv >= floor && cv > kNegInf && beats(cv, ci, kth, kth_i);
        unsigned who = __ballot_sync(0xffffffffu, in);
        if (!who) return;
        if (n + __popc(who) > kListCap) {
            keep(k, lane);
            in = in && beats(cv, ci, kth, kth_i);
            who = __ballot_sync(0xffffffffu, in);
        }
        if (in) {
            const int at = n + __popc(who & ((1u << lane) - 1u));
            v[at] = cv;
            i[at] = ci;
        }
        n += __popc(who);
    }
};

constexpr int kRowWarps = 8;  // warps of a CTA

// 16 bytes of elements as pairs.
__device__ __forceinline__ void unpack2(const uint4& v, float2* x, const float*) {
    x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, const __nv_bfloat16*) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, const __half*) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ void unpack2(const uint4& v, float2* x, const T* t) {
    x[0] = pair_of(v.x, t);
    x[1] = pair_of(v.y, t);
    x[2] = pair_of(v.z, t);
    x[3] = pair_of(v.w, t);
}

template <bool TOP>
struct RowProbShared {
    float m[kRowWarps], s[kRowWarps], u[kRowWarps];
};
template <>
struct RowProbShared<true> {
    float m[kRowWarps], s[kRowWarps], u[kRowWarps];
    float high[kRowWarps * 4];  // the four largest lane maxima of each warp
    int from[kRowWarps][32];    // first vectors of the lanes that are read again
    int n[kRowWarps];
    float lv[kRowWarps][kListCap];
    int li[kRowWarps][kListCap];
    float ov[32];  // this CTA's best k, sorted
    int oi[32];
};

// The best k of `lists` unsorted lists of at most 32 entries into ov / oi
// (-inf and -1 where there are fewer). All threads of the CTA.
__device__ __forceinline__ void select_best(RowProbShared<true>& sh, int lists, int k) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int total = 0, before = 0;
    for (int l = 0; l < lists; ++l) {
        if (l < warp) before += sh.n[l];
        total += sh.n[l];
    }
    if (threadIdx.x < 32) {
        sh.ov[lane] = kNegInf;
        sh.oi[lane] = -1;
    }
    if (total <= 32) {
        // one warp: an entry to a lane
        if (warp == 0) {
            float v = kNegInf;
            int i = INT_MAX, from = 0;
            for (int l = 0; l < lists; ++l) {
                const int n = sh.n[l];
                if (lane >= from && lane < from + n) {
                    v = sh.lv[l][lane - from];
                    i = sh.li[l][lane - from];
                }
                from += n;
            }
            __syncwarp();
            int rank = 0;
            for (int l = 0; l < total; ++l)
                rank += beats(__shfl_sync(0xffffffffu, v, l), __shfl_sync(0xffffffffu, i, l), v, i);
            if (lane < total && rank < k) {
                sh.ov[rank] = v;
                sh.oi[rank] = i;
            }
        }
    } else {
        __syncthreads();
        if (warp < lists && lane < sh.n[warp]) {
            const float v = sh.lv[warp][lane];
            const int i = sh.li[warp][lane];
            int rank = 0;
            for (int l = 0; l < lists; ++l)
                for (int j = 0; j < sh.n[l]; ++j)
                    rank += beats(sh.lv[l][j], sh.li[l][j], v, i);
            if (rank < k) {
                sh.ov[rank] = v;
                sh.oi[rank] = i;
            }
        }
    }
    __syncthreads();
}

// WARPS == 1: a warp per row, 8 rows per CTA, no cluster. WARPS == 8: a CTA or
// a cluster of CTAs per row, joined over distributed shared memory by rank 0.
// A step is U vectors of 16 bytes a lane; as each pair of them is unpacked, the
// loads of the next step take its registers, so that a warp keeps U KB / 2 in
// flight. U == 1 is for rows of a single step (and keeps its values).
template <typename T, int SHAPE, bool TOP, int WARPS, int U>
__global__ void __launch_bounds__(256, SHAPE ? 3 : 4) k_row_probs(const RowProbArgs A) {
    constexpr int V = Vec<T>::n;
    constexpr int H = U == 1 ? 1 : 16 / V;  // vectors folded at once: 16 values
    static_assert(U % H == 0, "whole folds");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ RowProbShared<TOP> sh;
    int64_t row;
    int part = 0, parts = 1;
    if (WARPS == 1) {
        row = (int64_t)blockIdx.x * kRowWarps + warp;
        if (row >= A.rows) return;
    } else {
        parts = cg::this_cluster().num_blocks();
        part = cg::this_cluster().block_rank();
        row = blockIdx.x / parts;
    }
    const int64_t b = row / A.N, n = row - b * A.N;
    const T* const X = reinterpret_cast<const T*>(A.X) + b * A.sXb + n * A.sXn;
    const int M = (int)A.M;
    const int lead = (int)row_lead(X, A.M);
    const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead);
    const float k2 = A.k * kLog2e;
    const bool empty = A.mask_a && !A.mask_a[row];
    const int nv = empty ? 0 : (M - lead) / V;
    const int k = A.top_k;
    const int wid = WARPS == 1 ? 0 : part * WARPS + warp;
    const int step = (WARPS == 1 ? 1 : parts * WARPS) * 32 * U;
    const uint4* const body = reinterpret_cast<const uint4*>(X + lead);

    Moments mo;
    float best = kNegInf;  // the lane's largest value among whole vectors
    float2 x[H * V / 2];

    auto fold = [&]() {
        float cm = kNegInf;
#pragma unroll
        for (int e = 0; e < H * V / 2; ++e) cm = fmaxf(cm, fmaxf(x[e].x, x[e].y));
        if (TOP) best = fmaxf(best, cm);
        mo.fold<SHAPE != kPlain>(x, cm, k2);
    };
    const int base = wid * 32 * U + lane;
    int i = base;  // this lane's first vector of the step
    if (U > 1 && wid * 32 * U + 32 * U <= nv) {
        uint4 raw[U];
#pragma unroll
        for (int q = 0; q < U; ++q) raw[q] = ld_stream16(body + i + q * 32);
        const int last = nv - (32 * U - lane);  // of the steps that are whole
        while (true) {
            const bool more = i + step <= last;
#pragma unroll
            for (int h = 0; h < U; h += H) {
#pragma unroll
                for (int q = 0; q < H; ++q) {
                    unpack2(raw[h + q], x + q * (V / 2), X);
                    if (more) raw[h + q] = ld_stream16(body + i + step + (h + q) * 32);
                    shape_pairs<SHAPE, V / 2>(x + q * (V / 2), rs,
                                             lead + (int64_t)(i + (h + q) * 32) * V);
                }
                fold();
            }
            i += step;
            if (!more) break;
        }
    }
    // the warp's last step, vector by vector
    for (; i - lane < nv; i += step) {
#pragma unroll
        for (int h = 0; h < U; h += H) {
#pragma unroll
            for (int q = 0; q < H; ++q) {
                const int at = i + (h + q) * 32;
                float2* const xq = x + q * (V / 2);
                if (at < nv) {
                    unpack2(ld_stream16(body + at), xq, X);
                    shape_pairs<SHAPE, V / 2>(xq, rs, lead + (int64_t)at * V);
                } else {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) xq[e] = make_float2(kNegInf, kNegInf);
                }
            }
            fold();
        }
    }
    // the row's ends, one column to a lane: up to V - 1 before the first vector
    // and as many behind the last
    const int tail = lead + nv * V;
    float end = kNegInf;
    int end_j = 0;
    if (!empty && wid == 0 && (lead > 0 || tail < M)) {
        end_j = lane < 16 ? lane : tail + lane - 16;
        if (lane < 16 ? lane < lead : end_j < M) end = shaped<SHAPE>(widen(X[end_j]), rs, end_j);
        const float2 e[1] = {make_float2(end, kNegInf)};
        mo.fold<true>(e, end, k2);
    }
    mo.join(k2);

    TopList top;
    if constexpr (TOP) {
        top.v = sh.lv[warp];
        top.i = sh.li[warp];
        top.offer(end, end_j, k, kNegInf, lane);
        if (U == 1) {
            const float bound = warp_rth_largest(best, k, lane);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                const bool in = best >= bound && base < nv;
                top.offer(in ? x[e].x : kNegInf, lead + base * V + 2 * e, k, bound, lane);
                top.offer(in ? x[e].y : kNegInf, lead + base * V + 2 * e + 1, k, bound, lane);
            }
        } else {
            float bound;
            if (WARPS == 1) {
                bound = warp_rth_largest(best, k, lane);
            } else {
                // four maxima of each warp stand for its lanes: k of these 32 are
                // k lanes, too
                unsigned o = ordered(best), high = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const unsigned t = __reduce_max_sync(0xffffffffu, o);
                    if (lane == r) high = t;
                    if (lane == __ffs(__ballot_sync(0xffffffffu, o == t)) - 1) o = 0;
                }
                if (lane < 4) sh.high[warp * 4 + lane] = unordered(high);
                __syncthreads();
                bound = warp_rth_largest(sh.high[lane], k, lane);
            }
            const bool held = best >= bound && best > kNegInf;
            const unsigned mine = __ballot_sync(0xffffffffu, held);
            // the vectors of those lanes, one to each lane of the warp at a time
            if (held) sh.from[warp][__popc(mine & ((1u << lane) - 1u))] = base;
            __syncwarp();
            const int per = (nv - wid * 32 * U + step - 1) / step * U;  // of a lane, at most
            const int all = __popc(mine) * per;
            for (int c = 0; c < all; c += 32) {
                const int f = c + lane, q = f / per, r = f - q * per;
                const int at = f < all ? sh.from[warp][q] + r / U * step + r % U * 32 : nv;
                float2 y[V / 2];
                if (at < nv) {
                    unpack2(ld_stream16(body + at), y, X);
                    shape_pairs<SHAPE, V / 2>(y, rs, lead + (int64_t)at * V);
                } else {
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) y[e] = make_float2(kNegInf, kNegInf);
                }
                unsigned marks = 0;  // values that pass (mostly one or none)
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    if (y[e].x >= bound) marks |= 1u << (2 * e);
                    if (y[e].y >= bound) marks |= 2u << (2 * e);
                }
                while (__any_sync(0xffffffffu, marks != 0)) {
                    float v = kNegInf;
                    const int e = marks ? __ffs(marks) - 1 : 0;
#pragma unroll
                    for (int p = 0; p < V / 2; ++p) {
                        if (e == 2 * p) v = y[p].x;
                        if (e == 2 * p + 1) v = y[p].y;
                    }
                    top.offer(marks ? v : kNegInf, lead + at * V + e, k, bound, lane);
                    marks &= marks - 1;
                }
            }
        }
        if (WARPS == 1 || top.n > 32) top.keep(k, lane);
    }

    if (WARPS > 1) {
        if (lane == 0) {
            sh.m[warp] = mo.m;
            sh.s[warp] = mo.s;
            sh.u[warp] = mo.u;
            if constexpr (TOP) sh.n[warp] = top.n;
        }
        __syncthreads();
        if constexpr (TOP) select_best(sh, WARPS, k);
        cg::cluster_group cluster = cg::this_cluster();
        if (parts > 1) {
            cluster.sync();
            if constexpr (TOP) {
                if (part == 0) {
                    // the peers' best k into this CTA's lists
                    if (warp < parts) {
                        const RowProbShared<TOP>* o = cluster.map_shared_rank(&sh, warp);
                        const float v = lane < k ? o->ov[lane] : kNegInf;
                        const int at = lane < k ? o->oi[lane] : -1;
                        sh.lv[warp][lane] = v;
                        sh.li[warp][lane] = at;
                        const int have = __popc(__ballot_sync(0xffffffffu, at >= 0));
                        if (lane == 0) sh.n[warp] = have;
                    }
                    __syncthreads();
                    select_best(sh, parts, k);
                }
            }
        }
        if (part == 0 && warp == 0) {
            // up to 8 x 8 parts, two to a lane
            mo = Moments();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = (lane + 32 * h) / WARPS, w = lane % WARPS;
                if (r < parts) {
                    const RowProbShared<TOP>* o =
                        parts > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
                    mo.merge(o->m[w], o->s[w], o->u[w], k2);
                }
            }
            mo.join(k2);
        }
        if (parts > 1) cluster.sync();  // rank 0 has read this CTA's shared memory
        if (part != 0 || warp != 0) return;
    }

    // an empty row keeps s = 0; a row of NaN alone has s = NaN
    const bool none = mo.m == kNegInf && mo.s == 0.f;
    const float logs = none ? 0.f : logf(mo.s);
    if (lane == 0) {
        if (A.stats) A.stats[row] = make_float2(none ? kNegInf : mo.m, logs);
        if (A.lse) A.lse[row] = none ? kNegInf : fmaf(mo.m, A.k, logs);
        if (A.entropy) A.entropy[row] = none ? 0.f : logs - kLn2 * (mo.u / mo.s);
        if (A.logprob) {
            const int64_t t = A.targets[row];
            float lp = 0.f;
            if (t >= A.M) lp = NAN;
            else if (t >= 0) {
                const float v = none ? kNegInf : shaped<SHAPE>(widen(X[t]), rs, t);
                lp = none ? kNegInf : fmaf(v - mo.m, A.k, -logs);
            }
            A.logprob[row] = lp;
        }
    }
    if constexpr (TOP) {
        if (lane < k) {
            const float* lv = WARPS == 1 ? top.v : sh.ov;
            const int* li = WARPS == 1 ? top.i : sh.oi;
            const bool held = WARPS == 1 ? lane < top.n : li[lane] >= 0;
            A.top_lp[row * k + lane] = held ? fmaf(lv[lane] - mo.m, A.k, -logs) : kNegInf;
            A.top_idx[row * k + lane] = held ? li[lane] : -1;
        }
    }
}

template <typename T, int SHAPE, bool TOP, int WARPS, int U>
int launch_rows(const RowProbArgs& A, int cluster, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    const int64_t ctas = WARPS == 1 ? (A.rows + 7) / 8 : A.rows * cluster;
    if (ctas > INT_MAX) return fail(SK_ERR_ARG, "B * N is too large");
    cfg.gridDim = dim3((unsigned)ctas);
    if (WARPS > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    SK_CUDA(cudaLaunchKernelEx(&cfg, k_row_probs<T, SHAPE, TOP, WARPS, U>, A));
    return SK_OK;
}

// How a row is split. A warp per row needs no join, and serves short rows and
// row counts that fill the SMs with warps; longer or fewer rows take a CTA, and
// where the rows alone leave SMs idle a cluster of up to 8 CTAs (each with at
// least one full step of its 8 warps).
template <typename T, int SHAPE, bool TOP>
int launch_rows_sized(const RowProbArgs& A, cudaStream_t s) {
    constexpr int U = 4;
    const int64_t bytes = A.M * (int64_t)sizeof(T);
    if (bytes <= 512) return launch_rows<T, SHAPE, TOP, 1, 1>(A, 1, s);
    if (bytes <= 2048 || (bytes <= 16384 && A.rows >= 148 * 16))
        return launch_rows<T, SHAPE, TOP, 1, U>(A, 1, s);
    int cluster = 1;
    while (cluster < 8 && A.rows * cluster * 2 <= 148 * 4 &&
           bytes > (int64_t)cluster * kRowWarps * 32 * U * 16)
        cluster *= 2;
    return launch_rows<T, SHAPE, TOP, kRowWarps, U>(A, cluster, s);
}

template <typename T, int SHAPE>
int launch_rows_shaped(const RowProbArgs& A, cudaStream_t s) {
    return A.top_k > 0 ? launch_rows_sized<T, SHAPE, true>(A, s)
                       : launch_rows_sized<T, SHAPE, false>(A, s);
}

template <typename T>
int launch_rows_typed(const RowProbArgs& A, bool masked, cudaStream_t s) {
    if (masked) return launch_rows_shaped<T, kMasked>(A, s);
    if (A.g || A.sign != 1.f) return launch_rows_shaped<T, kAffine>(A, s);
    return launch_rows_shaped<T, kPlain>(A, s);
}

// mask_b folded into g in the workspace; *g is then that.
int fold_mask(const float** g, const uint8_t* mask_b, int64_t BM, void* workspace,
              cudaStream_t s) {
    if (!mask_b) return SK_OK;
    k_masked_g<<<(unsigned)std::min<int64_t>((BM + 255) / 256, 148 * 8), 256, 0, s>>>(
        *g, mask_b, (float*)workspace, BM);
    SK_LAUNCHED("k_masked_g");
    *g = (const float*)workspace;
    return SK_OK;
}

// ---------------------------------------------------------------- backward
//
// With A = the upstream gradient of the given log probability, t_j those of
// the alternatives, c of lse and h of the entropy,
//     dz_v = p_v (c - A - sum t_j - h (log p_v + H)) + A [v = target]
//            + sum_j t_j [v = top_j],
// dX = sign dz / eps and dg = sum over the rows of dz / eps. Elementwise but
// for dg: a CTA takes a tile of columns and a band of rows, its row constants
// in shared memory, so that a thread's columns stay its own and dg needs no
// atomics (bands are summed in a fixed order by a second kernel).

struct RowProbBwdArgs {
    const void* X;
    int64_t N, M, sXb, sXn;
    int64_t B;
    const float* g;  // as in RowProbArgs
    float sign, k;
    const int64_t* targets;
    int top_k;
    const int64_t* top_idx;
    const float2* stats;
    const float* entropy;
    const float *g_lse, *g_lp, *g_ent, *g_top;
    void* dX;        // dense (B,N,M) or NULL
    float* partial;  // (B, bands, M) or NULL
    int64_t bands, band_rows;
};

constexpr int kBwdThreads = 256;
constexpr int kBwdRows = 64;  // most rows of a band held in shared memory at once
constexpr int kBwdVecs = 2;   // vectors of a row to a thread

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half narrow<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t pack2(float2 v, const __half*) {
    const __half2 h = __float22half2_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float2 v, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 bytes of elements, each rounded once from fp32.
template <typename T>
__device__ __forceinline__ uint4 pack16(const float2* x, const T* t) {
    return make_uint4(pack2(x[0], t), pack2(x[1], t), pack2(x[2], t), pack2(x[3], t));
}
__device__ __forceinline__ uint4 pack16(const float2* x, const float*) {
    return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x),
                      __float_as_uint(x[1].y));
}

// dX_v = p_v (c - h lp2) + at [v = target], lp2 = log2 p_v = (x_v - m) k2 - l2;
// every factor has sign / eps in it already.
struct RowConst {
    float m, l2, c, h, at;
    int target;
};

// COLS: the column sums are wanted; a thread then keeps its columns over all
// rows (vectors only where every row is aligned, VEC). Otherwise vectors start
// at each row's own 16-byte boundary.
template <typename T, int SHAPE, bool TOP, bool COLS, bool VEC>
__global__ void __launch_bounds__(kBwdThreads, 4) k_row_probs_bwd(const RowProbBwdArgs A,
                                                                  int tx) {
    constexpr int V = VEC ? Vec<T>::n : 2, V2 = V / 2, U = kBwdVecs;
    __shared__ RowConst rc[kBwdRows];
    __shared__ float red[COLS ? kBwdThreads * V * U : 1];
    const int ty = kBwdThreads / tx;
    const int cx = threadIdx.x % tx, cy = threadIdx.x / tx;
    const int M = (int)A.M;
    const int64_t col0 = ((int64_t)blockIdx.x * tx * U + cx) * V;  // before the row's lead
    const float k2 = A.k * kLog2e, ks = A.k * A.sign;

    for (int64_t band = blockIdx.y; band < A.B * A.bands; band += gridDim.y) {
        const int64_t b = band / A.bands;
        const int64_t r0 = (band - b * A.bands) * A.band_rows;
        const int64_t r1 = min(A.N, r0 + A.band_rows);
        const T* const Xb = reinterpret_cast<const T*>(A.X) + b * A.sXb;
        T* const Db = reinterpret_cast<T*>(A.dX) + b * A.N * A.M;
        float2 acc[COLS ? U * V2 : 1];
#pragma unroll
        for (int e = 0; e < (COLS ? U * V2 : 1); ++e) acc[e] = make_float2(0.f, 0.f);

        for (int64_t rb0 = r0; rb0 < r1; rb0 += kBwdRows) {
            const int nr = (int)min((int64_t)kBwdRows, r1 - rb0);
            __syncthreads();  // the last rows' constants and sums are read
            for (int r = threadIdx.x; r < nr; r += kBwdThreads) {
                const int64_t row = b * A.N + rb0 + r;
                const float2 st = A.stats[row];
                RowConst q;
                q.target = -1;
                q.at = q.h = q.c = 0.f;
                q.m = st.x;
                q.l2 = st.y * kLog2e;
                if (st.x == kNegInf && st.y == 0.f) {
                    q.m = 0.f;  // an empty row: log p = -inf everywhere
                    q.l2 = INFINITY;
                } else {
                    if (A.g_lp) {
                        const int64_t t = A.targets[row];
                        bool given = t >= 0 && t < A.M;
                        if (given) {
                            // a column without probability passes nothing
                            const RowShape ts = row_shape(A.g, A.sign, b, A.M, 0);
                            given = shaped<SHAPE>(widen(Xb[(rb0 + r) * A.sXn + t]), ts, t) !=
                                    kNegInf;
                        }
                        if (given) {
                            q.at = A.g_lp[row];
                            q.target = (int)t;
                        }
                    }
                    if (A.g_lse) q.c = A.g_lse[row];
                    if (A.g_ent) {
                        q.h = A.g_ent[row];
                        q.c -= q.h * A.entropy[row];
                    }
                    float t = q.at;
                    if (TOP)
                        for (int j = 0; j < A.top_k; ++j)
                            if (A.top_idx[row * A.top_k + j] >= 0)
                                t += A.g_top[row * A.top_k + j];
                    q.c = (q.c - t) * ks;
                    q.h *= ks * kLn2;
                    q.at *= ks;
                }
                rc[r] = q;
            }
            __syncthreads();
            uint4 raw[U];
            auto load = [&](int r) {
                const T* const X = Xb + (rb0 + r) * A.sXn;
                const int lead = COLS ? 0 : (int)row_lead(X, A.M);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t j = lead + col0 + (int64_t)u * tx * V;
                    if (j + V <= M) raw[u] = ld_stream16(X + j);
                }
            };
            if (VEC && cy < nr) load(cy);
            for (int r = cy; r < nr; r += ty) {
                const RowConst q = rc[r];
                const int64_t row = b * A.N + rb0 + r;
                const T* const X = Xb + (rb0 + r) * A.sXn;
                T* const D = A.dX ? Db + (rb0 + r) * A.M : nullptr;
                const int lead = COLS || !VEC ? 0 : (int)row_lead(X, A.M);
                const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead);
                float2 x[U * V2];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t j = lead + col0 + (int64_t)u * tx * V;
                    if constexpr (VEC) {
                        unpack2(raw[u], x + u * V2, X);
                        if (j + V <= M) shape_pairs<SHAPE, V2>(x + u * V2, rs, j);
                    } else {
                        x[u].x = j < M ? shaped<SHAPE>(widen(X[j]), rs, j) : kNegInf;
                        x[u].y = j + 1 < M ? shaped<SHAPE>(widen(X[j + 1]), rs, j + 1) : kNegInf;
                    }
                }
                if (VEC && r + ty < nr) load(r + ty);
                const float2 nm = make_float2(-q.m, -q.m), kk = make_float2(k2, k2);
                const float2 nl = make_float2(-q.l2, -q.l2), cc = make_float2(q.c, q.c);
                const float2 nh = make_float2(-q.h, -q.h);
                auto slope = [&](float2 v) {
                    float2 y = __ffma2_rn(__fadd2_rn(v, nm), kk, nl);
                    const float2 p = make_float2(ex2(y.x), ex2(y.y));
                    y = make_float2(fmaxf(y.x, kFarBelow), fmaxf(y.y, kFarBelow));
                    return __fmul2_rn(p, __ffma2_rn(y, nh, cc));
                };
                // the upstream gradients of single columns
                auto extra = [&](int64_t j) {
                    float d = j == q.target ? q.at : 0.f;
                    if (TOP)
                        for (int t = 0; t < A.top_k; ++t)
                            if (__ldg(A.top_idx + row * A.top_k + t) == j)
                                d = fmaf(__ldg(A.g_top + row * A.top_k + t), ks, d);
                    return d;
                };
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t j = lead + col0 + (int64_t)u * tx * V;
                    if (j >= M) break;
                    float2* const d = x + u * V2;
                    if (VEC && j + V > M) {
                        // the row's last columns, fewer than a vector
#pragma unroll
                        for (int e = 0; e < V2; ++e) {
                            const int64_t i = j + 2 * e;
                            d[e].x = i < M ? shaped<SHAPE>(widen(X[i]), rs, i) : kNegInf;
                            d[e].y = i + 1 < M ? shaped<SHAPE>(widen(X[i + 1]), rs, i + 1)
                                               : kNegInf;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < V2; ++e) d[e] = slope(d[e]);
                    if (q.target >= j && q.target < j + V) {
#pragma unroll
                        for (int e = 0; e < V2; ++e) {
                            if (q.target == j + 2 * e) d[e].x += q.at;
                            if (q.target == j + 2 * e + 1) d[e].y += q.at;
                        }
                    }
                    if (TOP) {
                        for (int t = 0; t < A.top_k; ++t) {
                            const int64_t at = __ldg(A.top_idx + row * A.top_k + t) - j;
                            if (at >= 0 && at < V) {
                                const float gt = __ldg(A.g_top + row * A.top_k + t) * ks;
#pragma unroll
                                for (int e = 0; e < V2; ++e) {
                                    if (at == 2 * e) d[e].x += gt;
                                    if (at == 2 * e + 1) d[e].y += gt;
                                }
                            }
                        }
                    }
                    if (COLS) {
#pragma unroll
                        for (int e = 0; e < V2; ++e)
                            acc[u * V2 + e] = __fadd2_rn(acc[u * V2 + e], d[e]);
                    }
                    if (D) {
                        bool whole = false;
                        if constexpr (VEC) {
                            whole = j + V <= M && (reinterpret_cast<uintptr_t>(D + j) & 15) == 0;
                            if (whole) *reinterpret_cast<uint4*>(D + j) = pack16(d, D);
                        }
                        if (!whole) {
#pragma unroll
                            for (int e = 0; e < V2; ++e) {
                                if (j + 2 * e < M) D[j + 2 * e] = narrow<T>(d[e].x);
                                if (j + 2 * e + 1 < M) D[j + 2 * e + 1] = narrow<T>(d[e].y);
                            }
                        }
                    }
                }
                if (!COLS && VEC && blockIdx.x == 0 && cx < lead && D) {
                    // the columns before the row's first vector, one to a thread
                    const float v = shaped<SHAPE>(widen(X[cx]), rs, cx);
                    D[cx] = narrow<T>(slope(make_float2(v, v)).x + extra(cx));
                }
            }
        }
        if (COLS) {
            // (a column sum is of dz / eps: without the sign)
#pragma unroll
            for (int e = 0; e < U * V2; ++e) {
                red[threadIdx.x * (U * V) + 2 * e] = acc[e].x;
                red[threadIdx.x * (U * V) + 2 * e + 1] = acc[e].y;
            }
            __syncthreads();
            if (cy == 0) {
                float* const out = A.partial + band * A.M;
#pragma unroll
                for (int e = 0; e < U * V; ++e) {
                    const int64_t j = col0 + (int64_t)(e / V) * tx * V + e % V;
                    float t = 0.f;
                    for (int y = 0; y < ty; ++y) t += red[(y * tx + cx) * (U * V) + e];
                    if (j < M) out[j] = A.sign * t;
                }
            }
        }
    }
}

// dg[b][j] = sum over the bands: 32 columns and 32 slices of the bands to a
// CTA, the slices added in order.
__global__ void __launch_bounds__(1024) k_band_sum(const float* partial, float* dg, int64_t BM,
                                                   int64_t M, int64_t bands) {
    __shared__ float part[32][33];
    const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float t = 0.f;
    if (i < BM) {
        const int64_t b = i / M, j = i - b * M;
        const float* p = partial + b * bands * M + j;
        const int64_t each = (bands + 31) / 32, q1 = min(bands, (threadIdx.y + 1) * each);
#pragma unroll 4
        for (int64_t q = threadIdx.y * each; q < q1; ++q) t += p[q * M];
    }
    part[threadIdx.y][threadIdx.x] = t;
    __syncthreads();
    if (threadIdx.y == 0 && i < BM) {
#pragma unroll
        for (int y = 1; y < 32; ++y) t += part[y][threadIdx.x];
        dg[i] = t;
    }
}

// Bands of the backward: enough CTAs for eight to an SM, whole groups of rows.
void bwd_bands(int64_t B, int64_t N, int64_t M, bool cols, int elem, int64_t* bands,
               int64_t* band_rows) {
    const int64_t tile = (int64_t)kBwdThreads * kBwdVecs * (16 / elem);
    const int64_t tiles = std::max<int64_t>(1, (M + tile - 1) / tile) * B;
    int64_t want = std::max<int64_t>(1, 148 * 8 / std::max<int64_t>(1, tiles));
    // without column sums bands are free; with them each costs a row of partials
    if (!cols) want = std::max<int64_t>(want, (N + kBwdRows - 1) / kBwdRows);
    const int64_t br = std::max<int64_t>((N + want - 1) / want, 1);
    *bands = (N + br - 1) / br;
    *band_rows = br;
}

template <typename T, int SHAPE, bool TOP>
int launch_bwd(const RowProbBwdArgs& A, float* dg, cudaStream_t s) {
    const bool cols = dg != nullptr;
    // every row's vectors start where the first's do
    const bool rows_aligned = (uintptr_t)A.X % 16 == 0 && (A.sXn * sizeof(T)) % 16 == 0 &&
                              (A.B == 1 || (A.sXb * sizeof(T)) % 16 == 0);
    const bool vec = !cols || rows_aligned;
    const int V = vec ? Vec<T>::n : 2;
    // threads along a row: a power of two that covers it, at least the V - 1
    // that the columns before its first vector take
    const int64_t cv = ((A.M + V - 1) / V + kBwdVecs - 1) / kBwdVecs;
    int tx = 8;
    while (tx < kBwdThreads && tx < cv) tx *= 2;
    const int64_t gx = (cv + tx - 1) / tx;
    const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>(A.bands * A.B, 65535));
    if (cols && vec)
        k_row_probs_bwd<T, SHAPE, TOP, true, true><<<grid, kBwdThreads, 0, s>>>(A, tx);
    else if (cols)
        k_row_probs_bwd<T, SHAPE, TOP, true, false><<<grid, kBwdThreads, 0, s>>>(A, tx);
    else
        k_row_probs_bwd<T, SHAPE, TOP, false, true><<<grid, kBwdThreads, 0, s>>>(A, tx);
    SK_LAUNCHED("k_row_probs_bwd");
    if (cols) {
        const int64_t BM = A.B * A.M;
        k_band_sum<<<(unsigned)((BM + 31) / 32), dim3(32, 32), 0, s>>>(A.partial, dg, BM, A.M, A.bands);
        SK_LAUNCHED("k_band_sum");
    }
    return SK_OK;
}

template <typename T, int SHAPE>
int launch_bwd_shaped(const RowProbBwdArgs& A, float* dg, cudaStream_t s) {
    return A.g_top ? launch_bwd<T, SHAPE, true>(A, dg, s) : launch_bwd<T, SHAPE, false>(A, dg, s);
}

template <typename T>
int launch_bwd_typed(const RowProbBwdArgs& A, bool masked, float* dg, cudaStream_t s) {
    if (masked) return launch_bwd_shaped<T, kMasked>(A, dg, s);
    if (A.g || A.sign != 1.f) return launch_bwd_shaped<T, kAffine>(A, dg, s);
    return launch_bwd_shaped<T, kPlain>(A, dg, s);
}

int check_rows(const void* X, int dtype, int64_t B, int64_t N, int64_t M, int64_t sXb,
               int64_t sXn, int64_t sXm, double epsilon, int top_k) {
    if (dtype < SK_FP32 || dtype > SK_FP16) return fail(SK_ERR_ARG, "unknown element type");
    const int rc = check_problem(reinterpret_cast<const float*>(X), B, N, M, epsilon);
    if (rc != SK_OK) return rc;
    if (M > INT_MAX || N > INT_MAX) return fail(SK_ERR_ARG, "N and M must be below 2^31");
    if (sXm != 1) return fail(SK_ERR_LAYOUT, "the rows must have unit column stride");
    if (sXb < 0 || sXn < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    if ((uintptr_t)X % (dtype == SK_FP32 ? 4 : 2) != 0)
        return fail(SK_ERR_LAYOUT, "the rows are not aligned to their elements");
    if (top_k < 0 || top_k > 32 || top_k > M)
        return fail(SK_ERR_ARG, "top_k must lie between 0 and min(32, M)");
    return SK_OK;
}

}  // namespace
}  // namespace sk

extern "C" {

size_t sk_row_logprobs_workspace_bytes(int64_t B, int64_t M) {
    if (B <= 0 || M <= 0) return 0;
    return sk::align_up(sizeof(float) * (size_t)B * M);
}

int sk_row_logprobs(const void* X, int dtype, int64_t B, int64_t N, int64_t M, int64_t sXb,
                    int64_t sXn, int64_t sXm, const float* g, double epsilon, int negate,
                    const uint8_t* mask_a, const uint8_t* mask_b, const int64_t* targets,
                    int top_k, float* lse, float* logprob, float* entropy, float* top_logprob,
                    int64_t* top_index, float* stats, void* workspace, size_t workspace_bytes,
                    void* stream) {
    using namespace sk;
    clear_error();
    const int rc = check_rows(X, dtype, B, N, M, sXb, sXn, sXm, epsilon, top_k);
    if (rc != SK_OK) return rc;
    if ((targets == nullptr) != (logprob == nullptr))
        return fail(SK_ERR_ARG, "targets and logprob go together");
    if (top_k > 0 && (!top_logprob || !top_index))
        return fail(SK_ERR_ARG, "top_k needs top_logprob and top_index");
    if (mask_b && (!workspace || workspace_bytes < sk_row_logprobs_workspace_bytes(B, M)))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_row_logprobs with mask_b");
    cudaStream_t s = (cudaStream_t)stream;
    const int fm = fold_mask(&g, mask_b, B * M, workspace, s);
    if (fm != SK_OK) return fm;
    RowProbArgs A{};
    A.X = X;
    A.N = N;
    A.M = M;
    A.sXb = sXb;
    A.sXn = sXn;
    A.rows = B * N;
    A.g = g;
    A.mask_a = mask_a;
    A.sign = negate ? -1.f : 1.f;
    A.k = (float)(1.0 / epsilon);
    A.targets = targets;
    A.top_k = top_k;
    A.lse = lse;
    A.logprob = logprob;
    A.entropy = entropy;
    A.top_lp = top_logprob;
    A.top_idx = top_index;
    A.stats = reinterpret_cast<float2*>(stats);
    const bool masked = mask_b != nullptr;
    if (dtype == SK_FP32) return launch_rows_typed<float>(A, masked, s);
    if (dtype == SK_BF16) return launch_rows_typed<__nv_bfloat16>(A, masked, s);
    return launch_rows_typed<__half>(A, masked, s);
}

size_t sk_row_logprobs_backward_workspace_bytes(int64_t B, int64_t N, int64_t M) {
    if (B <= 0 || N <= 0 || M <= 0) return 0;
    int64_t nb = 0, br = 0, most = 1;
    for (int elem = 2; elem <= 4; elem += 2) {
        sk::bwd_bands(B, N, M, true, elem, &nb, &br);
        most = std::max(most, nb);
    }
    return sk_row_logprobs_workspace_bytes(B, M) + sk::align_up(sizeof(float) * (size_t)B * most * M);
}

int sk_row_logprobs_backward(const void* X, int dtype, int64_t B, int64_t N, int64_t M,
                             int64_t sXb, int64_t sXn, int64_t sXm, const float* g,
                             double epsilon, int negate, const uint8_t* mask_b,
                             const int64_t* targets, int top_k, const int64_t* top_index,
                             const float* stats, const float* entropy, const float* grad_lse,
                             const float* grad_logprob, const float* grad_entropy,
                             const float* grad_top, void* dX, float* dg, void* workspace,
                             size_t workspace_bytes, void* stream) {
    using namespace sk;
    clear_error();
    const int rc = check_rows(X, dtype, B, N, M, sXb, sXn, sXm, epsilon, top_k);
    if (rc != SK_OK) return rc;
    if (!stats) return fail(SK_ERR_ARG, "stats is NULL");
    if (grad_logprob && !targets) return fail(SK_ERR_ARG, "grad_logprob needs targets");
    if (grad_entropy && !entropy) return fail(SK_ERR_ARG, "grad_entropy needs entropy");
    if (grad_top && (top_k <= 0 || !top_index))
        return fail(SK_ERR_ARG, "grad_top needs top_k and top_index");
    if (!dX && !dg) return fail(SK_ERR_ARG, "dX and dg are both NULL");
    if (dX && (uintptr_t)dX % 16 != 0) return fail(SK_ERR_LAYOUT, "dX is not 16-byte aligned");
    if ((dg || mask_b) && (!workspace || workspace_bytes <
                                             sk_row_logprobs_backward_workspace_bytes(B, N, M)))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_row_logprobs_backward");
    cudaStream_t s = (cudaStream_t)stream;
    const int fm = fold_mask(&g, mask_b, B * M, workspace, s);
    if (fm != SK_OK) return fm;
    RowProbBwdArgs A{};
    A.X = X;
    A.N = N;
    A.M = M;
    A.sXb = sXb;
    A.sXn = sXn;
    A.B = B;
    A.g = g;
    A.sign = negate ? -1.f : 1.f;
    A.k = (float)(1.0 / epsilon);
    A.targets = targets;
    A.top_k = top_k;
    A.top_idx = top_index;
    A.stats = reinterpret_cast<const float2*>(stats);
    A.entropy = entropy;
    A.g_lse = grad_lse;
    A.g_lp = grad_logprob;
    A.g_ent = grad_entropy;
    A.g_top = grad_top;
    A.dX = dX;
    if (dg) A.partial = (float*)((char*)workspace + sk_row_logprobs_workspace_bytes(B, M));
    bwd_bands(B, N, M, dg != nullptr, dtype == SK_FP32 ? 4 : 2, &A.bands, &A.band_rows);
    const bool masked = mask_b != nullptr;
    if (dtype == SK_FP32) return launch_bwd_typed<float>(A, masked, dg, s);
    if (dtype == SK_BF16) return launch_bwd_typed<__nv_bfloat16>(A, masked, dg, s);
    return launch_bwd_typed<__half>(A, masked, dg, s);
}

}  // extern "C"
