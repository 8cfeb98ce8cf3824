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
#include <float.h>
#include <limits.h>

#include <algorithm>
#include <cmath>

#include "sk_common.cuh"
#include "sk_internal.h"
#include "sk_tma.cuh"

namespace sk {
namespace {

namespace cg = cooperative_groups;

constexpr float kNegInf = -INFINITY;
// An exponent (base 2, or e) that stands for all lower ones, -inf among them,
// where it is a factor of its own power: that power is 0 far above it, and
// 0 * -inf would be NaN.
constexpr float kFarBelow = -1e4f;

// Measured on a B200 (a copy: 6.55 TB/s): 8192 x 65536 bf16 187 us (5.7 TB/s); 4096 x
// 50001 bf16 85 us (4.8 TB/s), 110 us with the best 5; 16 x 2048 x 2048 fp32 59 us (4.6
// TB/s), 64 us with g and a mask, 86 us with the best 4 too; 1 x 131072 bf16 with the
// best 20 12 us. Issue slots are 55-74% busy: about 8 instructions a value where the
// arithmetic needs 5.
struct RowProbArgs {
    const void* X;
    int64_t N, M, sXb, sXn;
    int64_t B;
    int per_cta;            // rows of one item to a CTA
    unsigned groups;        // CTAs of an item
    bool staged;            // each CTA holds g (and mask_b) in shared memory
    bool vectors;           // every row starts on 16 bytes
    const float* g;         // (B,M) or NULL; -inf where mask_b leaves a column out
    const uint8_t* mask_b;  // (B,M) or NULL: still to be folded in (staged)
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
// kMasked: the same, and -inf where g_j is -inf whatever X holds: a column mask is
// folded into g beforehand, because in the rows' loop a byte mask cost as much as
// all the rest (16 x 2048 x 2048 fp32 on a B200: 154 us against 93 us with g
// alone). g is read from shared memory where it fits: loads from L1 come back
// behind the row's own, out of DRAM (115 us against 60 us without g).
enum Shape { kPlain = 0, kAffine = 1, kMasked = 2 };

extern __shared__ __align__(16) float staged_g[];

struct RowShape {
    const float* g;  // this item's, or NULL
    float sign;
    bool staged;  // g is in staged_g
    bool vec;     // g is 16-byte aligned at the row's vectors
};

template <int SHAPE>
__device__ __forceinline__ float shaped1(float v, float g, float sign) {
    const float x = fmaf(v, sign, g);  // exact product: one rounding
    return SHAPE == kMasked && g == kNegInf ? kNegInf : x;
}

template <int SHAPE>
__device__ __forceinline__ float shaped(float v, const RowShape& rs, int64_t j) {
    if (SHAPE == kPlain) return v;
    const float g = rs.staged ? staged_g[j] : rs.g ? __ldg(rs.g + j) : 0.f;
    return shaped1<SHAPE>(v, g, rs.sign);
}

// 2 * V2 consecutive values from column j on.
template <int SHAPE, int V2>
__device__ __forceinline__ void shape_pairs(float2* x, const RowShape& rs, int64_t j) {
    if (SHAPE == kPlain) return;
    float2 g[V2];
    if (rs.staged) {
        const float* const p = staged_g + j;
        if (rs.vec) {
#pragma unroll
            for (int e = 0; e < V2; e += 2) {
                const float4 v = *reinterpret_cast<const float4*>(p + 2 * e);
                g[e] = make_float2(v.x, v.y);
                g[e + 1] = make_float2(v.z, v.w);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V2; ++e) g[e] = make_float2(p[2 * e], p[2 * e + 1]);
        }
    } else if (!rs.g) {
#pragma unroll
        for (int e = 0; e < V2; ++e) g[e] = make_float2(0.f, 0.f);
    } else if (rs.vec) {
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
                                              int64_t lead, bool staged = false) {
    RowShape rs;
    rs.g = g ? g + b * M : nullptr;
    rs.sign = sign;
    rs.staged = staged;
    rs.vec = staged ? (lead & 3) == 0 : (reinterpret_cast<uintptr_t>(rs.g + lead) & 15) == 0;
    return rs;
}

__host__ __device__ constexpr int align16(int bytes) { return (bytes + 15) / 16 * 16; }

// An item's g with its mask folded in, into staged_g, by the CTA.
__device__ __forceinline__ void stage_g(const RowProbArgs& A, int64_t b, int threads) {
    for (int j = threadIdx.x; j < (int)A.M; j += threads) {
        const float v = A.g ? A.g[b * A.M + j] : 0.f;
        staged_g[j] = A.mask_b && !A.mask_b[b * A.M + j] ? kNegInf : v;
    }
    __syncthreads();
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
        constexpr int C = V2 >= 8 ? V2 / 4 : 1;  // chains of sums side by side
        float2 ss[C], uu[C];
#pragma unroll
        for (int c = 0; c < C; ++c) ss[c] = uu[c] = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < V2; ++e) {
            const float2 y = __fmul2_rn(__fadd2_rn(x[e], nm), kk);
            const float2 t = make_float2(ex2(y.x), ex2(y.y));
            ss[e % C] = __fadd2_rn(ss[e % C], t);
            uu[e % C] = __ffma2_rn(
                t, BOUND ? make_float2(fmaxf(y.x, kFarBelow), fmaxf(y.y, kFarBelow)) : y,
                uu[e % C]);
        }
#pragma unroll
        for (int c = C / 2; c > 0; c /= 2)
#pragma unroll
            for (int i = 0; i < c; ++i) {
                ss[i] = __fadd2_rn(ss[i], ss[i + c]);
                uu[i] = __fadd2_rn(uu[i], uu[i + c]);
            }
        float du = uu[0].x + uu[0].y;
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
        s += ss[0].x + ss[0].y;
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

constexpr int kListCap = 64;  // entries of a warp's list, two to a lane

// Sort a warp's list of n entries in shared memory and keep the best k; the
// number kept. (Out of line: it is called where a list is full and once a row.)
__device__ __noinline__ int keep_best(float* v, int* i, int n, int k, int lane) {
    __syncwarp();
    if (n <= 32) {
        const float ev = lane < n ? v[lane] : kNegInf;
        const int ei = lane < n ? i[lane] : INT_MAX;
        int rank = lane < n ? 0 : 32;
        for (int l = 0; l < n; ++l)
            rank +=
                beats(__shfl_sync(0xffffffffu, ev, l), __shfl_sync(0xffffffffu, ei, l), ev, ei);
        if (rank < k) {
            v[rank] = ev;
            i[rank] = ei;
        }
    } else {
        constexpr int P = kListCap / 32;
        float ev[P];
        int ei[P], rank[P];
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
            for (int q = 0; q < P; ++q) rank[q] += beats(w, wi, ev[q], ei[q]);
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < P; ++q)
            if (rank[q] < k) {
                v[rank[q]] = ev[q];
                i[rank[q]] = ei[q];
            }
    }
    __syncwarp();
    return min(n, k);
}

// A warp's candidates for the best k, in shared memory, in any order.
struct TopList {
    float* v;
    int* i;
    int n = 0;
    float kth = kNegInf;  // the k-th when the list last ran full
    int kth_i = INT_MAX;

    __device__ __forceinline__ void keep(int k, int lane) { n = keep_best(v, i, n, k, lane); }
    // One candidate a lane; -inf, NaN, what is below `floor` and what does not
    // beat the k-th entry are passed over.
    __device__ __forceinline__ void offer(float cv, int ci, int k, float floor, int lane) {
        bool in = cv >= floor && cv > kNegInf && beats(cv, ci, kth, kth_i);
        unsigned who = __ballot_sync(0xffffffffu, in);
        if (!who) return;
        if (n + __popc(who) > kListCap) {
            keep(k, lane);  // (more than k were in it)
            kth = v[k - 1];
            kth_i = i[k - 1];
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
    // Of the lane's 2 * P values those from `floor` on (mostly one or none);
    // column(e): the column of value e.
    template <int P, typename F>
    __device__ __forceinline__ void offer_pairs(const float2* x, F column, int k, float floor,
                                                int lane) {
        unsigned marks = 0;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            if (x[e].x >= floor) marks |= 1u << (2 * e);
            if (x[e].y >= floor) marks |= 2u << (2 * e);
        }
        if (kth >= floor) {
            // the list ran full: rows of equal values end here
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if (!beats(x[e].x, column(2 * e), kth, kth_i)) marks &= ~(1u << (2 * e));
                if (!beats(x[e].y, column(2 * e + 1), kth, kth_i)) marks &= ~(2u << (2 * e));
            }
        }
        while (__any_sync(0xffffffffu, marks != 0)) {
            float w = kNegInf;
            const int at = marks ? __ffs(marks) - 1 : 0;
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if (at == 2 * e) w = x[e].x;
                if (at == 2 * e + 1) w = x[e].y;
            }
            offer(marks ? w : kNegInf, column(at), k, floor, lane);
            marks &= marks - 1;
        }
    }
};

constexpr int kRowWarps = 8;  // most warps of a CTA

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

constexpr int kStash = 32;

// What the W warps of a row share.
template <bool TOP, int W>
struct RowShared {
    float m[W], s[W], u[W];
};
template <int W>
struct RowShared<true, W> {
    float m[W], s[W], u[W];
    float high[32];    // the largest lane maxima of each warp, 32 in all
    int from[W][32];   // first vectors of the lanes that are read again
    int n[W];
    float lv[W][kListCap];
    int li[W][kListCap];
    float ov[32];  // the best k, sorted
    int oi[32];
};

// Vectors with a candidate, of rows that are held in registers.
template <bool ON>
struct RowStash {};
template <>
struct RowStash<true> {
    uint4 v[kRowWarps][kStash];
    int at[kRowWarps][kStash], n[kRowWarps];
};

// The best k of `lists` unsorted lists of at most 32 entries into ov / oi (-inf
// and -1 where there are fewer), by the row's warps, at least as many as lists;
// `sync` is their barrier.
template <int W, typename Sync>
__device__ __forceinline__ void select_best(RowShared<true, W>& sh, int lists, int k, int warp,
                                            int lane, Sync sync) {
    int total = 0;
    for (int l = 0; l < lists; ++l) total += sh.n[l];
    if (warp == 0) {
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
        sync();
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
    sync();
}

// W warps' lane maxima to a value that at least k lanes reach: 32 / W maxima of
// each warp stand for its lanes.
template <int W, typename Sync>
__device__ __forceinline__ float lane_bound(RowShared<true, W>& sh, float best, int k, int warp,
                                            int lane, Sync sync) {
    if (W == 1) return fmaxf(warp_rth_largest(best, k, lane), -FLT_MAX);
    constexpr int HI = 32 / W;
    unsigned o = ordered(best), mine = 0;
#pragma unroll
    for (int q = 0; q < HI; ++q) {
        const unsigned t = __reduce_max_sync(0xffffffffu, o);
        if (lane == q) mine = t;
        if (lane == __ffs(__ballot_sync(0xffffffffu, o == t)) - 1) o = 0;
    }
    if (lane < HI) sh.high[warp * HI + lane] = unordered(mine);
    sync();
    return fmaxf(warp_rth_largest(sh.high[lane], k, lane), -FLT_MAX);
}

// Read the vectors of the warp's lanes that reach `bound` again, one to each lane
// at a time: lane l's are base0 + l + q * 32 + c * step, q < U.
template <typename T, int SHAPE, int U>
__device__ __forceinline__ void offer_again(TopList& top, int* from, float best, float bound,
                                            const T* X, const RowShape& rs, int lead, int nv,
                                            int base0, int step, int k, int lane) {
    constexpr int V = Vec<T>::n, V2 = V / 2;
    const bool held = best >= bound;
    const unsigned who = __ballot_sync(0xffffffffu, held);
    if (held) from[__popc(who & ((1u << lane) - 1u))] = base0 + lane;
    __syncwarp();
    const int per = (nv - base0 + step - 1) / step * U;  // of a lane, at most
    const int all = __popc(who) * per;
    const uint4* const body = reinterpret_cast<const uint4*>(X + lead);
    for (int c = 0; c < all; c += 32) {
        const int f = c + lane, q = f / per, s = f - q * per;
        const int at = f < all ? from[q] + s / U * step + s % U * 32 : nv;
        float2 y[V2];
        if (at < nv) {
            unpack2(ld_stream16(body + at), y, X);
            shape_pairs<SHAPE, V2>(y, rs, lead + (int64_t)at * V);
        } else {
#pragma unroll
            for (int e = 0; e < V2; ++e) y[e] = make_float2(kNegInf, kNegInf);
        }
        top.offer_pairs<V2>(y, [&](int e) { return lead + at * V + e; }, k, bound, lane);
    }
}

// A finished row's statistics, written by one lane (`writes`); value(t) is x of
// column t. Returns log s.
template <typename F>
__device__ __forceinline__ float write_stats(const RowProbArgs& A, int64_t row, const Moments& mo,
                                             bool writes, F value) {
    // an empty row keeps s = 0; a row of NaN alone has s = NaN
    const bool none = mo.m == kNegInf && mo.s == 0.f;
    const float logs = none ? 0.f : logf(mo.s);
    if (writes) {
        if (A.stats) A.stats[row] = make_float2(none ? kNegInf : mo.m, logs);
        if (A.lse) A.lse[row] = none ? kNegInf : fmaf(mo.m, A.k, logs);
        if (A.entropy) A.entropy[row] = none ? 0.f : logs - kLn2 * (mo.u / mo.s);
        if (A.logprob) {
            const int64_t t = A.targets[row];
            float lp = 0.f;
            if (t >= A.M) lp = NAN;
            else if (t >= 0) lp = none ? kNegInf : fmaf(value(t) - mo.m, A.k, -logs);
            A.logprob[row] = lp;
        }
    }
    return logs;
}

// Its `at`-th best column; `held` is false where there are fewer.
__device__ __forceinline__ void write_best(const RowProbArgs& A, int64_t row, const Moments& mo,
                                           float logs, int at, bool held, float v, int i) {
    A.top_lp[row * A.top_k + at] = held ? fmaf(v - mo.m, A.k, -logs) : kNegInf;
    A.top_idx[row * A.top_k + at] = held ? i : -1;
}

// A finished row's outputs, by one warp; its best columns are lv / li [k].
template <typename T, int SHAPE, bool TOP>
__device__ __forceinline__ void write_row(const RowProbArgs& A, int64_t row, const T* X,
                                          const RowShape& rs, const Moments& mo, const float* lv,
                                          const int* li, int have, int lane) {
    const float logs = write_stats(A, row, mo, lane == 0, [&](int64_t t) {
        return shaped<SHAPE>(widen(X[t]), rs, t);
    });
    if (TOP && lane < A.top_k) {
        const bool held = lane < have && li[lane] >= 0;
        write_best(A, row, mo, logs, lane, held, held ? lv[lane] : 0.f, held ? li[lane] : -1);
    }
}

// The row's ends, one column to a lane: up to V - 1 before the first whole
// vector and as many behind the last.
template <typename T, int SHAPE>
__device__ __forceinline__ float row_ends(const T* X, const RowShape& rs, int lead, int tail,
                                          int M, int lane, int& column) {
    column = lane < 16 ? lane : tail + lane - 16;
    const bool on = lane < 16 ? lane < lead : column < M;
    return on ? shaped<SHAPE>(widen(X[column]), rs, column) : kNegInf;
}

constexpr int kGroupTop = 8;  // most best columns in k_row_group: one to a lane

// Rows of up to G * P columns, as a router's experts: G lanes to a row, P values
// each, 32 / G rows to a warp at once, since joining 32 lanes costs such rows more
// than reading them. A lane's columns are the same in every row of an item, so g
// and its mask stay in registers. A best column costs a maximum over the lanes'
// own best ones, after which the lane that held it looks for its next.
// 16 x 32768 x 64 fp32 with g, best 2: 76 us (335 us by a warp to a row); 4 x 8192:
// 8 us (27 us). 32768 x 128 bf16, best 8: 22 us (42 us).
template <typename T, int SHAPE, bool TOP, int P, int G>
__global__ void __launch_bounds__(32 * kRowWarps, P == 8 ? 4 : 3)
    k_row_group(const RowProbArgs A) {
    constexpr int V = Vec<T>::n, Q = P / V;
    constexpr int kGroups = 32 * kRowWarps / G;
    static_assert(P % V == 0, "whole vectors");
    const int gl = threadIdx.x % G, group = threadIdx.x / G;
    const unsigned item = blockIdx.x / A.groups;
    const int64_t b = item, r0 = (int64_t)(blockIdx.x - item * A.groups) * A.per_cta;
    const int64_t r1 = min(A.N, r0 + A.per_cta);
    const T* const Xb = reinterpret_cast<const T*>(A.X) + b * A.sXb;
    const int M = (int)A.M, k = A.top_k;
    const float k2 = A.k * kLog2e;
    // column of the lane's value e
    auto column = [&](int e) { return (e / V * G + gl) * V + e % V; };
    auto g_at = [&](int64_t j) {
        const float v = A.g ? A.g[b * M + j] : 0.f;
        return SHAPE == kMasked && A.mask_b && !A.mask_b[b * M + j] ? kNegInf : v;
    };
    uint4 raw[Q];
    bool off = true;  // a row behind the last, or left out by mask_a
    auto load = [&](int64_t r) {
        off = r >= r1 || (A.mask_a && !A.mask_a[b * A.N + r]);
        const T* const X = Xb + r * A.sXn;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int j = column(q * V);
            raw[q] = make_uint4(0, 0, 0, 0);
            if (off || j >= M) continue;
            if (A.vectors && j + V <= M) {
                raw[q] = ld_stream16(X + j);
            } else {
                T t[V];
#pragma unroll
                for (int e = 0; e < V; ++e) t[e] = j + e < M ? X[j + e] : T(0.f);
                memcpy(&raw[q], t, 16);
            }
        }
    };
    load(r0 + group);
    float2 g[P / 2];  // -inf behind the last column
#pragma unroll
    for (int e = 0; e < P; e += 2) {
        const int j = column(e);
        g[e / 2].x = j >= M ? kNegInf : SHAPE == kPlain ? 0.f : g_at(j);
        g[e / 2].y = j + 1 >= M ? kNegInf : SHAPE == kPlain ? 0.f : g_at(j + 1);
    }

    // every lane of a warp stays to the end: the groups share its shuffles
    for (int64_t r = r0 + group; r - group < r1; r += kGroups) {
        const int64_t row = b * A.N + r;
        const bool out = off, in = r < r1;
        float2 x[P / 2];
#pragma unroll
        for (int q = 0; q < Q; ++q) unpack2(raw[q], x + q * (V / 2), (const T*)nullptr);
        load(r + kGroups);
        float cm = kNegInf;
#pragma unroll
        for (int e = 0; e < P / 2; ++e) {
            if (SHAPE != kPlain) x[e] = __ffma2_rn(x[e], make_float2(A.sign, A.sign), g[e]);
            // masked columns, whatever was read there (and what is no column, where
            // the sum with g has not made it so)
            if (out || (SHAPE != kAffine && g[e].x == kNegInf)) x[e].x = kNegInf;
            if (out || (SHAPE != kAffine && g[e].y == kNegInf)) x[e].y = kNegInf;
            cm = fmaxf(cm, fmaxf(x[e].x, x[e].y));
        }
        Moments mo;
        mo.fold<true>(x, cm, k2);
        float m = mo.m;
#pragma unroll
        for (int d = G / 2; d > 0; d /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        mo.move_to(m, k2);
#pragma unroll
        for (int d = G / 2; d > 0; d /= 2) {
            mo.s += __shfl_xor_sync(0xffffffffu, mo.s, d);
            mo.u += __shfl_xor_sync(0xffffffffu, mo.u, d);
        }

        float bv = kNegInf;  // the lane's entry of the best k
        int bj = INT_MAX;
        if constexpr (TOP) {
            for (int i = 0; i < k; ++i) {
                float v = kNegInf;  // the lane's best value that is left
                int j = INT_MAX;
#pragma unroll
                for (int e = 0; e < P / 2; ++e) {
                    if (x[e].x > v) v = x[e].x, j = column(2 * e);
                    if (x[e].y > v) v = x[e].y, j = column(2 * e + 1);
                }
                float w = v;
                int wj = j;
#pragma unroll
                for (int d = G / 2; d > 0; d /= 2) {
                    const float ov = __shfl_xor_sync(0xffffffffu, w, d);
                    const int oj = __shfl_xor_sync(0xffffffffu, wj, d);
                    if (beats(ov, oj, w, wj)) w = ov, wj = oj;
                }
                if (gl == i) bv = w, bj = wj;
                if (j == wj) {  // this lane's: not again (INT_MAX: none is left)
#pragma unroll
                    for (int e = 0; e < P / 2; ++e) {
                        if (column(2 * e) == wj) x[e].x = kNegInf;
                        if (column(2 * e + 1) == wj) x[e].y = kNegInf;
                    }
                }
            }
        }
        if (!in) continue;
        const float logs = write_stats(A, row, mo, gl == 0, [&](int64_t t) {
            const float v = widen(Xb[r * A.sXn + t]);
            return SHAPE == kPlain ? v : shaped1<SHAPE>(v, g_at(t), A.sign);
        });
        if (TOP && gl < k) write_best(A, row, mo, logs, gl, bj != INT_MAX, bv, bj);
    }
}

// Short rows: a warp to a row, which is at most U vectors of 16 bytes a lane,
// loaded at once and held in registers.
template <typename T, int SHAPE, bool TOP, int U>
__global__ void __launch_bounds__(32 * kRowWarps, U == 1 ? 4 : 3)
    k_row_held(const RowProbArgs A) {
    constexpr int V = Vec<T>::n, V2 = V / 2;
    constexpr int H = U == 1 ? 1 : 16 / V;  // vectors folded at once: 16 values
    static_assert(U % H == 0, "whole folds");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ RowStash<TOP> stash;
    __shared__ RowShared<TOP, 1> shared[kRowWarps];
    RowShared<TOP, 1>& sh = shared[warp];
    const unsigned item = blockIdx.x / A.groups;  // (64-bit divisions cost as much as a row)
    const int64_t b = item, r0 = (int64_t)(blockIdx.x - item * A.groups) * A.per_cta;
    const T* const Xb = reinterpret_cast<const T*>(A.X) + b * A.sXb;
    const int M = (int)A.M, k = A.top_k;
    const float k2 = A.k * kLog2e;
    const int64_t r1 = min(A.N, r0 + A.per_cta);
    const T* X = nullptr;
    int lead = 0, nv = 0;
    uint4 raw[U];
    auto load = [&](int64_t r) {
        X = Xb + r * A.sXn;
        lead = (int)row_lead(X, A.M);
        nv = A.mask_a && !A.mask_a[b * A.N + r] ? 0 : (M - lead) / V;
        const uint4* const body = reinterpret_cast<const uint4*>(X + lead);
#pragma unroll
        for (int q = 0; q < U; ++q)
            if (lane + q * 32 < nv) raw[q] = ld_stream16(body + lane + q * 32);
    };
    if (r0 + warp < r1) load(r0 + warp);
    if (SHAPE != kPlain && A.staged) stage_g(A, b, 32 * kRowWarps);

    for (int64_t r = r0 + warp; r < r1; r += kRowWarps) {
        if (r != r0 + warp) load(r);
        const int64_t row = b * A.N + r;
        const bool masked_row = A.mask_a && !A.mask_a[row];
        const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead, A.staged);
        const int tail = lead + nv * V;
        float end = kNegInf;
        int end_j = 0;
        if (!masked_row && (lead > 0 || tail < M))
            end = row_ends<T, SHAPE>(X, rs, lead, tail, M, lane, end_j);

        Moments mo;
        float high[U];  // largest value of each vector
#pragma unroll
        for (int h = 0; h < U; h += H) {
            float2 x[H * V2];
            float cm = kNegInf;
#pragma unroll
            for (int q = 0; q < H; ++q) {
                const int at = lane + (h + q) * 32;
                float2* const y = x + q * V2;
                unpack2(raw[h + q], y, X);
                if (at < nv) {
                    shape_pairs<SHAPE, V2>(y, rs, lead + (int64_t)at * V);
                } else {
#pragma unroll
                    for (int e = 0; e < V2; ++e) y[e] = make_float2(kNegInf, kNegInf);
                }
                float vm = fmaxf(y[0].x, y[0].y);
#pragma unroll
                for (int e = 1; e < V2; ++e) vm = fmaxf(vm, fmaxf(y[e].x, y[e].y));
                high[h + q] = vm;
                cm = fmaxf(cm, vm);
            }
            mo.fold<SHAPE != kPlain>(x, cm, k2);
        }
        if (!masked_row && (lead > 0 || tail < M)) {
            const float2 e[1] = {make_float2(end, kNegInf)};
            mo.fold<true>(e, end, k2);
        }
        mo.join(k2);

        TopList top;
        if constexpr (TOP) {
            top.v = sh.lv[0];
            top.i = sh.li[0];
            if (lead > 0 || tail < M) top.offer(end, end_j, k, kNegInf, lane);
            float best = kNegInf;
#pragma unroll
            for (int q = 0; q < U; ++q) best = fmaxf(best, high[q]);
            const float bound = fmaxf(warp_rth_largest(best, k, lane), -FLT_MAX);
            // vectors with a candidate to shared memory, then a value to a lane
            if (lane == 0) stash.n[warp] = 0;
            __syncwarp();
#pragma unroll
            for (int q = 0; q < U; ++q)
                if (high[q] >= bound) {
                    const int at = atomicAdd(&stash.n[warp], 1);
                    if (at < kStash) {
                        stash.v[warp][at] = raw[q];
                        stash.at[warp][at] = lane + q * 32;
                    }
                }
            __syncwarp();
            const int have = stash.n[warp];
            if (have <= kStash) {
                for (int c = 0; c < have * V; c += 32) {
                    float v = kNegInf;
                    int j = 0;
                    if (c + lane < have * V) {
                        const int q = (c + lane) / V, e = (c + lane) % V;
                        j = lead + stash.at[warp][q] * V + e;
                        v = shaped<SHAPE>(
                            widen(reinterpret_cast<const T*>(&stash.v[warp][q])[e]), rs, j);
                    }
                    top.offer(v, j, k, bound, lane);
                }
            } else {  // many equal values
                offer_again<T, SHAPE, U>(top, sh.from[0], best, bound, X, rs, lead, nv, 0,
                                         32 * U, k, lane);
            }
            top.keep(k, lane);
        }
        write_row<T, SHAPE, TOP>(A, row, X, rs, mo, top.v, top.i, top.n, lane);
        __syncwarp();  // the list is read
    }
}

// Long rows: a CTA of 8 warps to a row, or a cluster of CTAs where there are few
// rows, joined over distributed shared memory by rank 0. As a step's vectors are
// unpacked the loads of the next one take their registers.
template <typename T, int SHAPE, bool TOP>
__global__ void __launch_bounds__(32 * kRowWarps, SHAPE ? 3 : 4)
    k_row_cta(const RowProbArgs A) {
    constexpr int V = Vec<T>::n, V2 = V / 2, U = 4;
    constexpr int H = 16 / V;  // vectors folded at once: 16 values
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ RowShared<TOP, kRowWarps> sh;
    const int parts = (int)cg::this_cluster().num_blocks();
    const int part = (int)cg::this_cluster().block_rank();
    const unsigned of_all = blockIdx.x / (unsigned)parts, item = of_all / (unsigned)A.N;
    const int64_t row = of_all, b = item, n = of_all - item * (unsigned)A.N;
    const T* const X = reinterpret_cast<const T*>(A.X) + b * A.sXb + n * A.sXn;
    const int M = (int)A.M, k = A.top_k;
    const int lead = (int)row_lead(X, A.M);
    const float k2 = A.k * kLog2e;
    const bool masked_row = A.mask_a && !A.mask_a[row];
    const int nv = masked_row ? 0 : (M - lead) / V;
    const int wid = part * kRowWarps + warp, step = parts * kRowWarps * 32 * U;
    const int base = wid * 32 * U + lane;
    const uint4* const body = reinterpret_cast<const uint4*>(X + lead);
    if (SHAPE != kPlain && A.staged) stage_g(A, b, 32 * kRowWarps);
    const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead, A.staged);
    auto sync = [] { __syncthreads(); };

    Moments mo;
    float best = kNegInf;  // the lane's largest value among whole vectors
    float2 x[H * V2];
    auto fold = [&] {
        float cm = kNegInf;
#pragma unroll
        for (int e = 0; e < H * V2; ++e) cm = fmaxf(cm, fmaxf(x[e].x, x[e].y));
        if (TOP) best = fmaxf(best, cm);
        mo.fold<SHAPE != kPlain>(x, cm, k2);
    };
    int i = base;
    if (wid * 32 * U + 32 * U <= nv) {
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
                    unpack2(raw[h + q], x + q * V2, X);
                    if (more) raw[h + q] = ld_stream16(body + i + step + (h + q) * 32);
                    shape_pairs<SHAPE, V2>(x + q * V2, rs,
                                           lead + (int64_t)(i + (h + q) * 32) * V);
                }
                fold();
            }
            i += step;
            if (!more) break;
        }
    }
    for (; i - lane < nv; i += step) {  // the warp's last step
#pragma unroll
        for (int h = 0; h < U; h += H) {
#pragma unroll
            for (int q = 0; q < H; ++q) {
                const int at = i + (h + q) * 32;
                float2* const y = x + q * V2;
                if (at < nv) {
                    unpack2(ld_stream16(body + at), y, X);
                    shape_pairs<SHAPE, V2>(y, rs, lead + (int64_t)at * V);
                } else {
#pragma unroll
                    for (int e = 0; e < V2; ++e) y[e] = make_float2(kNegInf, kNegInf);
                }
            }
            fold();
        }
    }
    const int tail = lead + nv * V;
    float end = kNegInf;
    int end_j = 0;
    if (!masked_row && wid == 0 && (lead > 0 || tail < M)) {
        end = row_ends<T, SHAPE>(X, rs, lead, tail, M, lane, end_j);
        const float2 e[1] = {make_float2(end, kNegInf)};
        mo.fold<true>(e, end, k2);
    }
    mo.join(k2);
    if (lane == 0) {
        sh.m[warp] = mo.m;
        sh.s[warp] = mo.s;
        sh.u[warp] = mo.u;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const float* lv = nullptr;
    const int* li = nullptr;
    if constexpr (TOP) {
        TopList top;
        top.v = sh.lv[warp];
        top.i = sh.li[warp];
        top.offer(end, end_j, k, kNegInf, lane);
        const float bound = lane_bound<kRowWarps>(sh, best, k, warp, lane, sync);
        offer_again<T, SHAPE, U>(top, sh.from[warp], best, bound, X, rs, lead, nv, wid * 32 * U,
                                 step, k, lane);
        if (top.n > 32) top.keep(k, lane);
        if (lane == 0) sh.n[warp] = top.n;
        __syncthreads();
        select_best<kRowWarps>(sh, kRowWarps, k, warp, lane, sync);
        if (parts > 1) {
            cluster.sync();
            if (part == 0) {
                // the peers' best k into this CTA's lists
                if (warp < parts) {
                    const auto* o = cluster.map_shared_rank(&sh, warp);
                    const float v = lane < k ? o->ov[lane] : kNegInf;
                    const int at = lane < k ? o->oi[lane] : -1;
                    sh.lv[warp][lane] = v;
                    sh.li[warp][lane] = at;
                    const int have = __popc(__ballot_sync(0xffffffffu, at >= 0));
                    if (lane == 0) sh.n[warp] = have;
                }
                __syncthreads();
                select_best<kRowWarps>(sh, parts, k, warp, lane, sync);
            }
        }
        lv = sh.ov;
        li = sh.oi;
    } else {
        if (parts > 1) cluster.sync();
        else __syncthreads();
    }
    if (part == 0 && warp == 0) {
        // up to 8 x 8 parts, two to a lane
        mo = Moments();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int q = (lane + 32 * h) / kRowWarps, w = lane % kRowWarps;
            if (q < parts) {
                const auto* o = parts > 1 ? cluster.map_shared_rank(&sh, q) : &sh;
                mo.merge(o->m[w], o->s[w], o->u[w], k2);
            }
        }
        mo.join(k2);
        write_row<T, SHAPE, TOP>(A, row, X, rs, mo, lv, li, k, lane);
    }
    if (parts > 1) cluster.sync();  // rank 0 has read this CTA's shared memory
}

// Many rows: one CTA of 20 or 28 warps to an SM. Each warp has 4 KB of shared
// memory that a bulk copy fills with its next piece of a row while it works on the
// last one in registers, across rows: the copy goes on while a row is joined and
// its best columns are found. (More stages a warp gained nothing and took the L1
// cache: 16 x 2048 x 2048 fp32 59 us with one, 65 us with two.) TEAM warps share a
// row (1 up to 16 KB, else 4), and the CTA's teams a run of consecutive rows, item
// by item; g stays in shared memory for an item.
constexpr int kAheadVecs = 8;  // vectors of a lane in a copy
constexpr int kAheadBytes = 32 * kAheadVecs * 16;
// Warps of a CTA. Without g 20 with 96 registers beat 28 with 72 (16384 x 4096
// bf16: 36 us against 54 us), with g it is the other way (16 x 2048 x 2048 with a
// mask and top 4: 96 us against 86 us).
template <int SHAPE>
constexpr int stream_warps() {
    return SHAPE == kPlain ? 20 : 28;
}

template <typename T, int SHAPE, bool TOP, int TEAM>
__global__ void __launch_bounds__(stream_warps<SHAPE>() * 32, 1) k_row_stream(const RowProbArgs A) {
    constexpr int V = Vec<T>::n, V2 = V / 2;
    constexpr int H = 32 / V < kAheadVecs ? 32 / V : kAheadVecs;  // vectors folded at once
    constexpr int WARPS = stream_warps<SHAPE>(), TEAMS = WARPS / TEAM;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int team = warp / TEAM, tw = warp % TEAM;
    __shared__ RowShared<TOP, TEAM> shared[TEAMS];
    __shared__ uint64_t bars[WARPS];
    RowShared<TOP, TEAM>& sh = shared[team];
    uint64_t* const full = &bars[warp];
    uint8_t* const buffer = reinterpret_cast<uint8_t*>(staged_g) +
                            (A.staged ? align16((int)A.M * 4) : 0) + warp * kAheadBytes;
    auto sync = [&] {
        if (TEAM == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(TEAM * 32) : "memory");
    };
    if (lane == 0) {
        mbar_init(full, 1);
        mbar_init_fence();
    }
    __syncwarp();

    const int64_t rows = A.B * A.N;  // below 2^31
    const int R0 = (int)(rows * blockIdx.x / gridDim.x);
    const int R1 = (int)(rows * (blockIdx.x + 1) / gridDim.x);
    const unsigned N = (unsigned)A.N;
    const int M = (int)A.M, k = A.top_k;
    const float k2 = A.k * kLog2e;
    const int first = tw * 32 * kAheadVecs, step = TEAM * 32 * kAheadVecs;
    // without g the CTA's rows are one run; with it, runs of an item
    auto run_end = [&](int r) {
        return SHAPE == kPlain ? R1 : (int)min((unsigned)R1, (r / N + 1) * N);
    };
    // a team's rows: of each run the team-th, and every TEAMS-th from there
    auto next_row = [&](int r, int& end) {
        r += TEAMS;
        while (r >= end && end < R1) {
            r = end + team;
            end = run_end(end);
        }
        return r;
    };
    // The copies: the row they are at, where this warp's next step of it lies and
    // how many vectors the row has from there on.
    int ahead_end = run_end(R0), ahead = next_row(R0 + team - TEAMS, ahead_end);
    const T* src = nullptr;
    int left = 0;
    auto open = [&](unsigned row) {
        const unsigned b = row / N;
        const T* const X =
            reinterpret_cast<const T*>(A.X) + b * A.sXb + (int64_t)(row - b * N) * A.sXn;
        const int lead = (int)row_lead(X, A.M);
        src = X + lead + first * V;
        left = A.mask_a && !A.mask_a[row] ? 0 : (M - lead) / V - first;
    };
    if (ahead < R1) open(ahead);
    uint32_t phase = 0;  // of `full`
    // the copy of the next step, once the buffer has been read
    auto issue = [&] {
        while (left <= 0) {
            if (ahead < R1) ahead = next_row(ahead, ahead_end);
            if (ahead >= R1) return;
            open(ahead);
        }
        if (lane == 0) {
            const uint32_t bytes = min(32 * kAheadVecs, left) * 16;
            mbar_expect_tx(full, bytes);
            bulk_g2s(buffer, src, bytes, full);
        }
        src += step * V;
        left -= step;
    };
    issue();

    bool ok = true;
    int end = run_end(R0);
    for (int run = R0; run < R1; run = end, end = run_end(run)) {
        const unsigned item0 = SHAPE == kPlain ? 0 : run / N;
        if (SHAPE != kPlain && A.staged) {
            __syncthreads();  // the last item's g is read
            stage_g(A, item0, WARPS * 32);
        }
        for (int row = run + team; row < end; row += TEAMS) {
            const unsigned b = SHAPE == kPlain ? row / N : item0;
            const int64_t n = row - b * N;
            const T* const X = reinterpret_cast<const T*>(A.X) + b * A.sXb + n * A.sXn;
            const int lead = (int)row_lead(X, A.M);
            const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead, A.staged);
            const bool masked_row = A.mask_a && !A.mask_a[row];
            const int nv = masked_row ? 0 : (M - lead) / V;
            Moments mo;
            float best = kNegInf;
            for (int i = first; i < nv; i += step) {
                if (!mbar_try_wait(full, phase)) ok = mbar_wait(full, phase) && ok;
                __syncwarp();
                phase ^= 1;
                const uint4* const p = reinterpret_cast<const uint4*>(buffer) + lane;
                const bool whole = i + 32 * kAheadVecs <= nv;
#pragma unroll
                for (int h = 0; h < kAheadVecs; h += H) {
                    uint4 raw[H];
#pragma unroll
                    for (int q = 0; q < H; ++q) raw[q] = p[(h + q) * 32];
                    if (h + H == kAheadVecs) {
                        // the buffer is read: loads that are still on their way would
                        // otherwise see what the copy brings
                        fence_async_smem();
                        __syncwarp();
                        issue();
                    }
                    float2 x[H * V2];
                    float cm = kNegInf;
#pragma unroll
                    for (int q = 0; q < H; ++q) {
                        const int at = i + (h + q) * 32 + lane;
                        float2* const y = x + q * V2;
                        unpack2(raw[q], y, X);
                        if (whole || at < nv) {
                            shape_pairs<SHAPE, V2>(y, rs, lead + (int64_t)at * V);
                        } else {
#pragma unroll
                            for (int e = 0; e < V2; ++e) y[e] = make_float2(kNegInf, kNegInf);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < H * V2; ++e) cm = fmaxf(cm, fmaxf(x[e].x, x[e].y));
                    if (TOP) best = fmaxf(best, cm);
                    mo.fold<SHAPE != kPlain>(x, cm, k2);
                }
            }
            const int tail = lead + nv * V;
            float endv = kNegInf;
            int end_j = 0;
            if (!masked_row && tw == 0 && (lead > 0 || tail < M)) {
                endv = row_ends<T, SHAPE>(X, rs, lead, tail, M, lane, end_j);
                const float2 e[1] = {make_float2(endv, kNegInf)};
                mo.fold<true>(e, endv, k2);
            }
            mo.join(k2);
            if (__any_sync(0xffffffffu, !ok)) mo.s = NAN;  // a copy never came: the row says so

            TopList top;
            if constexpr (TOP) {
                top.v = sh.lv[tw];
                top.i = sh.li[tw];
                top.offer(endv, end_j, k, kNegInf, lane);
                const float bound = lane_bound<TEAM>(sh, best, k, tw, lane, sync);
                offer_again<T, SHAPE, kAheadVecs>(top, sh.from[tw], best, bound, X, rs,
                                                 lead, nv, first, step, k, lane);
                if (TEAM == 1 || top.n > 32) top.keep(k, lane);
            }
            if constexpr (TEAM == 1) {
                write_row<T, SHAPE, TOP>(A, row, X, rs, mo, top.v, top.i, top.n, lane);
                __syncwarp();
            } else {
                if (lane == 0) {
                    sh.m[tw] = mo.m;
                    sh.s[tw] = mo.s;
                    sh.u[tw] = mo.u;
                    if constexpr (TOP) sh.n[tw] = top.n;
                }
                sync();
                if constexpr (TOP) select_best<TEAM>(sh, TEAM, k, tw, lane, sync);
                if (tw == 0) {
                    mo = Moments();
                    if (lane < TEAM) mo.merge(sh.m[lane], sh.s[lane], sh.u[lane], k2);
                    mo.join(k2);
                    const float* lv = nullptr;
                    const int* li = nullptr;
                    if constexpr (TOP) {
                        lv = sh.ov;
                        li = sh.oi;
                    }
                    write_row<T, SHAPE, TOP>(A, row, X, rs, mo, lv, li, k, lane);
                }
                sync();  // what the team shares of this row is read
            }
        }
    }
    // a copy that a wait gave up on may still be on its way
    if (!ok) mbar_wait(full, phase ^ 1, 1u << 16);
}

constexpr int64_t kStagedMax = 16384;  // columns of g that are held in shared memory

// Let a kernel have `most` bytes of dynamic shared memory where a launch takes more
// than any kernel may. The limit is one value for all threads of the process: it is
// the kernel's largest, whatever this launch takes, so that no call lowers another's.
template <typename K>
int allow_smem(K kernel, size_t bytes, size_t most) {
    if (bytes > 16384)
        SK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)most));
    return SK_OK;
}
constexpr size_t kStagedBytes = kStagedMax * sizeof(float);

template <typename T, int SHAPE, bool TOP, int U>
int launch_held(RowProbArgs A, int per_cta, cudaStream_t s) {
    A.per_cta = per_cta;
    // a row of one vector a lane waits longer for the CTA's g than for its own from L1
    if (U == 1 && !A.mask_b) A.staged = false;
    A.groups = (unsigned)((A.N + per_cta - 1) / per_cta);
    const int64_t ctas = A.groups * A.B;
    if (ctas > INT_MAX) return fail(SK_ERR_ARG, "B * N is too large");
    const size_t smem = A.staged ? align16((int)A.M * 4) : 0;  // at most 4 KB
    k_row_held<T, SHAPE, TOP, U><<<(unsigned)ctas, 32 * kRowWarps, smem, s>>>(A);
    SK_LAUNCHED("k_row_held");
    return SK_OK;
}

template <typename T, int SHAPE, bool TOP, int P, int G>
int launch_group(RowProbArgs A, cudaStream_t s) {
    constexpr int groups = 32 * kRowWarps / G;
    // one wave of CTAs, 4 an SM, then more rows each
    const int64_t want = (A.B * A.N / (148 * 4) + groups - 1) / groups * groups;
    A.per_cta = (int)std::max<int64_t>(groups, std::min<int64_t>(want, 8 * groups));
    A.groups = (unsigned)((A.N + A.per_cta - 1) / A.per_cta);
    const int64_t ctas = A.groups * A.B;
    if (ctas > INT_MAX) return fail(SK_ERR_ARG, "B * N is too large");
    const int64_t align = 16 / (int64_t)sizeof(T);
    A.vectors = (uintptr_t)A.X % 16 == 0 && A.sXb % align == 0 && A.sXn % align == 0;
    k_row_group<T, SHAPE, TOP, P, G><<<(unsigned)ctas, 32 * kRowWarps, 0, s>>>(A);
    SK_LAUNCHED("k_row_group");
    return SK_OK;
}

template <typename T, int SHAPE, bool TOP>
int launch_cta(const RowProbArgs& A, int cluster, cudaStream_t s) {
    const int64_t ctas = A.B * A.N * cluster;
    if (ctas > INT_MAX) return fail(SK_ERR_ARG, "B * N is too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(32 * kRowWarps);
    cfg.dynamicSmemBytes = A.staged ? align16((int)A.M * 4) : 0;
    cfg.stream = s;
    const int rc = allow_smem(k_row_cta<T, SHAPE, TOP>, cfg.dynamicSmemBytes, kStagedBytes);
    if (rc != SK_OK) return rc;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SK_CUDA(cudaLaunchKernelEx(&cfg, k_row_cta<T, SHAPE, TOP>, A));
    return SK_OK;
}

template <typename T, int SHAPE, bool TOP, int TEAM>
int launch_stream(const RowProbArgs& A, cudaStream_t s) {
    constexpr int warps = stream_warps<SHAPE>(), teams = warps / TEAM;
    constexpr size_t ahead = (size_t)warps * kAheadBytes, most = kStagedBytes + ahead;
    static_assert(most + teams * sizeof(RowShared<TOP, TEAM>) + warps * 8 <= 232448,
                  "shared memory of one CTA");
    const size_t smem = (A.staged ? align16((int)A.M * 4) : 0) + ahead;
    const int rc = allow_smem(k_row_stream<T, SHAPE, TOP, TEAM>, smem, most);
    if (rc != SK_OK) return rc;
    const int64_t rows = A.B * A.N;
    const unsigned grid = (unsigned)std::min<int64_t>(148, (rows + teams - 1) / teams);
    k_row_stream<T, SHAPE, TOP, TEAM><<<grid, warps * 32, smem, s>>>(A);
    SK_LAUNCHED("k_row_stream");
    return SK_OK;
}

// How the rows are split. Up to 512 columns several lanes hold a row, as long as the
// best k are few: each costs a scan of the lanes' values (32768 x 512 fp32 with
// g, none: 22 us against 28 us by a warp to a row; best 8: 87 us against 54 us; 256
// columns, best 8: 46 us against 51 us). Other rows up to 2 KB are held by a warp and
// nothing is joined or read twice; a CTA takes at least a row of an item to each warp.
// Longer rows are streamed where there are enough to keep 148 CTAs busy (and, with
// a g that is staged per item, items of some length): up to 16 KB by a warp each
// (16384 x 8192 bf16: 61 us, by four 83 us, by a CTA each 88 us; with the best 5 90,
// 129 and 151 us; with the best 20 165, 160 and 176 us), beyond that by four. Else a
// row takes a CTA, or a cluster of up to 8 where the rows alone leave SMs idle (each
// with at least one full step of its warps). Without g, rows beyond 16 KB stay with a
// CTA each: its 32 warps an SM hide more than the stream (8192 x 65536 bf16: 183 us
// against 206 us by a warp and 219 us by four).
template <typename T, int SHAPE, bool TOP>
int launch_rows_sized(const RowProbArgs& A, cudaStream_t s) {
    const int64_t bytes = A.M * (int64_t)sizeof(T), rows = A.B * A.N;
    if (A.M <= (A.top_k <= 2 ? 512 : 256) && A.top_k <= kGroupTop) {
        if (A.M <= 64) return launch_group<T, SHAPE, TOP, 8, 8>(A, s);
        if (A.M <= 128) return launch_group<T, SHAPE, TOP, 16, 8>(A, s);
        if (A.M <= 256) return launch_group<T, SHAPE, TOP, 16, 16>(A, s);
        return launch_group<T, SHAPE, TOP, 16, 32>(A, s);
    }
    if (bytes <= 2048) {
        const int64_t want = rows / (148 * 24) / kRowWarps * kRowWarps;
        const int per = (int)std::max<int64_t>(kRowWarps, std::min<int64_t>(want, 32));
        return bytes <= 512 ? launch_held<T, SHAPE, TOP, 1>(A, per, s)
                            : launch_held<T, SHAPE, TOP, 4>(A, per, s);
    }
    const bool runs = (SHAPE == kPlain || A.N >= 64) && rows < INT_MAX / 2;
    if (bytes <= 16384 && rows >= 148 * 16 && runs) return launch_stream<T, SHAPE, TOP, 1>(A, s);
    if constexpr (SHAPE != kPlain)
        if (bytes > 8192 && rows >= 148 * 4 && runs) return launch_stream<T, SHAPE, TOP, 4>(A, s);
    int cluster = 1;
    while (cluster < 8 && rows * cluster * 2 <= 148 * 4 &&
           bytes > (int64_t)cluster * kRowWarps * 32 * 4 * 16)
        cluster *= 2;
    return launch_cta<T, SHAPE, TOP>(A, cluster, s);
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
// atomics (bands are summed in a fixed order by a second kernel). One read and one
// write, bound by DRAM: 8192 x 65536 bf16 357 us, 6.0 TB/s, 92% of a copy.

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
// every factor has sign / eps in it already. l2 = inf marks a row that passes nothing:
// an empty one, or one whose upstream gradients are all zero. Such a row may hold
// anything (what mask_a leaves out, positions without a token): -inf takes its values'
// place, so that p is 0 and no factor meets a NaN.
struct RowConst {
    float m, l2, c, h, at;
    int target;

    __device__ __forceinline__ bool silent() const { return l2 == INFINITY; }
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
    const unsigned M = (unsigned)A.M, next_vec = tx * V;
    const unsigned col0 = (blockIdx.x * tx * U + cx) * V;  // before the row's lead
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
            // (32-bit columns and stepped rows: the kernel is bound by instructions)
            const T* X = Xb + (rb0 + cy) * A.sXn;
            T* D = A.dX ? Db + (rb0 + cy) * A.M : nullptr;
            const int64_t x_step = ty * A.sXn, d_step = A.dX ? ty * A.M : 0;
            uint4 raw[U];
            auto load = [&](const T* X) {
                const unsigned j = (COLS ? 0 : (unsigned)row_lead(X, A.M)) + col0;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (j + u * next_vec + V <= M) raw[u] = ld_stream16(X + j + u * next_vec);
            };
            if (VEC && cy < nr) load(X);  // on their way beside the rows' constants
            __syncthreads();  // the last rows' constants and sums are read
            for (int r = threadIdx.x; r < nr; r += kBwdThreads) {
                const int64_t row = b * A.N + rb0 + r;
                const float2 st = A.stats[row];
                RowConst q;
                q.target = -1;
                q.at = q.h = q.c = 0.f;
                q.m = st.x;
                q.l2 = st.y * kLog2e;
                bool asked = false;  // of a row that is not empty
                if (st.x != kNegInf || st.y != 0.f) {
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
                    asked = q.at != 0.f || q.c != 0.f;
                    if (A.g_ent) {
                        q.h = A.g_ent[row];
                        asked = asked || q.h != 0.f;
                        q.c -= q.h * A.entropy[row];
                    }
                    float t = q.at;
                    if (TOP)
#pragma unroll 4
                        for (int j = 0; j < A.top_k; ++j)
                            if (A.top_idx[row * A.top_k + j] >= 0) {
                                const float gt = A.g_top[row * A.top_k + j];
                                asked = asked || gt != 0.f;
                                t += gt;
                            }
                    q.c = (q.c - t) * ks;
                    q.h *= ks * kLn2;
                    q.at *= ks;
                }
                if (!asked) {
                    q.m = q.c = q.h = q.at = 0.f;
                    q.l2 = INFINITY;
                }
                rc[r] = q;
            }
            __syncthreads();
            for (int r = cy; r < nr; r += ty, X += x_step, D += d_step) {
                const RowConst q = rc[r];
                const int64_t row = b * A.N + rb0 + r;
                const unsigned lead = COLS || !VEC ? 0 : (unsigned)row_lead(X, A.M);
                const unsigned j0 = lead + col0;
                const RowShape rs = row_shape(A.g, A.sign, b, A.M, lead);
                const bool aligned = (reinterpret_cast<uintptr_t>(D + lead) & 15) == 0;
                const bool inside = j0 + (U - 1) * next_vec + V <= M;
                float2 x[U * V2];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const unsigned j = j0 + u * next_vec;
                    float2* const d = x + u * V2;
                    if constexpr (VEC) {
                        unpack2(raw[u], d, X);
                        if (inside || j + V <= M) {
                            shape_pairs<SHAPE, V2>(d, rs, j);
                        } else {  // the row's last columns, fewer than a vector
#pragma unroll
                            for (int e = 0; e < V2; ++e) {
                                const unsigned i = j + 2 * e;
                                d[e].x = i < M ? shaped<SHAPE>(widen(X[i]), rs, i) : kNegInf;
                                d[e].y = i + 1 < M ? shaped<SHAPE>(widen(X[i + 1]), rs, i + 1)
                                                   : kNegInf;
                            }
                        }
                    } else {
                        d->x = j < M ? shaped<SHAPE>(widen(X[j]), rs, j) : kNegInf;
                        d->y = j + 1 < M ? shaped<SHAPE>(widen(X[j + 1]), rs, j + 1) : kNegInf;
                    }
                }
                if (VEC && r + ty < nr) load(X + x_step);
                if (q.silent()) {
#pragma unroll
                    for (int e = 0; e < U * V2; ++e) x[e] = make_float2(kNegInf, kNegInf);
                }
                const float2 nm = make_float2(-q.m, -q.m), kk = make_float2(k2, k2);
                const float2 nl = make_float2(-q.l2, -q.l2), cc = make_float2(q.c, q.c);
                const float2 nh = make_float2(-q.h, -q.h);
                auto slope = [&](float2 v) {
                    float2 y = __ffma2_rn(__fadd2_rn(v, nm), kk, nl);
                    const float2 p = make_float2(ex2(y.x), ex2(y.y));
                    y = make_float2(fmaxf(y.x, kFarBelow), fmaxf(y.y, kFarBelow));
                    return __fmul2_rn(p, __ffma2_rn(y, nh, cc));
                };
                if (!COLS && VEC && blockIdx.x == 0 && cx < (int)lead && D) {
                    // the columns before the row's first vector, one to a thread
                    const float v =
                        q.silent() ? kNegInf : shaped<SHAPE>(widen(X[cx]), rs, cx);
                    float d = slope(make_float2(v, v)).x + (cx == q.target ? q.at : 0.f);
                    if (TOP)
                        for (int t = 0; t < A.top_k; ++t)
                            if (__ldg(A.top_idx + row * A.top_k + t) == cx)
                                d = fmaf(__ldg(A.g_top + row * A.top_k + t), ks, d);
                    D[cx] = narrow<T>(d);
                }
                if (q.h == 0.f) {  // no gradient of the entropy
#pragma unroll
                    for (int e = 0; e < U * V2; ++e) {
                        const float2 y = __ffma2_rn(__fadd2_rn(x[e], nm), kk, nl);
                        x[e] = __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), cc);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < U * V2; ++e) x[e] = slope(x[e]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const unsigned j = j0 + u * next_vec;
                    float2* const d = x + u * V2;
                    // the upstream gradients of single columns
                    if ((unsigned)q.target - j < (unsigned)V) {
                        const unsigned at = q.target - j;
#pragma unroll
                        for (int e = 0; e < V2; ++e) {
                            if (at == 2 * e) d[e].x += q.at;
                            if (at == 2 * e + 1) d[e].y += q.at;
                        }
                    }
                    if (TOP) {
                        for (int t = 0; t < A.top_k; ++t) {
                            const unsigned at =
                                (unsigned)__ldg(A.top_idx + row * A.top_k + t) - j;
                            if (at < (unsigned)V) {
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
                            whole = aligned && (inside || j + V <= M);
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

// Bands of the backward: CTAs in whole waves of 4 to an SM. Column sums take one
// wave, since each band is a row of partials (4 x 8192 x 64 fp32: 13 us, with two
// waves 19 us); without them a band is at most the rows that are held at once (8192 x
// 65536 bf16: 357 us in four waves, 370 us in 3.5).
void bwd_bands(int64_t B, int64_t N, int64_t M, bool cols, int elem, int64_t* bands,
               int64_t* band_rows) {
    constexpr int64_t wave = 148 * 4;
    const int64_t tile = (int64_t)kBwdThreads * kBwdVecs * (16 / elem);
    const int64_t tiles = std::max<int64_t>(1, (M + tile - 1) / tile) * B;
    const int64_t few = cols ? 1 : (N + kBwdRows - 1) / kBwdRows;
    const int64_t waves = std::max<int64_t>(1, (tiles * few + wave - 1) / wave);
    const int64_t want = std::max<int64_t>(few, cols && waves > 1 ? 1 : waves * wave / tiles);
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
    if (!std::isfinite((float)(1.0 / epsilon)))
        return fail(SK_ERR_ARG, "1 / epsilon is beyond fp32");
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
    if (B <= 0 || M <= sk::kStagedMax) return 0;
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
    if (mask_b && M > kStagedMax &&
        (!workspace || (uintptr_t)workspace % 16 != 0 ||
         workspace_bytes < sk_row_logprobs_workspace_bytes(B, M)))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_row_logprobs with mask_b");
    cudaStream_t s = (cudaStream_t)stream;
    RowProbArgs A{};
    A.staged = (g || mask_b) && M <= kStagedMax;
    if (A.staged) {
        A.mask_b = mask_b;
    } else {
        const int fm = fold_mask(&g, mask_b, B * M, workspace, s);
        if (fm != SK_OK) return fm;
    }
    A.X = X;
    A.N = N;
    A.M = M;
    A.sXb = sXb;
    A.sXn = sXn;
    A.B = B;
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
    return sk::align_up(sizeof(float) * (size_t)B * M) +
           sk::align_up(sizeof(float) * (size_t)B * most * M);
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
    if ((dg || mask_b) &&
        (!workspace || (uintptr_t)workspace % 16 != 0 ||
         workspace_bytes < sk_row_logprobs_backward_workspace_bytes(B, N, M)))
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
    if (dg) A.partial = (float*)((char*)workspace + align_up(sizeof(float) * (size_t)B * M));
    bwd_bands(B, N, M, dg != nullptr, dtype == SK_FP32 ? 4 : 2, &A.bands, &A.band_rows);
    const bool masked = mask_b != nullptr;
    if (dtype == SK_FP32) return launch_bwd_typed<float>(A, masked, dg, s);
    if (dtype == SK_BF16) return launch_bwd_typed<__nv_bfloat16>(A, masked, dg, s);
    return launch_bwd_typed<__half>(A, masked, dg, s);
}

}  // extern "C"
