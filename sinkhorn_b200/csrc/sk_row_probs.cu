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
// The best k are kept by each warp as a sorted list, one entry per lane
// (k <= 32), ordered by (x descending, column ascending). A chunk of 32 x 32
// values only looks at the list when its maximum passes the k-th entry, which
// happens O(k log(M / k)) times a row in any order but an ascending one.
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
    const float* g;         // (B,M) or NULL
    const uint8_t* mask_a;  // (B,N) or NULL
    const uint8_t* mask_b;  // (B,M) or NULL
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

__device__ __forceinline__ void unpack(const uint4& v, float (&x)[4], const float*) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8], const __nv_bfloat16*) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8], const __half*) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// The row's view of the column potential and mask.
struct RowBias {
    const float* g;       // this item's g, or NULL
    const uint8_t* mask;  // this item's column mask, or NULL
    float sign;
    bool g16, mask_vec;   // vector loads of g / mask are aligned at the row's vectors
};

template <bool BIAS>
__device__ __forceinline__ float shaped(float v, const RowBias& rb, int64_t j) {
    if (BIAS) {
        v *= rb.sign;
        if (rb.g) v = __ldg(rb.g + j) + v;
        if (rb.mask && !__ldg(rb.mask + j)) v = kNegInf;
    }
    return v;
}

template <bool BIAS, int V>
__device__ __forceinline__ void shape_vec(float (&x)[V], const RowBias& rb, int64_t j) {
    if (!BIAS) return;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] *= rb.sign;
    if (rb.g) {
        if (rb.g16) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const float4 v = ld_vec4(rb.g + j + e);
                x[e] = v.x + x[e];
                x[e + 1] = v.y + x[e + 1];
                x[e + 2] = v.z + x[e + 2];
                x[e + 3] = v.w + x[e + 3];
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = __ldg(rb.g + j + e) + x[e];
        }
    }
    if (rb.mask) {
        if (rb.mask_vec) {
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const uchar4 v = __ldg(reinterpret_cast<const uchar4*>(rb.mask + j + e));
                if (!v.x) x[e] = kNegInf;
                if (!v.y) x[e + 1] = kNegInf;
                if (!v.z) x[e + 2] = kNegInf;
                if (!v.w) x[e + 3] = kNegInf;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (!__ldg(rb.mask + j + e)) x[e] = kNegInf;
        }
    }
}

__device__ __forceinline__ RowBias row_bias(const float* g, const uint8_t* mask, float sign,
                                            int64_t b, int64_t M, int64_t lead) {
    RowBias rb;
    rb.g = g ? g + b * M : nullptr;
    rb.mask = mask ? mask + b * M : nullptr;
    rb.sign = sign;
    rb.g16 = (reinterpret_cast<uintptr_t>(rb.g + lead) & 15) == 0;
    rb.mask_vec = (reinterpret_cast<uintptr_t>(rb.mask + lead) & 3) == 0;
    return rb;
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
    template <int V>
    __device__ __forceinline__ void fold(const float (&x)[V], float cm, float k2) {
        const float mn = fmaxf(m, cm);
        if (mn == kNegInf) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (isnan(x[e])) s = x[e];
            return;
        }
        if (mn != m) move_to(mn, k2);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float y = (x[e] - mn) * k2;
            const float t = ex2(y);
            s += t;
            u = fmaf(t, fmaxf(y, kFarBelow), u);
        }
    }
};

// A warp's best entries, sorted over the lanes by (value desc, column asc),
// and the k-th of them.
struct TopList {
    float v = kNegInf, kv = kNegInf;
    int i = INT_MAX, ki = INT_MAX;

    __device__ __forceinline__ void insert(float cv, int ci, int k, int lane) {
        const bool ahead = v > cv || (v == cv && i < ci);
        const int at = __popc(__ballot_sync(0xffffffffu, ahead));
        const float uv = __shfl_up_sync(0xffffffffu, v, 1);
        const int ui = __shfl_up_sync(0xffffffffu, i, 1);
        if (lane == at) {
            v = cv;
            i = ci;
        } else if (lane > at) {
            v = uv;
            i = ui;
        }
        kv = __shfl_sync(0xffffffffu, v, k - 1);
        ki = __shfl_sync(0xffffffffu, i, k - 1);
    }
    // One candidate per lane; -inf, NaN and what lies below `floor` or behind
    // the k-th entry are passed over.
    __device__ __forceinline__ void offer(float cv, int ci, int k, float floor, int lane) {
        bool in = cv >= floor && cv > kNegInf;
        unsigned todo;
        while ((todo = __ballot_sync(0xffffffffu,
                                     in && (cv > kv || (cv == kv && ci < ki)))) != 0) {
            const int src = __ffs(todo) - 1;
            insert(__shfl_sync(0xffffffffu, cv, src), __shfl_sync(0xffffffffu, ci, src), k,
                   lane);
            if (lane == src) in = false;
        }
    }
};

// Floats as unsigned integers of the same order (atomicMax).
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <int WARPS>
struct RowProbShared {
    float m[WARPS], s[WARPS], u[WARPS];
    float tv[WARPS][32];
    int ti[WARPS][32];
    unsigned thr;  // a k-th best value that some warp of the row has reached
};

// WARPS == 1: a warp per row, 8 rows per CTA, no cluster. WARPS == 8: a CTA or
// a cluster of CTAs per row, joined over distributed shared memory by rank 0.
// U vectors of 16 bytes per lane and step.
template <typename T, bool BIAS, bool TOP, int WARPS, int U>
__global__ void __launch_bounds__(256) k_row_probs(const RowProbArgs A) {
    constexpr int V = Vec<T>::n;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ RowProbShared<WARPS> sh;
    int64_t row;
    int part = 0, parts = 1;
    if (WARPS == 1) {
        row = (int64_t)blockIdx.x * 8 + warp;
        if (row >= A.rows) return;
    } else {
        parts = cg::this_cluster().num_blocks();
        part = cg::this_cluster().block_rank();
        row = blockIdx.x / parts;
        if (TOP) {
            if (threadIdx.x == 0) sh.thr = 0u;
            __syncthreads();
        }
    }
    const int64_t b = row / A.N, n = row - b * A.N;
    const T* const X = reinterpret_cast<const T*>(A.X) + b * A.sXb + n * A.sXn;
    const int64_t lead = row_lead(X, A.M);
    const RowBias rb = row_bias(A.g, A.mask_b, A.sign, b, A.M, lead);
    const float k2 = A.k * kLog2e;
    const bool empty = A.mask_a && !A.mask_a[row];
    const int64_t nv = (A.M - lead) / V;

    Moments mo;
    TopList top;
    float thr = kNegInf;
    const int wid = WARPS == 1 ? 0 : part * WARPS + warp;
    const int64_t step = (int64_t)(WARPS == 1 ? 1 : parts * WARPS) * 32 * U;

    auto one = [&](int64_t j, bool on) {  // a single column per lane (row ends)
        float x[1] = {kNegInf};
        if (on) x[0] = shaped<BIAS>(widen(X[j]), rb, j);
        mo.fold(x, x[0], k2);
        if (TOP) top.offer(x[0], (int)j, A.top_k, kNegInf, lane);
    };

    if (!empty) {
        if (wid == 0 && lead > 0) one(lane, lane < lead);
        for (int64_t base = (int64_t)wid * 32 * U; base < nv; base += step) {
            float x[U][V];
            uint4 raw[U];
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int64_t i = base + q * 32 + lane;
                if (i < nv) raw[q] = ld_stream16(X + lead + i * V);
            }
            float cm = kNegInf;
#pragma unroll
            for (int q = 0; q < U; ++q) {
                const int64_t i = base + q * 32 + lane;
                if (i < nv) {
                    unpack(raw[q], x[q], X);
                    shape_vec<BIAS, V>(x[q], rb, lead + i * V);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) x[q][e] = kNegInf;
                }
#pragma unroll
                for (int e = 0; e < V; ++e) cm = fmaxf(cm, x[q][e]);
            }
            mo.fold(reinterpret_cast<const float(&)[U * V]>(x), cm, k2);
            if (TOP) {
                if (base == (int64_t)wid * 32 * U && base + step < nv) {
                    // first of several steps: k lanes hold a value at or above the
                    // k-th best of the lane maxima, so nothing below it counts
                    int rank = 0;
#pragma unroll
                    for (int l = 0; l < 32; ++l) {
                        const float o = __shfl_sync(0xffffffffu, cm, l);
                        rank += o > cm || (o == cm && l < lane);
                    }
                    const unsigned at = __ballot_sync(0xffffffffu, rank == A.top_k - 1);
                    // (a NaN maximum beats nothing and is beaten by nothing: no lane
                    // may have that rank)
                    if (at) thr = fmaxf(thr, __shfl_sync(0xffffffffu, cm, __ffs(at) - 1));
                }
                if (WARPS > 1)
                    thr = fmaxf(thr, unordered(*reinterpret_cast<volatile unsigned*>(&sh.thr)));
                // the list's entries are of earlier steps and lower columns: only a
                // larger value gets past the k-th
                if (__any_sync(0xffffffffu, cm >= thr && cm > top.kv)) {
#pragma unroll
                    for (int q = 0; q < U; ++q)
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            top.offer(x[q][e],
                                      (int)(lead + (base + q * 32 + lane) * V + e), A.top_k,
                                      thr, lane);
                    if (WARPS > 1) {
                        if (lane == 0 && top.kv > kNegInf) atomicMax(&sh.thr, ordered(top.kv));
                    }
                }
            }
        }
        const int64_t tail = lead + nv * V;
        if (wid == 0 && tail < A.M) one(tail + lane, tail + lane < A.M);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, mo.m, o);
        const float s2 = __shfl_xor_sync(0xffffffffu, mo.s, o);
        const float u2 = __shfl_xor_sync(0xffffffffu, mo.u, o);
        mo.merge(m2, s2, u2, k2);
    }
    if (WARPS > 1) {
        if (lane == 0) {
            sh.m[warp] = mo.m;
            sh.s[warp] = mo.s;
            sh.u[warp] = mo.u;
        }
        if (TOP) {
            sh.tv[warp][lane] = top.v;
            sh.ti[warp][lane] = top.i;
        }
        cg::cluster_group cluster = cg::this_cluster();
        if (parts > 1) cluster.sync();
        else __syncthreads();
        if (part == 0 && warp == 0) {
            mo = Moments();
            for (int r = 0; r < parts; ++r) {
                const RowProbShared<WARPS>* o = parts > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) mo.merge(o->m[w], o->s[w], o->u[w], k2);
                if (TOP) {
                    for (int w = r == 0 ? 1 : 0; w < WARPS; ++w) {
                        const bool in = lane < A.top_k;
                        top.offer(in ? o->tv[w][lane] : kNegInf, in ? o->ti[w][lane] : INT_MAX,
                                  A.top_k, kNegInf, lane);
                    }
                }
            }
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
                const float x = none ? kNegInf : shaped<BIAS>(widen(X[t]), rb, t);
                lp = none ? kNegInf : fmaf(x - mo.m, A.k, -logs);
            }
            A.logprob[row] = lp;
        }
    }
    if (TOP && lane < A.top_k) {
        const bool held = top.v > kNegInf;
        A.top_lp[row * A.top_k + lane] = held ? fmaf(top.v - mo.m, A.k, -logs) : kNegInf;
        A.top_idx[row * A.top_k + lane] = held ? top.i : -1;
    }
}

template <typename T, bool BIAS, bool TOP, int WARPS, int U>
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
    SK_CUDA(cudaLaunchKernelEx(&cfg, k_row_probs<T, BIAS, TOP, WARPS, U>, A));
    return SK_OK;
}

// How a row is split. A warp per row needs no join, and serves short rows and
// row counts that fill the SMs with warps; longer or fewer rows take a CTA, and
// where the rows alone leave SMs idle a cluster of up to 8 CTAs (each with at
// least one full step of its 8 warps).
template <typename T, bool BIAS, bool TOP>
int launch_rows_sized(const RowProbArgs& A, cudaStream_t s) {
    const int64_t bytes = A.M * (int64_t)sizeof(T);
    if (bytes <= 512) return launch_rows<T, BIAS, TOP, 1, 1>(A, 1, s);
    if (bytes <= 2048 || (bytes <= 16384 && A.rows >= 148 * 16))
        return launch_rows<T, BIAS, TOP, 1, 4>(A, 1, s);
    int cluster = 1;
    while (cluster < 8 && A.rows * cluster * 2 <= 148 * 4 &&
           bytes > (int64_t)cluster * 8 * 32 * 4 * 16)
        cluster *= 2;
    return launch_rows<T, BIAS, TOP, 8, 4>(A, cluster, s);
}

template <typename T>
int launch_rows_typed(const RowProbArgs& A, cudaStream_t s) {
    const bool bias = A.g || A.mask_b || A.sign != 1.f;
    if (A.top_k > 0)
        return bias ? launch_rows_sized<T, true, true>(A, s)
                    : launch_rows_sized<T, false, true>(A, s);
    return bias ? launch_rows_sized<T, true, false>(A, s)
                : launch_rows_sized<T, false, false>(A, s);
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
    const float* g;
    const uint8_t* mask_b;
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

__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 bytes of elements, each rounded once from fp32.
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2(x[0], x[1], p), pack2(x[2], x[3], p), pack2(x[4], x[5], p),
                   pack2(x[6], x[7], p));
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

struct RowConst {
    float m, logs, c0, h, a;
    int target;
};

// COLS: the column sums are wanted; a thread then keeps its columns over all
// rows (vectors only where every row is aligned, VEC). Otherwise vectors start
// at each row's own 16-byte boundary.
template <typename T, bool BIAS, bool TOP, bool COLS, bool VEC>
__global__ void __launch_bounds__(kBwdThreads) k_row_probs_bwd(const RowProbBwdArgs A, int tx) {
    constexpr int V = VEC ? Vec<T>::n : 1;
    __shared__ RowConst rc[kBwdRows];
    __shared__ float red[COLS ? kBwdThreads * V : 1];
    const int ty = kBwdThreads / tx;
    const int cx = threadIdx.x % tx, cy = threadIdx.x / tx;
    const int64_t col = ((int64_t)blockIdx.x * tx + cx) * V;  // before the row's lead
    const float l2e = kLog2e;
    for (int64_t band = blockIdx.y; band < A.B * A.bands; band += gridDim.y) {
    const int64_t b = band / A.bands;
    const int64_t r0 = (band - b * A.bands) * A.band_rows;
    const int64_t r1 = min(A.N, r0 + A.band_rows);
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;

    for (int64_t rb0 = r0; rb0 < r1; rb0 += kBwdRows) {
        const int nr = (int)min((int64_t)kBwdRows, r1 - rb0);
        __syncthreads();
        for (int r = threadIdx.x; r < nr; r += kBwdThreads) {  // (also: red is read)
            const int64_t row = b * A.N + rb0 + r;
            const float2 st = A.stats[row];
            RowConst q;
            q.target = -1;
            q.a = q.h = q.c0 = 0.f;
            q.m = st.x;
            q.logs = st.y;
            if (st.x == kNegInf && st.y == 0.f) {
                q.m = 0.f;  // an empty row: log p = -inf everywhere
                q.logs = INFINITY;
            } else {
                if (A.g_lp) {
                    const int64_t t = A.targets[row];
                    bool given = t >= 0 && t < A.M;
                    if (given) {
                        // a column without probability passes nothing
                        RowBias tb;
                        tb.g = A.g ? A.g + b * A.M : nullptr;
                        tb.mask = A.mask_b ? A.mask_b + b * A.M : nullptr;
                        tb.sign = A.sign;
                        const T* X = reinterpret_cast<const T*>(A.X) + b * A.sXb +
                                     (rb0 + r) * A.sXn;
                        given = shaped<BIAS>(widen(X[t]), tb, t) != kNegInf;
                    }
                    if (given) {
                        q.a = A.g_lp[row];
                        q.target = (int)t;
                    }
                }
                if (A.g_lse) q.c0 = A.g_lse[row];
                if (A.g_ent) {
                    q.h = A.g_ent[row];
                    q.c0 -= q.h * A.entropy[row];
                }
                float t = q.a;
                if (TOP)
                    for (int j = 0; j < A.top_k; ++j)
                        if (A.top_idx[row * A.top_k + j] >= 0) t += A.g_top[row * A.top_k + j];
                q.c0 -= t;
            }
            rc[r] = q;
        }
        __syncthreads();
        for (int r = cy; r < nr; r += ty) {
            const RowConst q = rc[r];
            const int64_t n = rb0 + r, row = b * A.N + n;
            const T* const X = reinterpret_cast<const T*>(A.X) + b * A.sXb + n * A.sXn;
            T* const D = A.dX ? reinterpret_cast<T*>(A.dX) + row * A.M : nullptr;
            const int64_t lead = COLS || !VEC ? 0 : row_lead(X, A.M);
            const RowBias rb = row_bias(A.g, A.mask_b, A.sign, b, A.M, lead);

            auto grad = [&](float x, int64_t j) {
                const float lp = fmaf(x - q.m, A.k, -q.logs);
                const float p = ex2(lp * l2e);
                float d = p * fmaf(-q.h, fmaxf(lp, kFarBelow), q.c0);
                if (j == q.target) d += q.a;
                return d;
            };
            auto single = [&](int64_t j) {
                float d = grad(shaped<BIAS>(widen(X[j]), rb, j), j);
                if (TOP)
                    for (int t = 0; t < A.top_k; ++t)
                        if (__ldg(A.top_idx + row * A.top_k + t) == j)
                            d += __ldg(A.g_top + row * A.top_k + t);
                return d * A.k;
            };
            const int64_t j0 = lead + col;
            if (!COLS && VEC && blockIdx.x == 0 && cx == 0)
                for (int64_t j = 0; j < lead; ++j)
                    if (D) D[j] = narrow<T>(A.sign * single(j));
            if (j0 + V <= A.M) {
                float x[V], d[V];
                if constexpr (VEC) {
                    unpack(ld_stream16(X + j0), x, X);
                    shape_vec<BIAS, V>(x, rb, j0);
                } else {
                    x[0] = shaped<BIAS>(widen(X[j0]), rb, j0);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = grad(x[e], j0 + e);
                if (TOP)
                    for (int t = 0; t < A.top_k; ++t) {
                        const int64_t at = __ldg(A.top_idx + row * A.top_k + t) - j0;
                        if (at >= 0 && at < V) {
                            const float gt = __ldg(A.g_top + row * A.top_k + t);
#pragma unroll
                            for (int e = 0; e < V; ++e)
                                if (e == at) d[e] += gt;
                        }
                    }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    d[e] *= A.k;
                    if (COLS) acc[e] += d[e];
                    d[e] *= A.sign;
                }
                if (D) {
                    bool whole = false;
                    if constexpr (VEC) {
                        whole = (reinterpret_cast<uintptr_t>(D + j0) & 15) == 0;
                        if (whole) store_vec<T>(D + j0, d);
                    }
                    if (!whole)
#pragma unroll
                        for (int e = 0; e < V; ++e) D[j0 + e] = narrow<T>(d[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (j0 + e >= A.M) break;
                    const float d = single(j0 + e);
                    if (COLS) acc[e] += d;
                    if (D) D[j0 + e] = narrow<T>(A.sign * d);
                }
            }
        }
    }
    if (COLS) {
#pragma unroll
        for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = acc[e];
        __syncthreads();
        if (cy == 0) {
            for (int y = 1; y < ty; ++y)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] += red[(y * tx + cx) * V + e];
            float* out = A.partial + band * A.M;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col + e < A.M) out[col + e] = acc[e];
        }
    }
    }
}

// dg[b][j] = sum over the bands, in order.
__global__ void __launch_bounds__(256) k_band_sum(const float* partial, float* dg, int64_t BM,
                                                  int64_t M, int64_t bands) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= BM) return;
    const int64_t b = i / M, j = i - b * M;
    const float* p = partial + b * bands * M + j;
    float t = 0.f;
    for (int64_t q = 0; q < bands; ++q) t += p[q * M];
    dg[i] = t;
}

// Bands of the backward: enough CTAs for four to an SM, whole groups of rows.
void bwd_bands(int64_t B, int64_t N, int64_t M, bool cols, int elem, int64_t* bands,
               int64_t* band_rows) {
    const int64_t tile = (int64_t)kBwdThreads * (16 / elem);
    const int64_t tiles = std::max<int64_t>(1, (M + tile - 1) / tile) * B;
    int64_t want = std::max<int64_t>(1, 148 * 8 / std::max<int64_t>(1, tiles));
    // without column sums bands are free; with them each costs a row of partials
    if (!cols) want = std::max<int64_t>(want, (N + kBwdRows - 1) / kBwdRows);
    int64_t br = (N + want - 1) / want;
    br = std::max<int64_t>(br, 1);
    *bands = (N + br - 1) / br;
    *band_rows = br;
}

template <typename T, bool BIAS, bool TOP>
int launch_bwd(RowProbBwdArgs A, float* dg, cudaStream_t s) {
    const bool cols = dg != nullptr;
    // every row's vectors start where the first's do
    const bool rows_aligned = (uintptr_t)A.X % 16 == 0 && (A.sXn * sizeof(T)) % 16 == 0 &&
                              (A.B == 1 || (A.sXb * sizeof(T)) % 16 == 0);
    const bool vec = !cols || rows_aligned;
    const int V = vec ? Vec<T>::n : 1;
    int64_t cv = (A.M + V - 1) / V;
    int tx = 32;
    while (tx > 1 && tx / 2 >= cv) tx /= 2;
    while (tx < kBwdThreads && tx < cv) tx *= 2;
    const int64_t gx = (cv + tx - 1) / tx;
    const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>(A.bands * A.B, 65535));
    if (cols && vec) k_row_probs_bwd<T, BIAS, TOP, true, true><<<grid, kBwdThreads, 0, s>>>(A, tx);
    else if (cols) k_row_probs_bwd<T, BIAS, TOP, true, false><<<grid, kBwdThreads, 0, s>>>(A, tx);
    else k_row_probs_bwd<T, BIAS, TOP, false, true><<<grid, kBwdThreads, 0, s>>>(A, tx);
    SK_LAUNCHED("k_row_probs_bwd");
    if (cols) {
        const int64_t BM = A.B * A.M;
        k_band_sum<<<(unsigned)((BM + 255) / 256), 256, 0, s>>>(A.partial, dg, BM, A.M, A.bands);
        SK_LAUNCHED("k_band_sum");
    }
    return SK_OK;
}

template <typename T>
int launch_bwd_typed(const RowProbBwdArgs& A, float* dg, cudaStream_t s) {
    const bool bias = A.g || A.mask_b || A.sign != 1.f;
    const bool top = A.g_top != nullptr;
    if (top)
        return bias ? launch_bwd<T, true, true>(A, dg, s) : launch_bwd<T, false, true>(A, dg, s);
    return bias ? launch_bwd<T, true, false>(A, dg, s) : launch_bwd<T, false, false>(A, dg, s);
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

int sk_row_logprobs(const void* X, int dtype, int64_t B, int64_t N, int64_t M, int64_t sXb,
                    int64_t sXn, int64_t sXm, const float* g, double epsilon, int negate,
                    const uint8_t* mask_a, const uint8_t* mask_b, const int64_t* targets,
                    int top_k, float* lse, float* logprob, float* entropy, float* top_logprob,
                    int64_t* top_index, float* stats, void* stream) {
    using namespace sk;
    clear_error();
    const int rc = check_rows(X, dtype, B, N, M, sXb, sXn, sXm, epsilon, top_k);
    if (rc != SK_OK) return rc;
    if ((targets == nullptr) != (logprob == nullptr))
        return fail(SK_ERR_ARG, "targets and logprob go together");
    if (top_k > 0 && (!top_logprob || !top_index))
        return fail(SK_ERR_ARG, "top_k needs top_logprob and top_index");
    RowProbArgs A{};
    A.X = X;
    A.N = N;
    A.M = M;
    A.sXb = sXb;
    A.sXn = sXn;
    A.rows = B * N;
    A.g = g;
    A.mask_a = mask_a;
    A.mask_b = mask_b;
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
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == SK_FP32) return launch_rows_typed<float>(A, s);
    if (dtype == SK_BF16) return launch_rows_typed<__nv_bfloat16>(A, s);
    return launch_rows_typed<__half>(A, s);
}

size_t sk_row_logprobs_backward_workspace_bytes(int64_t B, int64_t N, int64_t M) {
    if (B <= 0 || N <= 0 || M <= 0) return 0;
    int64_t nb = 0, br = 0, most = 1;
    for (int elem = 2; elem <= 4; elem += 2) {
        sk::bwd_bands(B, N, M, true, elem, &nb, &br);
        most = std::max(most, nb);
    }
    return sk::align_up(sizeof(float) * (size_t)B * most * M);
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
    if (dg && (!workspace ||
               workspace_bytes < sk_row_logprobs_backward_workspace_bytes(B, N, M)))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_row_logprobs_backward");
    RowProbBwdArgs A{};
    A.X = X;
    A.N = N;
    A.M = M;
    A.sXb = sXb;
    A.sXn = sXn;
    A.B = B;
    A.g = g;
    A.mask_b = mask_b;
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
    A.partial = (float*)workspace;
    bwd_bands(B, N, M, dg != nullptr, dtype == SK_FP32 ? 4 : 2, &A.bands, &A.band_rows);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == SK_FP32) return launch_bwd_typed<float>(A, dg, s);
    if (dtype == SK_BF16) return launch_bwd_typed<__nv_bfloat16>(A, dg, s);
    return launch_bwd_typed<__half>(A, dg, s);
}

}  // extern "C"
