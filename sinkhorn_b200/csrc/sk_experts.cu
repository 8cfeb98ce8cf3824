// sk_experts.cu -- rows into the order of their experts and back.
//
// A router gives each token k experts (index, (T,k)). The S = T k slots are
// put into expert order by a stable counting sort -- slot s = t k + j goes to
//     position[s] = offsets[e] + #{s' < s : index[s'] = e},  e = index[s],
// so the result does not depend on how the kernels are scheduled -- and the
// tokens' rows are copied there (dispatch) and summed back with the gates'
// weights (combine). Slots whose index is no expert are dropped; the rows
// that no slot holds, those behind offsets[E] among them, are zero.
//
// All three row kernels go by token, one warp each: the token's row is read or
// written once, its k slots are whole rows elsewhere. They are bound by DRAM: 32768
// x 2 rows of 2048 bf16 64 us (6.3 TB/s, 96% of a copy), and back with their
// gradients for 16385 x 4 rows of 1536 45 us and 78 us (5.6 and 5.8 TB/s, each called in
// a row). The sort is two launches of 6 us and 8 us for 65536 slots, one of 5 us up to
// 2048.
// The kernels are launched as programmatic dependents of one another (see
// sk_common.cuh): sort and copy of 32768 x 2 rows 83 us apart, 76 us so. What a kernel
// before may still be writing when they start is read by plain loads behind pdl_wait():
// the read-only path is for data that nothing writes while the kernel lives.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "sk_common.cuh"
#include "sk_internal.h"

namespace sk {
namespace {

constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortTile = 2048;  // slots of a CTA at once
// Every CTA of the second launch adds up the counts of all, so there are at most two
// to an SM: more slots are more tiles of a CTA's run, one after the other, and the work
// grows with the slots and not with their square (8M slots, 256 experts: 1324 us with a
// tile to each CTA, 209 us so; 65536 slots take a tile each in both).
constexpr int kSortCtas = 2 * 148;
constexpr int kMaxExperts = 1024;

__device__ __forceinline__ int expert_of(const int64_t* index, int64_t s, int64_t S, int E) {
    if (s >= S) return -1;
    const int64_t e = index[s];
    return e >= 0 && e < E ? (int)e : -1;
}

// hist[run][e]: the slots of each expert in a CTA's run of `run` slots.
__global__ void __launch_bounds__(kSortThreads) k_expert_count(const int64_t* index, int64_t S,
                                                              int64_t run, int E, int* hist) {
    __shared__ int count[kMaxExperts];
    pdl_wait();
    pdl_trigger();
    for (int e = threadIdx.x; e < E; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const int64_t end = min(S, (blockIdx.x + 1) * run);
    for (int64_t s0 = blockIdx.x * run; s0 < end; s0 += kSortTile) {
#pragma unroll
        for (int i = 0; i < kSortTile / kSortThreads; ++i) {
            const int e = expert_of(index, s0 + i * kSortThreads + threadIdx.x, S, E);
            if (e >= 0) atomicAdd(&count[e], 1);  // counts only: their order is no matter
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kSortThreads)
        hist[(int64_t)blockIdx.x * E + e] = count[e];
}

// Places of the slots of a CTA's run, tile by tile. A warp takes consecutive slots of a
// tile, 32 at a time; lanes of one expert rank themselves by match.any.
__global__ void __launch_bounds__(kSortThreads) k_expert_place(const int64_t* index, int64_t S,
                                                              int64_t run, int E,
                                                              const int* hist,
                                                              int* order, int* position,
                                                              int* offsets) {
    extern __shared__ int sm[];
    int* const start = sm;      // [E] first place of the tile's slots of an expert
    int* const wcount = sm + E;  // [warps][E]
    __shared__ int wsum[kSortWarps];
    __shared__ int carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t end = min(S, (blockIdx.x + 1) * run);
    int64_t tile = blockIdx.x * run;
    constexpr int R = kSortTile / kSortThreads;
    int e[R];
    auto slot = [&](int i) {
        return tile + warp * (kSortTile / kSortWarps) + i * 32 + lane;
    };
    // the warp's slots of each expert
    auto count = [&] {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const unsigned same = __match_any_sync(0xffffffffu, e[i]);
            if (e[i] >= 0 && lane == __ffs(same) - 1) wcount[warp * E + e[i]] += __popc(same);
            __syncwarp();
        }
    };
    // the earlier warps' counts in place of each one's; their sum
    auto sum_warps = [&](int x) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
            const int c = wcount[w * E + x];
            wcount[w * E + x] = sum;
            sum += c;
        }
        return sum;
    };
    // every slot of the tile to its place; each warp's counts are added to the earlier ones
    auto place = [&] {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const unsigned same = __match_any_sync(0xffffffffu, e[i]);
            const int64_t s = slot(i);
            int at = -1;
            if (e[i] >= 0) {
                at = start[e[i]] + wcount[warp * E + e[i]] + __popc(same & ((1u << lane) - 1u));
                if (at < S) order[at] = (int)s;
            }
            if (s < S) position[s] = at;
            __syncwarp();
            if (e[i] >= 0 && lane == __ffs(same) - 1) wcount[warp * E + e[i]] += __popc(same);
            __syncwarp();
        }
    };
    for (int i = threadIdx.x; i < kSortWarps * E; i += kSortThreads) wcount[i] = 0;
    if (threadIdx.x == 0) carry = 0;
    pdl_wait();
    pdl_trigger();
#pragma unroll
    for (int i = 0; i < R; ++i) e[i] = expert_of(index, slot(i), S, E);
    __syncthreads();
    count();
    __syncthreads();
    // Per expert: the earlier warps' counts, the earlier CTAs', and the total,
    // whose running sum over the experts gives the offsets.
    for (int base = 0; base < E; base += kSortThreads) {
        const int x = base + threadIdx.x;
        int total = 0, before = 0;
        if (x < E) {
            total = sum_warps(x);  // (a single CTA has a single tile)
            if (gridDim.x > 1) {
                total = 0;
#pragma unroll 8
                for (int t = 0; t < (int)gridDim.x; ++t) {
                    const int c = hist[(int64_t)t * E + x];
                    if (t < (int)blockIdx.x) before += c;
                    total += c;
                }
            }
        }
        int scan = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) wsum[warp] = scan;
        __syncthreads();
        int add = carry;
        for (int w = 0; w < warp; ++w) add += wsum[w];
        if (x < E) {
            start[x] = add + scan - total + before;
            if (blockIdx.x == 0) offsets[x] = add + scan - total;
        }
        __syncthreads();
        if (threadIdx.x == kSortThreads - 1) carry = add + scan;
        __syncthreads();
    }
    const int held = carry;
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = held;
    place();
    for (tile += kSortTile; tile < end; tile += kSortTile) {
#pragma unroll
        for (int i = 0; i < R; ++i) e[i] = expert_of(index, slot(i), S, E);
        __syncthreads();  // the last tile is placed: its last warp's counts are its sums
        for (int x = threadIdx.x; x < E; x += kSortThreads) {
            start[x] += wcount[(kSortWarps - 1) * E + x];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) wcount[w * E + x] = 0;
        }
        __syncthreads();
        count();
        __syncthreads();
        for (int x = threadIdx.x; x < E; x += kSortThreads) sum_warps(x);
        __syncthreads();
        place();
    }
    // places behind the last group
    for (int64_t p = held + (int64_t)blockIdx.x * kSortThreads + threadIdx.x; p < S;
         p += (int64_t)gridDim.x * kSortThreads)
        order[p] = -1;
}

// ------------------------------------------------------------------- rows

// Words of W bytes: the widest that rows, strides and widths are multiples of.
template <int W>
struct WordOf;
template <>
struct WordOf<16> {
    using type = uint4;
};
template <>
struct WordOf<8> {
    using type = uint2;
};
template <>
struct WordOf<4> {
    using type = uint32_t;
};
template <>
struct WordOf<2> {
    using type = uint16_t;
};

template <typename T, int W>
struct Elems {
    static constexpr int n = W / (int)sizeof(T);
    union {
        typename WordOf<W>::type word;
        T e[n > 0 ? n : 1];
    };
    __device__ __forceinline__ Elems() {}
    __device__ __forceinline__ float get(int i) const { return (float)e[i]; }
    __device__ __forceinline__ void set(int i, float v) { e[i] = (T)v; }
};

struct RowsArgs {
    const void *x, *y;  // rows by token (x) and by place (y)
    void *ox, *oy;
    int64_t ldx, ldy, ldox, ldoy;  // row strides in words
    int64_t T;
    int k;
    int words;
    const int* order;  // the slot at each place, or NULL: positions alone count
    const int* position;
    const int* offsets;  // its last entry: rows that are held
    int E;
    const float* w;  // (T,k) or NULL
    float* dw;       // (T,k)
};

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;  // most words of a row to a lane at once

// Places that can be held: those before the last offset.
__device__ __forceinline__ int places(const RowsArgs& A) {
    return (int)min((int64_t)max(A.offsets[A.E], 0), A.T * A.k);
}

// The slot's place p of n, -1 where it has none. A slot holds its place where the place
// names it, too: of a plan that was edited (slots dropped for an expert over its
// capacity, two slots at one place) each row has one writer then, and rows without one
// are known to the place alone (gap_at).
__device__ __forceinline__ int named_place(const RowsArgs& A, int n, int64_t slot) {
    const int p = A.position[slot];
    return (unsigned)p < (unsigned)n ? p : -1;
}
__device__ __forceinline__ bool holds(const RowsArgs& A, int64_t slot, int p) {
    return !A.order || A.order[p] == (int)slot;
}
__device__ __forceinline__ bool gap_at(const RowsArgs& A, int64_t p) {
    const int s = A.order[p];
    return s < 0 || s >= A.T * A.k || A.position[s] != (int)p;
}

template <int W>
__device__ __forceinline__ void zero_row(const RowsArgs& A, int64_t p, int lane) {
    using Word = typename WordOf<W>::type;
    Word* const o = reinterpret_cast<Word*>(A.oy) + p * A.ldoy;
    for (int c = lane; c < A.words; c += 32) o[c] = Word{};
}

// Rows that no slot writes: those behind the last group, and gaps before it (looked for
// by the last warps first, which have the least to copy).
template <int W>
__device__ __forceinline__ void zero_unheld(const RowsArgs& A, int n, int64_t gw, int64_t nw,
                                            int lane) {
    for (int64_t p = n + gw; p < A.T * A.k; p += nw) zero_row<W>(A, p, lane);
    if (!A.order) return;
    for (int64_t p0 = (nw - 1 - gw) * 32; p0 < n; p0 += nw * 32) {
        unsigned gaps = __ballot_sync(0xffffffffu, p0 + lane < n && gap_at(A, p0 + lane));
        for (; gaps; gaps &= gaps - 1) zero_row<W>(A, p0 + __ffs(gaps) - 1, lane);
    }
}

template <int W>
__global__ void __launch_bounds__(kCopyThreads) k_dispatch_rows(const RowsArgs A) {
    using Word = typename WordOf<W>::type;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t gw = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) >> 5;
    const int64_t nw = (int64_t)gridDim.x * (kCopyThreads / 32);
    const int held = places(A);
    for (int64_t t = gw; t < A.T; t += nw) {
        const Word* const x = reinterpret_cast<const Word*>(A.x) + t * A.ldx;
        for (int c = lane; c < A.words; c += 32 * kCopyUnroll) {
            Word v[kCopyUnroll];
#pragma unroll
            for (int u = 0; u < kCopyUnroll; ++u)
                if (c + u * 32 < A.words) v[u] = x[c + u * 32];
            for (int j = 0; j < A.k; ++j) {
                const int p = named_place(A, held, t * A.k + j);
                if (p < 0 || !holds(A, t * A.k + j, p)) continue;
                Word* const o = reinterpret_cast<Word*>(A.oy) + p * A.ldoy;
#pragma unroll
                for (int u = 0; u < kCopyUnroll; ++u)
                    if (c + u * 32 < A.words) o[c + u * 32] = v[u];
            }
        }
    }
    zero_unheld<W>(A, held, gw, nw, lane);
}

// ox[t] = sum_j w[t,j] y[position[t,j]], in fp32, rounded once.
template <typename T, int W, int U>
__global__ void __launch_bounds__(kCopyThreads) k_combine_rows(const RowsArgs A) {
    using Word = typename WordOf<W>::type;
    pdl_wait();
    pdl_trigger();
    constexpr int n = W / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    const int64_t gw = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) >> 5;
    const int64_t nw = (int64_t)gridDim.x * (kCopyThreads / 32);
    const int held = places(A);
    for (int64_t t = gw; t < A.T; t += nw) {
        Word* const o = reinterpret_cast<Word*>(A.ox) + t * A.ldox;
        for (int c = lane; c < A.words; c += 32 * U) {
            float sum[U][n];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < n; ++i) sum[u][i] = 0.f;
            for (int j = 0; j < A.k; ++j) {
                const int p = named_place(A, held, t * A.k + j);
                if (p < 0) continue;
                const bool own = holds(A, t * A.k + j, p);  // (on its way beside the row)
                const float w = A.w ? A.w[t * A.k + j] : 1.f;
                const Word* const y = reinterpret_cast<const Word*>(A.y) + p * A.ldy;
                Elems<T, W> v[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (c + u * 32 < A.words) v[u].word = y[c + u * 32];
                if (!own) continue;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (c + u * 32 < A.words)
#pragma unroll
                        for (int i = 0; i < n; ++i) sum[u][i] = fmaf(w, v[u].get(i), sum[u][i]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + u * 32 < A.words) {
                    Elems<T, W> v;
#pragma unroll
                    for (int i = 0; i < n; ++i) v.set(i, sum[u][i]);
                    o[c + u * 32] = v.word;
                }
        }
    }
}

// The adjoint of combine: with d = x[t] the upstream row of token t,
//     oy[position[t,j]] = w[t,j] d,   dw[t,j] = <d, y[position[t,j]]>.
// Either of oy and dw may be NULL.
template <typename T, int W, int U>
__global__ void __launch_bounds__(kCopyThreads) k_combine_rows_bwd(const RowsArgs A) {
    using Word = typename WordOf<W>::type;
    pdl_wait();
    pdl_trigger();
    constexpr int n = W / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    const int64_t gw = ((int64_t)blockIdx.x * kCopyThreads + threadIdx.x) >> 5;
    const int64_t nw = (int64_t)gridDim.x * (kCopyThreads / 32);
    const int held = places(A);
    for (int64_t t = gw; t < A.T; t += nw) {
        const Word* const x = reinterpret_cast<const Word*>(A.x) + t * A.ldx;
        for (int j = 0; j < A.k; ++j) {
            const int p = named_place(A, held, t * A.k + j);
            float dot = 0.f;
            if (p >= 0) {
                const bool own = holds(A, t * A.k + j, p);  // (on its way beside the rows)
                const float w = A.w ? A.w[t * A.k + j] : 1.f;
                const Word* const y = reinterpret_cast<const Word*>(A.y) + p * A.ldy;
                Word* const o = reinterpret_cast<Word*>(A.oy) + p * A.ldoy;
                for (int c = lane; c < A.words; c += 32 * U) {
                    Elems<T, W> d[U], v[U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u * 32 < A.words) {
                            d[u].word = x[c + u * 32];
                            if (A.dw) v[u].word = y[c + u * 32];
                        }
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u * 32 < A.words) {
                            if (A.dw)
#pragma unroll
                                for (int i = 0; i < n; ++i)
                                    dot = fmaf(d[u].get(i), v[u].get(i), dot);
                            if (A.oy && own) {
#pragma unroll
                                for (int i = 0; i < n; ++i) d[u].set(i, w * d[u].get(i));
                                o[c + u * 32] = d[u].word;
                            }
                        }
                }
                if (!own) dot = 0.f;
            }
            if (A.dw) {
                dot = warp_sum(dot);
                if (lane == 0) A.dw[t * A.k + j] = dot;
            }
        }
    }
    if (A.oy) zero_unheld<W>(A, held, gw, nw, lane);
}

unsigned rows_grid(int64_t T) {
    const int64_t ctas = (T + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ctas, 148 * 64));
}

// The widest word (2 to 16 bytes) that every address, stride and width allows.
int word_bytes(int64_t D, int elem, std::initializer_list<const void*> p,
               std::initializer_list<int64_t> ld) {
    int w = 16;
    auto fit = [&](uint64_t v) {
        while (v % w) w /= 2;
    };
    fit((uint64_t)D * elem);
    for (const void* q : p) fit((uint64_t)(uintptr_t)q);
    for (int64_t l : ld) fit((uint64_t)l * elem);
    return w;
}

int check_rows_args(int dtype, int64_t T, int k, int64_t D, int E, const int* position,
                    const int* offsets) {
    if (dtype < SK_FP32 || dtype > SK_FP16) return fail(SK_ERR_ARG, "unknown element type");
    if (T <= 0 || k <= 0 || D <= 0) return fail(SK_ERR_ARG, "T, k and D must be positive");
    if (T > INT32_MAX / k || D > INT32_MAX / 4)
        return fail(SK_ERR_ARG, "T * k must be below 2^31 and D below 2^29");
    if (E <= 0 || E > kMaxExperts) return fail(SK_ERR_ARG, "experts must lie in 1..1024");
    if (!position || !offsets) return fail(SK_ERR_ARG, "position or offsets is NULL");
    return SK_OK;
}

template <int W>
int run_dispatch(const RowsArgs& A, cudaStream_t s) {
    launch_pdl(k_dispatch_rows<W>, dim3(rows_grid(A.T)), dim3(kCopyThreads), 0, s, A);
    SK_LAUNCHED("k_dispatch_rows");
    return SK_OK;
}

template <typename T, int W, int U>
int run_combine(const RowsArgs& A, bool bwd, cudaStream_t s) {
    const dim3 grid(rows_grid(A.T)), block(kCopyThreads);
    if (bwd) launch_pdl(k_combine_rows_bwd<T, W, U>, grid, block, 0, s, A);
    else launch_pdl(k_combine_rows<T, W, U>, grid, block, 0, s, A);
    SK_LAUNCHED(bwd ? "k_combine_rows_bwd" : "k_combine_rows");
    return SK_OK;
}

// A row takes the fewest passes of up to kCopyUnroll words a lane, of equal width:
// 192 words go in two passes of 3, not of 4 and 2 (16385 x 4 rows of 1536 bf16:
// 50 us against 54 us).
template <typename T>
int run_combine_wide(const RowsArgs& A, int w, bool bwd, cudaStream_t s) {
    if (w == 16) {
        const int lane = (A.words + 31) / 32, passes = (lane + kCopyUnroll - 1) / kCopyUnroll;
        const int u = (lane + passes - 1) / passes;
        if (u == 1) return run_combine<T, 16, 1>(A, bwd, s);
        if (u == 2) return run_combine<T, 16, 2>(A, bwd, s);
        if (u == 3) return run_combine<T, 16, 3>(A, bwd, s);
        return run_combine<T, 16, 4>(A, bwd, s);
    }
    if (w == 8) return run_combine<T, 8, kCopyUnroll>(A, bwd, s);
    if constexpr (sizeof(T) == 2) {
        if (w == 4) return run_combine<T, 4, kCopyUnroll>(A, bwd, s);
        return run_combine<T, 2, kCopyUnroll>(A, bwd, s);
    }
    return run_combine<T, 4, kCopyUnroll>(A, bwd, s);
}

int run_combine_typed(RowsArgs A, int dtype, int64_t D, bool bwd, cudaStream_t s) {
    const int elem = dtype == SK_FP32 ? 4 : 2;
    const int w = word_bytes(D, elem, {A.x, A.y, A.ox, A.oy}, {A.ldx, A.ldy, A.ldox, A.ldoy});
    if (w < elem) return fail(SK_ERR_LAYOUT, "rows are not aligned to their elements");
    const int per = w / elem;
    A.words = (int)(D / per);
    A.ldx /= per;
    A.ldy /= per;
    A.ldox /= per;
    A.ldoy /= per;
    if (dtype == SK_FP32) return run_combine_wide<float>(A, w, bwd, s);
    if (dtype == SK_BF16) return run_combine_wide<__nv_bfloat16>(A, w, bwd, s);
    return run_combine_wide<__half>(A, w, bwd, s);
}

int dispatch_rows(const void* x, int dtype, int64_t T, int k, int64_t D, int64_t ldx,
                  const int* order, const int* position, const int* offsets, int experts,
                  void* rows, cudaStream_t s) {
    const int rc = check_rows_args(dtype, T, k, D, experts, position, offsets);
    if (rc != SK_OK) return rc;
    if (!x || !rows) return fail(SK_ERR_ARG, "x or rows is NULL");
    if (ldx < 0) return fail(SK_ERR_LAYOUT, "negative row stride");
    const int elem = dtype == SK_FP32 ? 4 : 2;
    const int w = word_bytes(D, elem, {x, rows}, {ldx, D});
    if (w < elem) return fail(SK_ERR_LAYOUT, "rows are not aligned to their elements");
    RowsArgs A{};
    A.x = x;
    A.oy = rows;
    A.ldx = ldx * elem / w;
    A.ldoy = D * elem / w;
    A.T = T;
    A.k = k;
    A.words = (int)(D * elem / w);
    A.order = order;
    A.position = position;
    A.offsets = offsets;
    A.E = experts;
    if (w == 16) return run_dispatch<16>(A, s);
    if (w == 8) return run_dispatch<8>(A, s);
    if (w == 4) return run_dispatch<4>(A, s);
    return run_dispatch<2>(A, s);
}

int combine_rows(const void* y, int dtype, int64_t T, int k, int64_t D, int64_t ldy,
                 const int* order, const int* position, const int* offsets, int experts,
                 const float* weights, void* out, cudaStream_t s) {
    const int rc = check_rows_args(dtype, T, k, D, experts, position, offsets);
    if (rc != SK_OK) return rc;
    if (!y || !out) return fail(SK_ERR_ARG, "y or out is NULL");
    if (ldy < 0) return fail(SK_ERR_LAYOUT, "negative row stride");
    RowsArgs A{};
    A.y = y;
    A.ox = out;
    A.ldy = ldy;
    A.ldox = D;
    A.T = T;
    A.k = k;
    A.order = order;
    A.position = position;
    A.offsets = offsets;
    A.E = experts;
    A.w = weights;
    return run_combine_typed(A, dtype, D, false, s);
}

int combine_rows_backward(const void* grad_out, const void* y, int dtype, int64_t T, int k,
                          int64_t D, int64_t ldg, int64_t ldy, const int* order,
                          const int* position, const int* offsets, int experts,
                          const float* weights, void* grad_y, float* grad_weights,
                          cudaStream_t s) {
    const int rc = check_rows_args(dtype, T, k, D, experts, position, offsets);
    if (rc != SK_OK) return rc;
    if (!grad_out) return fail(SK_ERR_ARG, "grad_out is NULL");
    if (!grad_y && !grad_weights) return fail(SK_ERR_ARG, "no gradient is asked for");
    if (grad_weights && !y) return fail(SK_ERR_ARG, "grad_weights needs y");
    if (ldg < 0 || ldy < 0) return fail(SK_ERR_LAYOUT, "negative row stride");
    RowsArgs A{};
    A.x = grad_out;
    A.y = y;
    A.oy = grad_y;
    A.ldx = ldg;
    A.ldy = ldy;
    A.ldoy = D;
    A.T = T;
    A.k = k;
    A.order = order;
    A.position = position;
    A.offsets = offsets;
    A.E = experts;
    A.w = weights;
    A.dw = grad_weights;
    return run_combine_typed(A, dtype, D, true, s);
}

// Slots of a CTA's run: whole tiles, one where there are few.
int64_t sort_run(int64_t S) {
    const int64_t tiles = (S + kSortTile - 1) / kSortTile;
    return (tiles + kSortCtas - 1) / kSortCtas * kSortTile;
}
int sort_ctas(int64_t S) {
    const int64_t run = sort_run(S);
    return (int)((S + run - 1) / run);
}

}  // namespace
}  // namespace sk

extern "C" {

size_t sk_expert_dispatch_workspace_bytes(int64_t slots, int experts) {
    if (slots <= sk::kSortTile || experts <= 0) return 0;  // one CTA counts for itself
    return sk::align_up(sizeof(int) * (size_t)sk::sort_ctas(slots) * experts);
}

int sk_expert_dispatch(const int64_t* index, int64_t slots, int experts, int* order,
                       int* position, int* offsets, void* workspace, size_t workspace_bytes,
                       void* stream) {
    using namespace sk;
    clear_error();
    if (!index || !order || !position || !offsets)
        return fail(SK_ERR_ARG, "index, order, position or offsets is NULL");
    if (slots <= 0 || slots > INT32_MAX) return fail(SK_ERR_ARG, "slots must lie in 1..2^31-1");
    if (experts <= 0 || experts > kMaxExperts)
        return fail(SK_ERR_ARG, "experts must lie in 1..1024");
    const size_t need = sk_expert_dispatch_workspace_bytes(slots, experts);
    if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 4 != 0))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_expert_dispatch");
    cudaStream_t s = (cudaStream_t)stream;
    const int ctas = sort_ctas(slots);
    const int64_t run = sort_run(slots);
    if (ctas > 1) {
        launch_pdl(k_expert_count, dim3(ctas), dim3(kSortThreads), 0, s, index, slots, run,
                   experts, (int*)workspace);
        SK_LAUNCHED("k_expert_count");
    }
    const size_t smem = sizeof(int) * (size_t)experts * (1 + kSortWarps);
    launch_pdl(k_expert_place, dim3(ctas), dim3(kSortThreads), smem, s, index, slots, run,
               experts, (const int*)workspace, order, position, offsets);
    SK_LAUNCHED("k_expert_place");
    return SK_OK;
}

int sk_dispatch_rows(const void* x, int dtype, int64_t T, int k, int64_t D, int64_t ldx,
                     const int* position, const int* offsets, int experts, void* rows,
                     void* stream) {
    sk::clear_error();
    return sk::dispatch_rows(x, dtype, T, k, D, ldx, nullptr, position, offsets, experts, rows,
                             (cudaStream_t)stream);
}

int sk_dispatch_plan_rows(const void* x, int dtype, int64_t T, int k, int64_t D, int64_t ldx,
                          const int* order, const int* position, const int* offsets,
                          int experts, void* rows, void* stream) {
    sk::clear_error();
    if (!order) return sk::fail(SK_ERR_ARG, "order is NULL");
    return sk::dispatch_rows(x, dtype, T, k, D, ldx, order, position, offsets, experts, rows,
                             (cudaStream_t)stream);
}

int sk_combine_rows(const void* y, int dtype, int64_t T, int k, int64_t D, int64_t ldy,
                    const int* position, const int* offsets, int experts, const float* weights,
                    void* out, void* stream) {
    sk::clear_error();
    return sk::combine_rows(y, dtype, T, k, D, ldy, nullptr, position, offsets, experts, weights,
                            out, (cudaStream_t)stream);
}

int sk_combine_plan_rows(const void* y, int dtype, int64_t T, int k, int64_t D, int64_t ldy,
                         const int* order, const int* position, const int* offsets, int experts,
                         const float* weights, void* out, void* stream) {
    sk::clear_error();
    if (!order) return sk::fail(SK_ERR_ARG, "order is NULL");
    return sk::combine_rows(y, dtype, T, k, D, ldy, order, position, offsets, experts, weights,
                            out, (cudaStream_t)stream);
}

int sk_combine_rows_backward(const void* grad_out, const void* y, int dtype, int64_t T, int k,
                             int64_t D, int64_t ldg, int64_t ldy, const int* position,
                             const int* offsets, int experts, const float* weights, void* grad_y,
                             float* grad_weights, void* stream) {
    sk::clear_error();
    return sk::combine_rows_backward(grad_out, y, dtype, T, k, D, ldg, ldy, nullptr, position,
                                     offsets, experts, weights, grad_y, grad_weights,
                                     (cudaStream_t)stream);
}

int sk_combine_plan_rows_backward(const void* grad_out, const void* y, int dtype, int64_t T,
                                  int k, int64_t D, int64_t ldg, int64_t ldy, const int* order,
                                  const int* position, const int* offsets, int experts,
                                  const float* weights, void* grad_y, float* grad_weights,
                                  void* stream) {
    sk::clear_error();
    if (!order) return sk::fail(SK_ERR_ARG, "order is NULL");
    return sk::combine_rows_backward(grad_out, y, dtype, T, k, D, ldg, ldy, order, position,
                                     offsets, experts, weights, grad_y, grad_weights,
                                     (cudaStream_t)stream);
}

}  // extern "C"
