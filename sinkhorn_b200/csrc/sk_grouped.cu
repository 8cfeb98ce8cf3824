// sk_grouped.cu -- matrix products grouped by expert over ragged runs of rows.
//
// With group e's rows r in [offsets[e], offsets[e+1]):
//     y[r]  = x[r] W_e                    (rows: the runs are an output dimension)
//     dW_e  = sum_{r in e} x[r]^T dy[r]   (weights: the runs are the contraction)
// and dx[r] = dy[r] W_e^T is the first with W's two axes exchanged.
//
// One tensor-core kernel does both. A tile of the output is computed as
//     D[m, c] = sum_k A[m, k] B[c, k],   out[c * ldo + m] = D[m, c],
// with m the output's contiguous dimension on the 128 lanes of tensor memory and
// c, of any multiple of 32 up to 256, on its columns. For `rows` c is the ragged
// dimension: the instruction's N is chosen per tile, so a group of r rows costs
// ceil(r / 32) * 32 columns and not whole tiles, and the weights are the operand
// that is always full.
//
// Two CTAs work on a tile of 256 lanes (cta_group::2): each brings its own 128
// lanes of A and half of the columns of B. Alone, a CTA would read 12 KB of
// shared memory for each 128 x 256 x 16 product and write as much, 192 cycles
// at 128 bytes for 128 cycles of products; the pair needs 8 KB and 8 KB.
//
// Measured on a B200 (a library's product of one matrix 1650 TFLOP/s in a burst,
// 1390 when it lasts): 8192 x 8192 x 2048 177 us, 1545 TFLOP/s; 16 groups of 1024 x
// 2048 x 4096 190 us, 1445; lasting, 1300. With 3 rows a group the weights are the
// bound: 64 x 2048 x 1024 48 us, 5.5 TB/s. A single thread's instructions between two
// stages bound it twice on the way there (1190, then 1390 TFLOP/s).
//
// For `weights` the last block of a run's contraction holds
// rows of the next group; they are cleared in shared memory before they are used
// (a zero in one operand alone would not do: 0 * inf).
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "sk_cluster.cuh"
#include "sk_common.cuh"
#include "sk_internal.h"
#include "sk_tcgen05.cuh"

namespace sk {
namespace {

constexpr int kBM = 128;     // lanes of a CTA: the output's contiguous dimension
constexpr int kPairM = 256;  // of the two
constexpr int kBK = 64;      // contraction of a stage: one 128-byte swizzled row
constexpr int kABytes = kBM * kBK * 2;
constexpr int kBox = 64 * kBK * 2;  // bytes of 64 x 64 elements
constexpr int kBandC = 8;    // column tiles that share a pass over the weights
constexpr int kThreads = 192;  // producer warp, MMA warp, four epilogue warps
constexpr int kMaxGroups = 1024;

constexpr int kBN = 256;     // most columns of a tile
constexpr int kHalf = kBN / 2;  // columns of B in each CTA
constexpr int kStageBytes = kABytes + kHalf * kBK * 2;
constexpr int kStages = 6;
constexpr uint32_t kTmemCols = 2 * kBN;  // two accumulators

struct GroupedArgs {
    CUtensorMap a, b, b32;  // b32: boxes of 32 columns, for narrow tiles
    void* out;
    int64_t ldo, out_group;  // elements from column to column, group to group
    const int* offsets;
    int E, S;   // groups, rows
    int m, c, k;  // extents; c (rows) or k (weights) is the ragged one and unused
    bool by_rows, a_mn, b_mn, bf16;
};

struct alignas(16) GroupedShared {
    // full (the leading CTA's): the copies of both CTAs of a stage have landed.
    // empty, acc_full: committed by the MMAs to both. A stage whose last rows are
    // cleared takes another way: the second CTA's copies complete on its own
    // `part`, and it signals the leading CTA's `ready` once they are cleared.
    uint64_t full[kStages], empty[kStages], part[kStages], ready[kStages];
    uint64_t acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int gave_up;  // a bounded wait ran out: the CTA's remaining tiles become NaN
    int tiles;
    // groups 0..E+1: the rows before the first group, the groups, the rows
    // behind the last; rows in no group are zero
    int first[kMaxGroups + 3];  // first row of each
    int tile0[kMaxGroups + 3];  // first tile of each (by_rows)
    alignas(16) uint8_t turn[4][2048];  // the epilogue warps' 32 x 32 elements
};

struct Tile {
    int group;      // 0..E-1, or -1: rows of no group
    int m0, c0;     // first lane / column of the output
    int cols;       // columns of the output
    int k0, depth;  // contraction: first index, extent
};

// A wait that ran out (or saw another run out) marks the CTA.
__device__ __forceinline__ bool flagged(GroupedShared* sh, bool ok) {
    if (!ok) *reinterpret_cast<volatile int*>(&sh->gave_up) = 1;
    return ok;
}
// The whole warp waits and agrees on the outcome.
__device__ __forceinline__ bool wait_warp(GroupedShared* sh, uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, flagged(sh, wait_full(bar, parity, &sh->gave_up)));
}
// An epilogue warp's wait lasts a tile: one lane looks every half microsecond
// (polling without a pause costs 2% of the products).
__device__ __forceinline__ bool wait_idle_warp(GroupedShared* sh, uint64_t* bar, uint32_t parity,
                                               int lane) {
    bool ok = true;
    if (lane == 0) {
        uint32_t i = 0;
        while (!mbar_try_wait(bar, parity)) {
            if (*reinterpret_cast<volatile int*>(&sh->gave_up) || ++i > kWaitPolls) {
                ok = flagged(sh, false);
                break;
            }
            __nanosleep(500);
        }
    }
    return __shfl_sync(0xffffffffu, (int)ok, 0);
}
__device__ __forceinline__ bool wait_peer_warp(GroupedShared* sh, uint64_t* bar, uint32_t parity,
                                               int lane) {
    const bool ok = lane != 0 || flagged(sh, wait_peer(bar, parity, &sh->gave_up));
    return __shfl_sync(0xffffffffu, (int)ok, 0);
}

__device__ __forceinline__ int column_tiles(int rows) {
    return (rows + kBN - 1) / kBN;
}

// A role's place among the groups: its tiles only go up.
struct Walk {
    int group = 0;
};

// Tile t of the launch.
__device__ __forceinline__ Tile tile_at(const GroupedArgs& A, const GroupedShared* sh, int t,
                                        Walk& walk) {
    Tile q;
    const int nm = (A.m + kPairM - 1) / kPairM;
    if (A.by_rows) {
        int lo = walk.group;  // the last group whose first tile is <= t
        while (lo <= A.E && sh->tile0[lo + 1] <= t) ++lo;
        walk.group = lo;
        const int r0 = sh->first[lo], rows = sh->first[lo + 1] - r0;
        const int nc = column_tiles(rows);
        // even tiles, in bands that reuse what of the weights they have loaded
        const int each = ((rows + nc - 1) / nc + 31) / 32 * 32;
        int l = t - sh->tile0[lo];
        const int band = l / (kBandC * nm);
        l -= band * kBandC * nm;
        const int wide = min(kBandC, nc - band * kBandC);
        const int c = band * kBandC + l % wide;
        q.group = lo >= 1 && lo <= A.E ? lo - 1 : -1;
        q.m0 = l / wide * kPairM;
        q.c0 = r0 + c * each;
        q.cols = min(each, rows - c * each);
        q.k0 = 0;
        q.depth = q.group >= 0 ? A.k : 0;
    } else {
        const int nc = column_tiles(A.c);
        q.group = t / (nm * nc);
        int l = t - q.group * nm * nc;
        const int band = l / (kBandC * nm);
        l -= band * kBandC * nm;
        const int wide = min(kBandC, nc - band * kBandC);
        q.m0 = l / wide * kPairM;
        q.c0 = (band * kBandC + l % wide) * kBN;
        q.cols = min(kBN, A.c - q.c0);
        q.k0 = sh->first[q.group + 1];
        q.depth = sh->first[q.group + 2] - q.k0;
    }
    return q;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Group bounds and tile counts, by one warp. Offsets that fall or leave [0, S]
// are brought back: no tile then reaches outside the rows.
__device__ void plan_groups(const GroupedArgs& A, GroupedShared* sh, int lane) {
    const int nm = (A.m + kPairM - 1) / kPairM;
    int reach = 0, tiles = 0;  // running maximum of the offsets, running tile count
    if (lane == 0) sh->first[0] = 0;
    for (int base = 0; base <= A.E + 1; base += 32) {
        // entry i: first row of group i + 1 (offsets[i]; S after the last)
        const int i = base + lane;
        int o = i <= A.E ? min(max(A.offsets[i], 0), A.S) : A.S;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, o, s);
            if (lane >= s) o = max(o, v);
        }
        o = max(o, reach);
        int before = __shfl_up_sync(0xffffffffu, o, 1);
        if (lane == 0) before = reach;
        int n = i <= A.E + 1 ? column_tiles(o - before) * nm : 0;  // tiles of group i
        int sum = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, s);
            if (lane >= s) sum += v;
        }
        if (i <= A.E + 1) {
            sh->first[i + 1] = o;
            sh->tile0[i] = tiles + sum - n;
        }
        reach = __shfl_sync(0xffffffffu, o, 31);
        tiles += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) sh->tiles = A.by_rows ? tiles : A.E * nm * column_tiles(A.c);
}

// The accumulators to memory. D has the output's contiguous dimension on the
// lanes, so 32 x 32 pieces are turned in the warp's corner of shared memory: 16-bit
// fragments are stored transposed, and leave as 16-byte pieces of output rows, 8
// rows of 64 bytes to an instruction. Where output rows do not start on 16 bytes a
// lane stores its elements one by one: 64 consecutive bytes of a row to an
// instruction (pairs read back from the corner were slower, 56 us against 20 us
// for 5003 x 1001 x 777).
// Byte of lane m of column `row` in the corner: 32 rows of 64 bytes, whose four
// 16-byte pieces are turned by the row's bits 1 and 2, which spreads the accesses
// over all banks.
__device__ __forceinline__ int turned(int row, int m) {
    return row * 64 + ((m >> 3 ^ (row >> 1 & 3)) << 4) + (m & 7) * 2;
}

template <typename T>
__device__ __forceinline__ void epilogue(const GroupedArgs& A, GroupedShared* sh, int rank,
                                         int quarter, int lane) {
    int used = 0;  // accumulators so far
    const uint32_t release0 = map_to_rank(&sh->acc_empty[0], 0);
    const uint32_t release1 = map_to_rank(&sh->acc_empty[1], 0);
    uint8_t* const turn = sh->turn[quarter];
    const uint32_t turn0 = smem_u32(turn);
    const bool wide = A.ldo % 8 == 0 && A.m % 8 == 0 && A.out_group % 8 == 0 &&
                      (reinterpret_cast<uintptr_t>(A.out) & 15) == 0;
    Walk walk;
    for (int t = blockIdx.x / 2; t < sh->tiles; t += gridDim.x / 2) {
        const Tile q = tile_at(A, sh, t, walk);
        const int m0 = q.m0 + rank * kBM + quarter * 32;  // the warp's lanes
        T* const out = reinterpret_cast<T*>(A.out) +
                       (A.by_rows ? 0 : q.group * A.out_group) + (int64_t)q.c0 * A.ldo + m0;
        const int buf = used & 1;
        bool ok = true;
        if (q.depth > 0) {
            ok = wait_idle_warp(sh, &sh->acc_full[buf], (used >> 1) & 1, lane);
            tc_fence_after();
        }
        const bool held = q.depth > 0 && ok;
        const uint32_t acc = sh->tmem + ((uint32_t)(quarter * 32) << 16) + buf * kBN;
        const uint32_t fill = __float_as_uint(ok ? 0.f : NAN);
        if (wide) {
            // piece lane % 4 of rows lane / 4 + 8 i
            const int r0 = lane >> 2, m = (lane & 3) * 8;
            T* o = out + (int64_t)r0 * A.ldo + m;
            for (int c = 0; c < q.cols; c += 32) {
                uint32_t v[2][16];
                if (held) {
                    tmem_ld16x32(acc + c, v[0]);
                    tmem_ld16x32(acc + (16u << 16) + c, v[1]);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[0][i] = v[1][i] = fill;
                }
                if (c + 32 >= q.cols && q.depth > 0) {
                    // the accumulator is read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_signal_cluster(buf ? release1 : release0);
                }
                __syncwarp();  // the last piece's reads of `turn` are done
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // lanes 16 h ..
#pragma unroll
                    for (int g = 0; g < 2; ++g) {  // columns 16 g ..: two fragments
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = pack_pair<T>(__uint_as_float(v[h][8 * g + 2 * i]),
                                                __uint_as_float(v[h][8 * g + 2 * i + 1]));
                        // matrix l / 8: its lanes 16 h + 8 (l / 8 % 2), columns 16 g + 8 (l / 16)
                        const int row = 16 * g + 8 * (lane >> 4) + (lane & 7);
                        const int p = 2 * h + (lane >> 3 & 1);
                        st_matrix4_trans(turn0 + turned(row, p * 8), w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r0 + 8 * i;
                    const uint4 x = *reinterpret_cast<const uint4*>(turn + turned(row, m));
                    if (m0 + m < A.m && c + row < q.cols)
                        *reinterpret_cast<uint4*>(o + (int64_t)i * 8 * A.ldo) = x;
                }
                o += 32 * A.ldo;
            }
        } else {
            T* o = out + lane;
            for (int c = 0; c < q.cols; c += 32) {
                uint32_t v[32];
                if (held) {
                    tmem_ld32(acc + c, v);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = fill;
                }
                if (m0 + lane < A.m) {
                    if (c + 32 <= q.cols) {
#pragma unroll
                        for (int i = 0; i < 32; ++i, o += A.ldo) *o = (T)__uint_as_float(v[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i, o += A.ldo)
                            if (c + i < q.cols) *o = (T)__uint_as_float(v[i]);
                    }
                }
                __syncwarp();
            }
            if (q.depth > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_signal_cluster(buf ? release1 : release0);
            }
        }
        if (q.depth > 0) ++used;
    }
}

// A place in the ring of stages: the stage, and how often the ring went round.
template <int N>
struct Ring {
    int s = 0;
    uint32_t lap = 0;
    __device__ __forceinline__ void next() {
        if (++s == N) {
            s = 0;
            ++lap;
        }
    }
    __device__ __forceinline__ void skip(int n) {
        s += n;
        lap += s / N;
        s %= N;
    }
};

// Rows behind the contraction that the last of its 16-deep steps reads: of the
// next group where the rows are the contraction (else the copy engine's zeros).
__device__ __forceinline__ int cleared_rows(const GroupedArgs& A, int left) {
    return A.by_rows || left >= kBK ? 0 : (left + 15) / 16 * 16 - left;
}

// Clear them in a stage of MN-major operands, by one warp: a row is 128 bytes of
// each box of 64 columns, whatever the swizzle.
__device__ __forceinline__ void clear_rows(uint8_t* stage, int n, int left, int rows, int lane) {
    const int boxes = 2 + (n / 2 + 63) / 64;
    for (int i = lane; i < boxes * rows * 8; i += 32) {
        const int x = i / (rows * 8), r = i / 8 % rows;
        *reinterpret_cast<uint4*>(stage + x * kBox + (left + r) * 128 + i % 8 * 16) =
            make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
    __syncwarp();
}

__global__ void __launch_bounds__(kThreads, 1) k_grouped(const __grid_constant__ GroupedArgs A) {
    extern __shared__ uint8_t dyn[];
    uint8_t* const stages =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    GroupedShared* const sh =
        reinterpret_cast<GroupedShared*>(stages + kStages * kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int t0 = blockIdx.x / 2, dt = gridDim.x / 2;  // the pair's tiles

    // launched as a programmatic dependent: the set-up runs beside the end of the
    // kernel before, nothing global is touched before pdl_wait() (64 groups of 3 rows
    // with their copies and sum: 49.6 -> 46.0 us)
    if (warp == 0) {
        pdl_wait();
        plan_groups(A, sh, lane);
    } else if (warp == 1) {
        tmem_alloc_pair(&sh->tmem, kTmemCols);
        if (lane == 0) {
            for (int s = 0; s < kStages; ++s) {
                mbar_init(&sh->full[s], 1);
                mbar_init(&sh->empty[s], 1);
                mbar_init(&sh->part[s], 1);
                mbar_init(&sh->ready[s], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->acc_full[i], 1);
                mbar_init(&sh->acc_empty[i], 8);  // four warps of each CTA
            }
            mbar_init(&sh->drain, 1);
            sh->gave_up = 0;
            mbar_init_fence();
        }
        tc_fence_before();
    } else if (warp == 2 && lane == 0) {
        tma_prefetch_map(&A.a);
        tma_prefetch_map(&A.b);
        tma_prefetch_map(&A.b32);
    }
    __syncthreads();
    cluster_barrier();  // the peer's barriers exist
    tc_fence_after();
    pdl_wait();
    pdl_trigger();

    // The producer's and the MMA's few instructions a stage are serial time of the
    // pipeline (a stage lasts 512 cycles). Both loops are run by whole warps with
    // one elected lane acting, so that addresses and descriptors stay in uniform
    // registers; they are stepped, and the next barrier is looked at before the
    // current stage is issued.
    if (warp == 0) {
        Ring<kStages> ring;
        const uint32_t full0 = map_to_rank(&sh->full[0], 0);  // the leading CTA's
        const uint32_t part0 = map_to_rank(&sh->part[0], 1);
        const bool leader = elect_one();
        bool ok = true;
        Walk walk;
        for (int t = t0; ok && t < sh->tiles; t += dt) {
            const Tile q = tile_at(A, sh, t, walk);
            // this CTA's lanes and its half of the columns
            const int m0 = q.m0 + rank * kBM;
            const int half = (q.cols + 31) / 32 * 16, c0 = q.c0 + rank * half;
            // boxes of 64 columns (MN-major), of 32 or one of all (K-major)
            const bool narrow = !A.b_mn && half <= 64;
            const int boxes = A.b_mn ? (half + 63) / 64 : narrow ? (half + 31) / 32 : 1;
            const int box = A.b_mn ? kBox : (narrow ? 32 : kHalf) * kBK * 2;
            const int z = A.by_rows ? q.group : 0;
            const uint32_t bytes = kABytes + boxes * box;
            const CUtensorMap* const mb = narrow ? &A.b32 : &A.b;
            const int end = q.k0 + q.depth;
            const int cleared = cleared_rows(A, (q.depth - 1) % kBK + 1);
            for (int k = q.k0; k < end; k += kBK) {
                if (ring.lap) ok = wait_warp(sh, &sh->empty[ring.s], (ring.lap - 1) & 1);
                if (!ok) break;
                if (leader) {
                    uint8_t* const sa = stages + ring.s * kStageBytes;
                    uint8_t* const sb = sa + kABytes;
                    const bool clear = cleared > 0 && k + kBK > end;
                    uint32_t bar = full0 + ring.s * 8;
                    if (rank == 0) {
                        mbar_expect_tx(&sh->full[ring.s], clear ? bytes : 2 * bytes);
                    } else if (clear) {
                        mbar_expect_tx(&sh->part[ring.s], bytes);
                        bar = part0 + ring.s * 8;
                    }
                    if (A.a_mn) {
                        tma_load_3d_pair(sa, &A.a, m0, k, z, bar);
                        tma_load_3d_pair(sa + kBox, &A.a, m0 + 64, k, z, bar);
                    } else {
                        tma_load_3d_pair(sa, &A.a, k, m0, z, bar);
                    }
                    if (A.b_mn) {
                        tma_load_3d_pair(sb, mb, c0, k, 0, bar);
                        if (boxes > 1) tma_load_3d_pair(sb + kBox, mb, c0 + 64, k, 0, bar);
                    } else {
                        tma_load_3d_pair(sb, mb, k, c0, 0, bar);
                        if (boxes > 1) tma_load_3d_pair(sb + box, mb, k, c0 + 32, 0, bar);
                    }
                }
                __syncwarp();
                ring.next();
            }
        }
        // Normally every copy has been consumed by the time the pair's last
        // accumulator is. After a wait that ran out, copies may be in flight
        // without a barrier of this CTA to tell: leave them a millisecond.
        if (*reinterpret_cast<volatile int*>(&sh->gave_up))
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncwarp();
    } else if (warp == 1) {
        Ring<kStages> ring;
        uint32_t parts = 0;  // bit s: phase of part[s] / ready[s]
        int used = 0;
        bool ok = true;
        const bool leader = elect_one();
        const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem, 0);
        const uint32_t sa0 = smem_u32(stages), sb0 = sa0 + kABytes;
        const uint64_t da0 = A.a_mn ? smem_desc(sa0, kBox, 1024) : smem_desc(sa0, 16, 1024);
        const uint64_t db0 = A.b_mn ? smem_desc(sb0, kBox, 1024) : smem_desc(sb0, 16, 1024);
        // a step of 16: 16 rows of 128 bytes, or 32 bytes along them
        const uint32_t ja = (A.a_mn ? 2048 : 32) >> 4, jb = (A.b_mn ? 2048 : 32) >> 4;
        Walk walk;
        for (int t = t0; ok && t < sh->tiles; t += dt) {
            const Tile q = tile_at(A, sh, t, walk);
            if (q.depth <= 0) continue;
            const int n = (q.cols + 31) / 32 * 32;
            const int blocks = (q.depth + kBK - 1) / kBK;
            const int left = q.depth - (blocks - 1) * kBK;  // of the last block
            const int cleared = cleared_rows(A, left);
            if (rank != 0) {
                // the second CTA: only what has to be cleared
                ring.skip(blocks - 1);
                if (cleared > 0) {
                    const int st = ring.s;
                    ok = wait_warp(sh, &sh->part[st], parts >> st & 1);
                    if (!ok) break;
                    parts ^= 1u << st;
                    clear_rows(stages + st * kStageBytes, n, left, cleared, lane);
                    if (lane == 0) mbar_arrive_cluster(map_to_rank(&sh->ready[st], 0));
                }
                ring.next();
                continue;
            }
            const int buf = used & 1;
            if (used >= 2) ok = wait_warp(sh, &sh->acc_empty[buf], (used / 2 - 1) & 1);
            if (!ok) break;
            const uint32_t d = tmem + buf * kBN;
            const uint32_t idesc = mma_idesc(A.bf16, A.a_mn, A.b_mn, kPairM, n);
            const int whole = left == kBK ? blocks : blocks - 1;
            bool seen = whole > 0 && mbar_try_wait(&sh->full[ring.s], ring.lap & 1);
            for (int i = 0; i < whole; ++i) {
                if (!__all_sync(0xffffffffu, seen))
                    ok = wait_warp(sh, &sh->full[ring.s], ring.lap & 1);
                if (!ok) break;
                const int st = ring.s;
                ring.next();
                seen = i + 1 < whole && mbar_try_wait(&sh->full[ring.s], ring.lap & 1);
                tc_fence_after();
                if (leader) {
                    const uint64_t da = da0 + st * (kStageBytes >> 4);
                    const uint64_t db = db0 + st * (kStageBytes >> 4);
                    mma_f16_pair(d, da, db, idesc, i > 0);
                    mma_f16_pair(d, da + ja, db + jb, idesc, true);
                    mma_f16_pair(d, da + 2 * ja, db + 2 * jb, idesc, true);
                    mma_f16_pair(d, da + 3 * ja, db + 3 * jb, idesc, true);
                    mma_commit_pair(&sh->empty[st]);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (whole < blocks) {  // the last block, of fewer steps
                const int st = ring.s;
                ok = wait_warp(sh, &sh->full[st], ring.lap & 1);
                if (!ok) break;
                if (cleared > 0) {
                    clear_rows(stages + st * kStageBytes, n, left, cleared, lane);
                    ok = wait_peer_warp(sh, &sh->ready[st], parts >> st & 1, lane);
                    if (!ok) break;
                    parts ^= 1u << st;
                }
                tc_fence_after();
                if (leader) {
                    const uint64_t da = da0 + st * (kStageBytes >> 4);
                    const uint64_t db = db0 + st * (kStageBytes >> 4);
                    for (int j = 0; j < (left + 15) / 16; ++j)
                        mma_f16_pair(d, da + j * ja, db + j * jb, idesc, whole + j > 0);
                    mma_commit_pair(&sh->empty[st]);
                }
                __syncwarp();
                ring.next();
            }
            if (leader) mma_commit_pair(&sh->acc_full[buf]);
            __syncwarp();
            ++used;
        }
        if (!ok && rank == 0) {
            if (leader) mma_commit_pair(&sh->drain);
            __syncwarp();
            mbar_wait(&sh->drain, 0);
        }
        __syncwarp();
    } else {
        if (A.bf16) epilogue<__nv_bfloat16>(A, sh, rank, warp & 3, lane);
        else epilogue<__half>(A, sh, rank, warp & 3, lane);
    }
    tc_fence_before();
    __syncthreads();
    cluster_barrier();  // neither CTA reads or signals the other any more
    if (warp == 1) {
        tc_fence_after();
        tmem_free_pair(sh->tmem, kTmemCols);
    }
}

// dst[g][r][0..ld) = src: an operand whose rows do not start on 16 bytes, laid
// out so that they do (ld is the width rounded up to 8 elements, the padding 0).
// Eight elements a thread, read one by one and written at once.
__global__ void __launch_bounds__(256) k_grouped_pack(const uint16_t* src, int64_t sg, int64_t sr,
                                                      unsigned rows, int width, unsigned pieces,
                                                      int64_t total, uint4* dst) {
    pdl_wait();
    pdl_trigger();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * 256) {
        const unsigned r = (unsigned)(i / pieces), x = (unsigned)(i - (int64_t)r * pieces) * 8;
        const uint16_t* const s = src + (int64_t)(r / rows) * sg + (int64_t)(r % rows) * sr + x;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (int)x + e < width ? s[e] : 0;
        dst[i] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16,
                            v[6] | v[7] << 16);
    }
}

// An operand: `groups` matrices of `rows` rows, `width` consecutive elements each.
struct Operand {
    const void* p;
    int64_t groups, rows, width, sg, sr;

    // what the copy engine takes: every row starts on 16 bytes
    bool aligned() const {
        return (uintptr_t)p % 16 == 0 && (rows == 1 || (sr % 8 == 0 && sr >= 8)) &&
               (groups == 1 || (sg % 8 == 0 && sg >= 8));
    }
};

PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (PFN_cuTensorMapEncodeTiled_v12000)p;
    }();
    return fn;
}

// Boxes of 64 x `box_rows` elements, 128-byte swizzle; outside reads as zero.
int encode(CUtensorMap* map, const Operand& o, bool bf16, uint32_t box_rows) {
    auto enc = map_encoder();
    if (!enc) return fail(SK_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int64_t sr = o.rows == 1 ? (o.width + 7) / 8 * 8 : o.sr;
    const int64_t sg = o.groups == 1 ? sr * o.rows : o.sg;
    const cuuint64_t dims[3] = {(cuuint64_t)o.width, (cuuint64_t)o.rows, (cuuint64_t)o.groups};
    const cuuint64_t strides[2] = {(cuuint64_t)sr * 2, (cuuint64_t)sg * 2};
    const cuuint32_t box[3] = {64, box_rows, 1};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r =
        enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            (void*)o.p, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(SK_ERR_LAYOUT, "an operand cannot be described to the copy engine (" +
                                       std::to_string((int)r) + "): " + std::to_string(o.width) +
                                       " x " + std::to_string(o.rows) + " x " +
                                       std::to_string(o.groups) + ", strides " +
                                       std::to_string(sr) + ", " + std::to_string(sg));
    return SK_OK;
}

constexpr size_t kGroupedSmem = 1024 + kStages * kStageBytes + sizeof(GroupedShared);
static_assert(kGroupedSmem <= 232448, "shared memory of one CTA");

int launch_grouped(GroupedArgs& A, const Operand& a, const Operand& b, int64_t tiles,
                   cudaStream_t s) {
    if (!a.aligned() || !b.aligned())
        return fail(SK_ERR_LAYOUT, "operand rows must start on 16 bytes (sk_grouped_pack)");
    // the runtime calls first: they bind the device's context to a thread that has
    // none yet (autograd's), which the map encoder needs
    int dev = 0, sms = 0;
    SK_CUDA(cudaGetDevice(&dev));
    SK_CUDA(cudaSetDevice(dev));
    SK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    SK_CUDA(cudaFuncSetAttribute(k_grouped, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kGroupedSmem));
    int rc = encode(&A.a, a, A.bf16, A.a_mn ? kBK : kBM);
    if (rc == SK_OK) rc = encode(&A.b, b, A.bf16, A.b_mn ? kBK : kHalf);
    if (rc == SK_OK) rc = encode(&A.b32, b, A.bf16, A.b_mn ? kBK : 32);
    if (rc != SK_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min<int64_t>(tiles, sms / 2));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kGroupedSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    SK_CUDA(cudaLaunchKernelEx(&cfg, k_grouped, A));
    return SK_OK;
}

int check_grouped(int dtype, int64_t S, int64_t K, int64_t N, int64_t E, const int* offsets) {
    if (dtype != SK_BF16 && dtype != SK_FP16)
        return fail(SK_ERR_ARG, "grouped products take bf16 or fp16");
    if (S <= 0 || K <= 0 || N <= 0 || E <= 0)
        return fail(SK_ERR_ARG, "S, K, N and E must be positive");
    if (E > kMaxGroups) return fail(SK_ERR_ARG, "at most 1024 groups");
    if (S > (1 << 30) || K > (1 << 30) || N > (1 << 30))
        return fail(SK_ERR_ARG, "S, K and N must be at most 2^30");
    if (E * std::max(K, N) > INT32_MAX)
        return fail(SK_ERR_ARG, "E * K and E * N must be below 2^31");
    if (!offsets) return fail(SK_ERR_ARG, "offsets is NULL");
    return SK_OK;
}

// Tiles of a launch, at most (the runs are known to the device alone).
int64_t most_tiles(int64_t m, int64_t c, int64_t groups) {
    return (m + kPairM - 1) / kPairM * ((c + kBN - 1) / kBN + groups);
}

// W_e's axes as an operand: rows of the unit-stride axis.
Operand weight_operand(const void* w, int64_t E, int64_t K, int64_t N, int64_t se, int64_t sk_,
                       int64_t sn) {
    if (sn == 1) return Operand{w, E, K, N, se, sk_};
    return Operand{w, E, N, K, se, sn};
}

int check_weight(int64_t se, int64_t sk_, int64_t sn) {
    if (se < 0 || sk_ < 0 || sn < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    if (sn != 1 && sk_ != 1)
        return fail(SK_ERR_LAYOUT, "one axis of the weights must have unit stride");
    return SK_OK;
}

}  // namespace
}  // namespace sk

extern "C" {

int sk_grouped_pack(const void* src, int64_t groups, int64_t rows, int64_t width, int64_t sg,
                    int64_t sr, void* dst, void* stream) {
    using namespace sk;
    clear_error();
    if (!src || !dst) return fail(SK_ERR_ARG, "src or dst is NULL");
    if (groups <= 0 || rows <= 0 || width <= 0)
        return fail(SK_ERR_ARG, "groups, rows and width must be positive");
    if (rows > INT32_MAX || width > (1 << 30) || groups > INT32_MAX / rows)
        return fail(SK_ERR_ARG, "groups * rows must be below 2^31 and width at most 2^30");
    if (sg < 0 || sr < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    if ((uintptr_t)src % 2 != 0 || (uintptr_t)dst % 16 != 0)
        return fail(SK_ERR_LAYOUT, "src must be 2-byte and dst 16-byte aligned");
    const int64_t pieces = (width + 7) / 8, total = groups * rows * pieces;
    const unsigned grid = (unsigned)std::min<int64_t>((total + 255) / 256, 148 * 32);
    launch_pdl(k_grouped_pack, dim3(grid), dim3(256), 0, (cudaStream_t)stream,
               (const uint16_t*)src, sg, sr, (unsigned)rows, (int)width, (unsigned)pieces, total,
               (uint4*)dst);
    SK_LAUNCHED("k_grouped_pack");
    return SK_OK;
}

int sk_grouped_matmul(const void* x, int dtype, int64_t S, int64_t K, int64_t ldx, const void* w,
                      int64_t E, int64_t N, int64_t swe, int64_t swk, int64_t swn,
                      const int* offsets, void* y, void* stream) {
    using namespace sk;
    clear_error();
    int rc = check_grouped(dtype, S, K, N, E, offsets);
    if (rc == SK_OK) rc = check_weight(swe, swk, swn);
    if (rc != SK_OK) return rc;
    if (!x || !w || !y) return fail(SK_ERR_ARG, "x, w or y is NULL");
    if (ldx < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    GroupedArgs A{};
    A.out = y;
    A.ldo = N;
    A.offsets = offsets;
    A.E = (int)E;
    A.S = (int)S;
    A.m = (int)N;
    A.k = (int)K;
    A.by_rows = true;
    A.a_mn = swn == 1;
    A.b_mn = false;
    A.bf16 = dtype == SK_BF16;
    const int64_t tiles = most_tiles(N, S, E + 2);
    if (tiles > INT32_MAX) return fail(SK_ERR_ARG, "the output has too many tiles");
    const Operand ow = weight_operand(w, E, K, N, swe, swk, swn);
    const Operand ox{x, 1, S, K, 0, ldx};
    return launch_grouped(A, ow, ox, tiles, (cudaStream_t)stream);
}

int sk_grouped_matmul_weight(const void* x, int dtype, int64_t S, int64_t K, int64_t ldx,
                             const void* dy, int64_t N, int64_t ldy, const int* offsets,
                             int64_t E, void* dw, int transposed, void* stream) {
    using namespace sk;
    clear_error();
    const int rc = check_grouped(dtype, S, K, N, E, offsets);
    if (rc != SK_OK) return rc;
    if (!x || !dy || !dw) return fail(SK_ERR_ARG, "x, dy or dw is NULL");
    if (ldx < 0 || ldy < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    GroupedArgs A{};
    A.out = dw;
    A.out_group = K * N;
    A.offsets = offsets;
    A.E = (int)E;
    A.S = (int)S;
    A.by_rows = false;
    A.a_mn = A.b_mn = true;
    A.bf16 = dtype == SK_BF16;
    Operand ox{x, 1, S, K, 0, ldx}, og{dy, 1, S, N, 0, ldy};
    A.m = (int)(transposed ? K : N);
    A.c = (int)(transposed ? N : K);
    A.ldo = A.m;
    const int64_t tiles = (A.m + kPairM - 1) / kPairM * (int64_t)((A.c + kBN - 1) / kBN) * E;
    if (tiles > INT32_MAX) return fail(SK_ERR_ARG, "the output has too many tiles");
    return launch_grouped(A, transposed ? ox : og, transposed ? og : ox, tiles,
                          (cudaStream_t)stream);
}

}  // extern "C"
