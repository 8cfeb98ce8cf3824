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
// c, of any multiple of 16 up to 256, on its columns. For `rows` c is the ragged
// dimension: the instruction's N is chosen per tile, so a group of r rows costs
// ceil(r / 16) * 16 columns and not whole tiles, and the weights are the operand
// that is always full. For `weights` the last block of a run's contraction holds
// rows of the next group; they are cleared in shared memory before they are used
// (a zero in one operand alone would not do: 0 * inf).
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "sk_internal.h"
#include "sk_tcgen05.cuh"

namespace sk {
namespace {

constexpr int kBM = 128;    // lanes: the output's contiguous dimension
constexpr int kBN = 256;    // most columns of a tile
constexpr int kBK = 64;     // contraction of a stage: one 128-byte swizzled row
constexpr int kStages = 4;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kBBytes = kBN * kBK * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kBandC = 8;   // column tiles that share a pass over the weights
constexpr int kThreads = 192;  // producer warp, MMA warp, four epilogue warps
constexpr int kMaxGroups = 1024;
constexpr uint32_t kTmemCols = 512;  // two accumulators

struct GroupedArgs {
    CUtensorMap a, b, b32;  // b32: boxes of 32 columns, for narrow tiles
    void* out;
    int64_t ldo, out_group;  // elements from column to column, group to group
    const int* offsets;
    int E, S;   // groups, rows
    int m, c, k;  // extents; c (rows) or k (weights) is the ragged one and unused
    bool by_rows, a_mn, b_mn, bf16;
};

struct alignas(8) GroupedShared {
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
    uint32_t tmem;
    int gave_up;  // a bounded wait ran out: the CTA's remaining tiles become NaN
    int tiles;
    // groups 0..E+1: the rows before the first group, the groups, the rows
    // behind the last; rows in no group are zero
    int first[kMaxGroups + 3];  // first row of each
    int tile0[kMaxGroups + 3];  // first tile of each (by_rows)
};

struct Tile {
    int group;      // 0..E-1, or -1: rows of no group
    int m0, c0;     // first lane / column of the output
    int cols;       // columns of the output
    int k0, depth;  // contraction: first index, extent
};

__device__ __forceinline__ bool wait_or_give_up(GroupedShared* sh, uint64_t* bar,
                                                uint32_t parity) {
    for (uint32_t i = 0; i < kWaitPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*reinterpret_cast<volatile int*>(&sh->gave_up)) return false;
    }
    *reinterpret_cast<volatile int*>(&sh->gave_up) = 1;
    return false;
}

__device__ __forceinline__ int column_tiles(int rows) { return (rows + kBN - 1) / kBN; }

// Tile t of the launch.
__device__ __forceinline__ Tile tile_at(const GroupedArgs& A, const GroupedShared* sh, int t) {
    Tile q;
    const int nm = (A.m + kBM - 1) / kBM;
    if (A.by_rows) {
        int lo = 0, hi = A.E + 1;  // the last group whose first tile is <= t
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (sh->tile0[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        const int r0 = sh->first[lo], rows = sh->first[lo + 1] - r0;
        const int nc = column_tiles(rows);
        // even tiles, in bands that reuse what of the weights they have loaded
        const int each = ((rows + nc - 1) / nc + 15) / 16 * 16;
        int l = t - sh->tile0[lo];
        const int band = l / (kBandC * nm);
        l -= band * kBandC * nm;
        const int wide = min(kBandC, nc - band * kBandC);
        const int c = band * kBandC + l % wide;
        q.group = lo >= 1 && lo <= A.E ? lo - 1 : -1;
        q.m0 = l / wide * kBM;
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
        q.m0 = l / wide * kBM;
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
    const int nm = (A.m + kBM - 1) / kBM;
    int reach = 0, tiles = 0;  // running maximum of the offsets, running tile count
    if (lane == 0) sh->first[0] = 0;
    for (int base = 0; base <= A.E + 1; base += 32) {
        // entry i: first row of group i + 1 (offsets[i]; S after the last)
        const int i = base + lane;
        int o = i <= A.E ? min(max(__ldg(A.offsets + i), 0), A.S) : A.S;
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

template <typename T>
__device__ __forceinline__ void epilogue(const GroupedArgs& A, GroupedShared* sh, int quarter,
                                         int lane) {
    int used = 0;  // accumulators so far
    for (int t = blockIdx.x; t < sh->tiles; t += gridDim.x) {
        const Tile q = tile_at(A, sh, t);
        T* const out = reinterpret_cast<T*>(A.out) +
                       (A.by_rows ? 0 : q.group * A.out_group) + (int64_t)q.c0 * A.ldo;
        const int m = q.m0 + quarter * 32 + lane;
        const int buf = used & 1;
        bool ok = true;
        if (q.depth > 0) {
            ok = wait_or_give_up(sh, &sh->acc_full[buf], (used >> 1) & 1);
            tc_fence_after();
        }
        // pairs of lanes exchange so that each stores two neighbours of a column
        const bool paired = A.ldo % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3) == 0;
        for (int c = 0; c < q.cols; c += 32) {
            uint32_t v[32];
            if (q.depth > 0 && ok) {
                tmem_ld32(sh->tmem + ((uint32_t)(quarter * 32) << 16) + buf * kBN + c, v);
                tmem_ld_wait();
            } else {
                const float fill = ok ? 0.f : NAN;
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fill);
            }
            if (paired) {
                const int odd = lane & 1;
                T* o = out + (int64_t)(c + odd) * A.ldo + (m - odd);
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float mine = __uint_as_float(odd ? v[i + 1] : v[i]);
                    const float send = __uint_as_float(odd ? v[i] : v[i + 1]);
                    const float other = __shfl_xor_sync(0xffffffffu, send, 1);
                    const uint32_t w = odd ? pack_pair<T>(other, mine) : pack_pair<T>(mine, other);
                    if (c + i + odd < q.cols) {
                        if (m - odd + 1 < A.m) *reinterpret_cast<uint32_t*>(o) = w;
                        else if (m - odd < A.m)
                            *reinterpret_cast<uint16_t*>(o) = (uint16_t)w;
                    }
                    o += 2 * A.ldo;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i < q.cols && m < A.m)
                        out[(int64_t)(c + i) * A.ldo + m] = (T)__uint_as_float(v[i]);
            }
        }
        if (q.depth > 0) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->acc_empty[buf]);
            ++used;
        }
    }
}

__global__ void __launch_bounds__(kThreads, 1) k_grouped(const __grid_constant__ GroupedArgs A) {
    extern __shared__ uint8_t dyn[];
    uint8_t* const stages =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);
    GroupedShared* const sh = reinterpret_cast<GroupedShared*>(stages + kStages * kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 0) {
        plan_groups(A, sh, lane);
    } else if (warp == 1) {
        tmem_alloc(&sh->tmem, kTmemCols);
        if (lane == 0) {
            for (int s = 0; s < kStages; ++s) {
                mbar_init(&sh->full[s], 1);
                mbar_init(&sh->empty[s], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->acc_full[i], 1);
                mbar_init(&sh->acc_empty[i], 4);
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
    tc_fence_after();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;  // stages filled
            for (int t = blockIdx.x; t < sh->tiles; t += gridDim.x) {
                const Tile q = tile_at(A, sh, t);
                bool ok = true;
                for (int kb = 0; kb < q.depth; kb += kBK, ++it) {
                    const int s = it % kStages;
                    if (it >= kStages)
                        ok = wait_or_give_up(sh, &sh->empty[s], (it / kStages - 1) & 1);
                    if (!ok) break;
                    uint8_t* const sa = stages + s * kStageBytes;
                    uint8_t* const sb = sa + kABytes;
                    uint64_t* const bar = &sh->full[s];
                    const int z = A.by_rows ? q.group : 0;
                    const int k = q.k0 + kb;
                    // columns to bring: 32 at a time (K-major), 64 (MN-major)
                    const bool narrow = !A.b_mn && q.cols <= kBN / 2;
                    const int boxes = A.b_mn ? (q.cols + 63) / 64
                                             : narrow ? (q.cols + 31) / 32 : 1;
                    const int box = A.b_mn ? 64 * kBK * 2 : narrow ? 32 * kBK * 2 : kBBytes;
                    mbar_expect_tx(bar, kABytes + boxes * box);
                    if (A.a_mn) {
                        tma_load_3d(sa, &A.a, q.m0, k, z, bar);
                        tma_load_3d(sa + kABytes / 2, &A.a, q.m0 + 64, k, z, bar);
                    } else {
                        tma_load_3d(sa, &A.a, k, q.m0, z, bar);
                    }
                    if (A.b_mn) {
                        for (int i = 0; i < boxes; ++i)
                            tma_load_3d(sb + i * box, &A.b, q.c0 + 64 * i, k, 0, bar);
                    } else if (narrow) {
                        for (int i = 0; i < boxes; ++i)
                            tma_load_3d(sb + i * box, &A.b32, k, q.c0 + 32 * i, 0, bar);
                    } else {
                        tma_load_3d(sb, &A.b, k, q.c0, 0, bar);
                    }
                }
                if (!ok) break;
            }
            // the copies of the last stages have landed before the CTA may end
            for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
                mbar_wait(&sh->full[i % kStages], (i / kStages) & 1);
        }
    } else if (warp == 1) {
        uint32_t it = 0;
        int used = 0;
        bool ok = true;
        const uint32_t sbase = smem_u32(stages);
        for (int t = blockIdx.x; ok && t < sh->tiles; t += gridDim.x) {
            const Tile q = tile_at(A, sh, t);
            if (q.depth <= 0) continue;
            const int buf = used & 1;
            if (used >= 2) ok = wait_or_give_up(sh, &sh->acc_empty[buf], (used / 2 - 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = sh->tmem + buf * kBN;
            const int n = (q.cols + 15) / 16 * 16;
            const uint32_t idesc = mma_idesc(A.bf16, A.a_mn, A.b_mn, kBM, n);
            for (int kb = 0; kb < q.depth; kb += kBK, ++it) {
                const int s = it % kStages;
                ok = wait_or_give_up(sh, &sh->full[s], (it / kStages) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t sa = sbase + s * kStageBytes, sb = sa + kABytes;
                const int left = min(kBK, q.depth - kb), steps = (left + 15) / 16;
                if (!A.by_rows && left < steps * 16) {
                    // rows of the next group: both operands cleared, row by row
                    // (a row is 128 bytes of each box, whatever the swizzle)
                    const int boxes = 2 + (q.cols + 63) / 64, rows = steps * 16 - left;
                    uint8_t* const base = stages + s * kStageBytes;
                    for (int i = lane; i < boxes * rows * 8; i += 32) {
                        const int x = i / (rows * 8), r = i / 8 % rows;
                        *reinterpret_cast<uint4*>(base + x * (64 * kBK * 2) +
                                                  (left + r) * 128 + i % 8 * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) {
                    for (int j = 0; j < steps; ++j) {
                        const uint64_t da =
                            A.a_mn ? smem_desc(sa + j * 2048, kABytes / 2, 1024)
                                   : smem_desc(sa + j * 32, 16, 1024);
                        const uint64_t db = A.b_mn
                                                ? smem_desc(sb + j * 2048, 64 * kBK * 2, 1024)
                                                : smem_desc(sb + j * 32, 16, 1024);
                        mma_f16(d, da, db, idesc, kb + j > 0);
                    }
                    mma_commit(&sh->empty[s]);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (lane == 0) mma_commit(&sh->acc_full[buf]);
            __syncwarp();
            ++used;
        }
        if (!ok) {
            if (lane == 0) mma_commit(&sh->drain);
            __syncwarp();
            mbar_wait(&sh->drain, 0);
        }
    } else {
        if (A.bf16) epilogue<__nv_bfloat16>(A, sh, warp & 3, lane);
        else epilogue<__half>(A, sh, warp & 3, lane);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free(sh->tmem, kTmemCols);
    }
}

// dst[g][r][0..ld) = src: an operand whose rows do not start on 16 bytes, laid
// out so that they do (ld is the width rounded up to 8 elements).
__global__ void __launch_bounds__(256) k_grouped_pack(const uint16_t* src, int64_t sg, int64_t sr,
                                                      int64_t rows, int64_t width, int64_t ld,
                                                      int64_t total_rows, uint16_t* dst) {
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < total_rows;
         r += (int64_t)gridDim.x * 8) {
        const uint16_t* const s = src + r / rows * sg + r % rows * sr;
        uint16_t* const d = dst + r * ld;
        for (int64_t i = threadIdx.x & 31; i < width; i += 32) d[i] = s[i];
    }
}

// An operand: `groups` matrices of `rows` rows, `width` consecutive elements each.
struct Operand {
    const void* p;
    int64_t groups, rows, width, sg, sr;

    bool ready() const {
        return (uintptr_t)p % 16 == 0 && (rows == 1 || (sr % 8 == 0 && sr >= 8)) &&
               (groups == 1 || (sg % 8 == 0 && sg >= 8));
    }
    size_t packed_bytes() const {
        return ready() ? 0 : align_up((size_t)groups * rows * ((width + 7) / 8 * 8) * 2);
    }
    int pack(char*& ws, cudaStream_t s) {
        if (ready()) return SK_OK;
        const int64_t ld = (width + 7) / 8 * 8, total = groups * rows;
        const unsigned grid = (unsigned)std::min<int64_t>((total + 7) / 8, 148 * 16);
        k_grouped_pack<<<grid, 256, 0, s>>>((const uint16_t*)p, sg, sr, rows, width, ld, total,
                                            (uint16_t*)ws);
        SK_LAUNCHED("k_grouped_pack");
        const size_t used = packed_bytes();
        p = ws;
        sr = ld;
        sg = ld * rows;
        ws += used;
        return SK_OK;
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

int launch_grouped(GroupedArgs& A, Operand a, Operand b, int64_t tiles, char* ws,
                   cudaStream_t s) {
    // the runtime calls first: they bind the device's context to a thread that has
    // none yet (autograd's), which the map encoder needs
    int dev = 0, sms = 0;
    SK_CUDA(cudaGetDevice(&dev));
    SK_CUDA(cudaSetDevice(dev));
    SK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    SK_CUDA(cudaFuncSetAttribute(k_grouped, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kGroupedSmem));
    int rc = a.pack(ws, s);
    if (rc == SK_OK) rc = b.pack(ws, s);
    if (rc == SK_OK) rc = encode(&A.a, a, A.bf16, A.a_mn ? kBK : kBM);
    if (rc == SK_OK) rc = encode(&A.b, b, A.bf16, A.b_mn ? kBK : kBN);
    if (rc == SK_OK) rc = encode(&A.b32, b, A.bf16, A.b_mn ? kBK : 32);
    if (rc != SK_OK) return rc;
    k_grouped<<<(unsigned)std::min<int64_t>(tiles, sms), kThreads, kGroupedSmem, s>>>(A);
    SK_LAUNCHED("k_grouped");
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
    if (!offsets) return fail(SK_ERR_ARG, "offsets is NULL");
    return SK_OK;
}

// Tiles of a launch, at most (the runs are known to the device alone).
int64_t most_tiles(int64_t m, int64_t c, int64_t groups) {
    return (m + kBM - 1) / kBM * ((c + kBN - 1) / kBN + groups);
}

// W_e's axes as an operand: rows of the unit-stride axis.
Operand weight_operand(const void* w, int64_t E, int64_t K, int64_t N, int64_t se, int64_t sk_,
                       int64_t sn) {
    if (sn == 1) return Operand{w, E, K, N, se, sk_};
    return Operand{w, E, N, K, se, sn};
}

int check_weight(int64_t K, int64_t N, int64_t se, int64_t sk_, int64_t sn) {
    if (se < 0 || sk_ < 0 || sn < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    if (sn != 1 && sk_ != 1)
        return fail(SK_ERR_LAYOUT, "one axis of the weights must have unit stride");
    (void)K;
    (void)N;
    return SK_OK;
}

}  // namespace
}  // namespace sk

extern "C" {

size_t sk_grouped_matmul_workspace_bytes(const void* x, int64_t S, int64_t K, int64_t ldx,
                                         const void* w, int64_t E, int64_t N, int64_t swe,
                                         int64_t swk, int64_t swn) {
    using namespace sk;
    if (S <= 0 || K <= 0 || N <= 0 || E <= 0) return 0;
    return Operand{x, 1, S, K, 0, ldx}.packed_bytes() +
           weight_operand(w, E, K, N, swe, swk, swn).packed_bytes();
}

int sk_grouped_matmul(const void* x, int dtype, int64_t S, int64_t K, int64_t ldx, const void* w,
                      int64_t E, int64_t N, int64_t swe, int64_t swk, int64_t swn,
                      const int* offsets, void* y, void* workspace, size_t workspace_bytes,
                      void* stream) {
    using namespace sk;
    clear_error();
    int rc = check_grouped(dtype, S, K, N, E, offsets);
    if (rc == SK_OK) rc = check_weight(K, N, swe, swk, swn);
    if (rc != SK_OK) return rc;
    if (!x || !w || !y) return fail(SK_ERR_ARG, "x, w or y is NULL");
    if (ldx < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    const size_t need =
        sk_grouped_matmul_workspace_bytes(x, S, K, ldx, w, E, N, swe, swk, swn);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_grouped_matmul");
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
    return launch_grouped(A, weight_operand(w, E, K, N, swe, swk, swn),
                          Operand{x, 1, S, K, 0, ldx}, tiles, (char*)workspace,
                          (cudaStream_t)stream);
}

size_t sk_grouped_matmul_weight_workspace_bytes(const void* x, int64_t S, int64_t K, int64_t ldx,
                                                const void* dy, int64_t N, int64_t ldy) {
    using namespace sk;
    if (S <= 0 || K <= 0 || N <= 0) return 0;
    return Operand{x, 1, S, K, 0, ldx}.packed_bytes() +
           Operand{dy, 1, S, N, 0, ldy}.packed_bytes();
}

int sk_grouped_matmul_weight(const void* x, int dtype, int64_t S, int64_t K, int64_t ldx,
                             const void* dy, int64_t N, int64_t ldy, const int* offsets,
                             int64_t E, void* dw, int transposed, void* workspace,
                             size_t workspace_bytes, void* stream) {
    using namespace sk;
    clear_error();
    const int rc = check_grouped(dtype, S, K, N, E, offsets);
    if (rc != SK_OK) return rc;
    if (!x || !dy || !dw) return fail(SK_ERR_ARG, "x, dy or dw is NULL");
    if (ldx < 0 || ldy < 0) return fail(SK_ERR_LAYOUT, "negative strides");
    const size_t need = sk_grouped_matmul_weight_workspace_bytes(x, S, K, ldx, dy, N, ldy);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(SK_ERR_WORKSPACE, "workspace too small for sk_grouped_matmul_weight");
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
    const int64_t tiles = (A.m + kBM - 1) / kBM * (int64_t)((A.c + kBN - 1) / kBN) * E;
    if (tiles > INT32_MAX) return fail(SK_ERR_ARG, "the output has too many tiles");
    return launch_grouped(A, transposed ? ox : og, transposed ? og : ox, tiles,
                          (char*)workspace, (cudaStream_t)stream);
}

}  // extern "C"
