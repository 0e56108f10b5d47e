// Matrix-product engine of the language-model operators: 16-bit operands, fp32 accumulation on the
// 5th-generation tensor cores.
//   D[m, n] = sum over segments s, k  A_s[m, k] B_s[n, k]
// Either operand may be stored with k contiguous ("K-major") or with its row index contiguous
// ("MN-major": A' or B' in memory); both land in shared memory through tiled TMA in the 128-byte
// swizzle that the tensor core reads, and whatever lies outside a matrix arrives as zeros.
//
// Persistent kernel, warp-specialised:
//   warp 0     one lane issues the TMA loads of a ring of stages (64 k per stage)
//   warp 1     one lane issues tcgen05.mma; accumulators live in TMEM, two of them, so that
//   warps 2-5  read and store one tile (Epi) while the next is being computed.
// CG = 2 pairs two SMs on a 256 x BN tile: each CTA loads its 128 rows of A and half of B's rows, so a byte
// of B feeds twice the arithmetic; the even CTA's issuer drives both.  CG = 1 (128 x BN) is for products
// with too few tiles to occupy the pairs.  Every wait is bounded; when one runs out, the CTA sets the
// context's error word, lets its copies in flight land, frees its TMEM and returns.
#pragma once

#include "lm_common.cuh"
#include "tma_util.cuh"

namespace fitre {
namespace {

constexpr int G_THREADS = 192;
constexpr int G_KB = 64;   // k per stage: 128 bytes, one swizzle row

// Which tiles there are and where their operands come from.
struct TileGrid {
    int tilesM, tilesN;   // tiles of one product
    int total;            // over all products of the batch
    int per;              // tiles per product
    int triangle;         // 1: only tiles with column <= row (the product is symmetric)
    int kblocks, nseg;    // stages per segment, segments (map index = segment)
    int za, zb;           // 1: the batch index is the operand map's third coordinate
    uint32_t idesc;
    int *err;
};

template <class P>
struct alignas(64) GemmArgs {
    CUtensorMap a[2], b[2];
    TileGrid g;
    P epi;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded: false after about a second.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(bar, parity))
        if (clock64() - t0 > (1LL << 31)) return false;
    return true;
}
template <int CG>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    if constexpr (CG == 2)   // `bar` may be the other CTA's of the pair
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on `bar` (of both CTAs of a pair) once every product issued so far has been computed.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
            ::"r"(bar), "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                     : "memory");
}
// 32 consecutive accumulator columns of this thread's row.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: rows 128 bytes apart, groups of 8 rows
// 1024 bytes apart.  MN-major: blocks of 64 rows x 64 k (8192 bytes, the leading offset), in each the
// 8-deep groups of k 1024 bytes apart.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(MN ? (8192 >> 4) : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// 16 k further on: 32 bytes along a swizzled row, or two 8-deep groups.
template <bool MN> constexpr uint32_t k_step = (MN ? 2048u : 32u) >> 4;

struct TileAt { int batch, m, n; };
__device__ __forceinline__ TileAt tile_at(const TileGrid &g, int t) {
    TileAt r;
    r.batch = t / g.per;
    int i = t - r.batch * g.per;
    if (g.triangle) {
        int row = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
        while (row * (row + 1) / 2 > i) --row;
        while ((row + 1) * (row + 2) / 2 <= i) ++row;
        r.m = row;
        r.n = i - row * (row + 1) / 2;
    } else {
        // bands of 8 tile rows, column by column: the tiles in flight share operands in L2
        const int band = i / (8 * g.tilesN), first = band * 8;
        const int high = min(8, g.tilesM - first);
        i -= band * 8 * g.tilesN;
        r.m = first + i % high;
        r.n = i / high;
    }
    return r;
}

template <int CG, int BN> struct GemmLayout {
    static constexpr int BROWS = BN / CG;                     // rows of B one CTA loads
    static constexpr int ABYTES = 128 * 128, BBYTES = BROWS * 128;
    static constexpr int STAGE = ABYTES + BBYTES;
    static constexpr int STAGES = 200 * 1024 / STAGE < 8 ? 200 * 1024 / STAGE : 8;
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;
    static constexpr int TMEM_COLS = 2 * BN;
};

// Epi: { using Params; static constexpr bool kTwoMaps (B's rows come half from map 0, half from map 1);
//        static void store(const Params &, TileAt, int row, uint32_t tmem) } -- called by all 128 epilogue threads,
// `row` = global row of the thread's accumulator row, `tmem` = address of its first column.
template <int CG, int BN, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(G_THREADS, 1)
tile_gemm_kernel(const __grid_constant__ GemmArgs<typename Epi::Params> p) {
    using L = GemmLayout<CG, BN>;
    constexpr int ST = L::STAGES;
    extern __shared__ unsigned char smraw[];
    unsigned char *sm = (unsigned char *)(((uintptr_t)smraw + 1023) & ~(uintptr_t)1023);
    unsigned long long *bars = (unsigned long long *)(sm + ST * L::STAGE);
    // [0, 8) stage full, [8, 16) stage free, [16, 18) accumulator full, [18, 20) accumulator free
    uint32_t *tmem_slot = (uint32_t *)(bars + 20);
    volatile int *gave_up = (volatile int *)(bars + 21);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const TileGrid &g = p.g;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const int iters = g.nseg * g.kblocks;

    if (tid == 0) {
        *gave_up = 0;
        for (int s = 0; s < ST; ++s) {
            mbar_init(smem_u32(bars + s), 1);
            mbar_init(smem_u32(bars + 8 + s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(bars + 16 + s), 1);
            mbar_init(smem_u32(bars + 18 + s), 4 * CG);   // one arrival per epilogue warp of the pair
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(L::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(L::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CG == 2) cluster_barrier();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        // ---------------- loads ----------------
        int s = 0, fills = 0;
        uint32_t phase = 1;   // of the free barriers: a fresh barrier passes a wait for the phase before its first
        bool ok = true;
        for (int t = first; ok && t < g.total; t += step) {
            const TileAt at = tile_at(g, t);
            const int za = g.za ? at.batch : 0, zb = g.zb ? at.batch : 0;
            const int arow = at.m * (128 * CG) + (int)rank * 128;
            for (int it = 0; it < iters; ++it) {
                if (*gave_up || !mbar_wait_bounded(smem_u32(bars + 8 + s), phase)) {
                    ok = false;
                    break;
                }
                const int seg = it / g.kblocks, k = (it - seg * g.kblocks) * G_KB;
                const uint32_t sa = smem_u32(sm + s * L::STAGE), sb = sa + L::ABYTES;
                uint32_t full = smem_u32(bars + s);
                if (rank == 0) mbar_expect_tx(full, CG * L::STAGE);
                if (CG == 2) full = map_to_rank(full, 0);
                if constexpr (A_MN) {
                    tma_tile<CG>(sa, &p.a[seg], full, arow, k, za);
                    tma_tile<CG>(sa + 8192, &p.a[seg], full, arow + 64, k, za);
                } else {
                    tma_tile<CG>(sa, &p.a[seg], full, k, arow, za);
                }
                if constexpr (Epi::kTwoMaps) {
                    const int brow = at.n * (BN / 2);
                    if constexpr (CG == 2) {
                        tma_tile<CG>(sb, &p.b[rank], full, k, brow, zb);
                    } else {
                        tma_tile<CG>(sb, &p.b[0], full, k, brow, zb);
                        tma_tile<CG>(sb + BN / 2 * 128, &p.b[1], full, k, brow, zb);
                    }
                } else if constexpr (B_MN) {
                    const int brow = at.n * BN + (int)rank * L::BROWS;
#pragma unroll
                    for (int i = 0; i < L::BROWS / 64; ++i)
                        tma_tile<CG>(sb + i * 8192, &p.b[seg], full, brow + i * 64, k, zb);
                } else {
                    tma_tile<CG>(sb, &p.b[seg], full, k, at.n * BN + (int)rank * L::BROWS, zb);
                }
                ++fills;
                if (++s == ST) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (!ok) {
            *gave_up = 1;
            // every stage's last fill has to land before the shared memory goes away
            if (rank == 0)
                for (int i = 0; i < ST && i < fills; ++i) {
                    const int n = (fills - 1 - i) / ST;   // which use of the ring stage i's last fill was
                    mbar_wait_bounded(smem_u32(bars + i), (uint32_t)(n & 1));
                }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---------------- products ----------------
        int s = 0, n = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first; ok && t < g.total; t += step, ++n) {
            const int buf = n & 1;
            if (*gave_up || !mbar_wait_bounded(smem_u32(bars + 18 + buf), (uint32_t)(((n >> 1) & 1) ^ 1))) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + buf * BN;
            for (int it = 0; it < iters; ++it) {
                if (!mbar_wait_bounded(smem_u32(bars + s), phase)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t sa = smem_u32(sm + s * L::STAGE);
                const uint64_t da = operand_desc<A_MN>(sa), db = operand_desc<B_MN>(sa + L::ABYTES);
#pragma unroll
                for (int k = 0; k < G_KB / 16; ++k)
                    mma_f16<CG>(d, da + k * k_step<A_MN>, db + k * k_step<B_MN>, g.idesc, it > 0 || k > 0 ? 1u : 0u);
                mma_commit<CG>(smem_u32(bars + 8 + s));
                if (++s == ST) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (ok) mma_commit<CG>(smem_u32(bars + 16 + buf));
        }
        if (!ok) *gave_up = 1;
    } else if (warp >= 2) {
        // ---------------- epilogue ----------------
        const int quarter = warp & 3;   // the TMEM lanes this warp may read
        const uint32_t freed = CG == 2 ? map_to_rank(smem_u32(bars + 18), 0) : smem_u32(bars + 18);
        int n = 0;
        for (int t = first; t < g.total; t += step, ++n) {
            const int buf = n & 1;
            if (!mbar_wait_bounded(smem_u32(bars + 16 + buf), (uint32_t)((n >> 1) & 1))) {
                *gave_up = 1;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const TileAt at = tile_at(g, t);
            const int row = at.m * (128 * CG) + (int)rank * 128 + quarter * 32 + lane;
            Epi::template store<BN>(p.epi, at, row, tmem + buf * BN + ((uint32_t)(quarter * 32) << 16));
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(freed + buf * 8);
                else mbar_arrive(freed + buf * 8);
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CG == 2) cluster_barrier();
    if (warp == 1) {
        if constexpr (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
    }
    if (tid == 0 && *gave_up) atomicExch(g.err, 1);
}

// 32 consecutive values of a row, columns [col, col + 32) of which those below `cols` exist; `wide`: the
// row starts on a 16-byte boundary.
template <class T>
__device__ __forceinline__ void store_row32(T *row, int col, int cols, bool wide, const float (&v)[32]) {
    if (wide && col + 32 <= cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Vec<T, 8> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = from_acc<T>(v[i * 8 + e]);
            store_vec<T, 8>(row + col + i * 8, o);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e)
            if (col + e < cols) row[col + e] = from_acc<T>(v[e]);
    }
}

// A plain product, rounded once: the batch index picks the output.
template <class T>
struct StoreEpi {
    struct Params {
        T *out[2];
        long ld[2];
        int M, N;
        bool wide;
    };
    static constexpr bool kTwoMaps = false;
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row, uint32_t tmem) {
        T *out = p.out[at.batch] + (long)row * p.ld[at.batch];
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            const int col = at.n * BN + c;
            if (col >= p.N) break;   // uniform over the warp
            float v[32];
            tmem_load32(tmem + c, v);
            if (row < p.M) store_row32(out, col, p.N, p.wide, v);
        }
    }
};

// ---- host side ----
enum { G_BF16 = 1, G_F16 = 0 };   // operand formats of the instruction descriptor

inline uint32_t gemm_idesc(int cg, int bn, bool a_mn, bool b_mn, int fmt) {
    return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(128 * cg >> 4) << 24);
}
// A batch of row-major matrices as TMA sees it; box: 64 contiguous elements x `box_rows` rows.
inline void gemm_map(CUtensorMap *map, const void *base, long cols, long rows, long batch, long ld, long batch_stride,
                     int box_rows, int fmt) {
    FITRE_REQUIRE(encode_fn(), FITRE_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(batch > 1 ? batch_stride : rows * ld) * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    FITRE_REQUIRE(encode(map, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                         fmt == G_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16),
                  FITRE_ERR_CUDA, "tensor map refused");
}
// What TMA can read in place.
inline bool tma_readable(const void *p, long ld) { return aligned16(p) && ld % 8 == 0; }

template <int CG, int BN, bool A_MN, bool B_MN, class Epi>
void gemm_launch(fitre_context *ctx, GemmArgs<typename Epi::Params> &args, int M, int N, int batch, bool triangle,
                 long K, int nseg, int fmt, const char *name) {
    using L = GemmLayout<CG, BN>;
    auto kernel = tile_gemm_kernel<CG, BN, A_MN, B_MN, Epi>;
    TileGrid &g = args.g;
    const int bn = Epi::kTwoMaps ? BN / 2 : BN;
    g.tilesM = (M + 128 * CG - 1) / (128 * CG);
    g.tilesN = (N + bn - 1) / bn;
    const long per = triangle ? (long)g.tilesM * (g.tilesM + 1) / 2 : (long)g.tilesM * g.tilesN;
    FITRE_REQUIRE(per * batch < (1l << 30), FITRE_ERR_TOO_LARGE, "too many tiles");
    g.per = (int)per;
    g.total = (int)per * batch;
    g.triangle = triangle;
    g.kblocks = (int)((K + G_KB - 1) / G_KB);
    g.nseg = nseg;
    g.idesc = gemm_idesc(CG, BN, A_MN, B_MN, fmt);
    g.err = (int *)(ctx->dscal + 4000);
    static thread_local int ready = -1;
    if (ready != ctx->device) {
        FITRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
        ready = ctx->device;
    }
    const int room = kLmSms / CG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((g.total < room ? g.total : room) * CG));
    cfg.blockDim = dim3(G_THREADS);
    cfg.dynamicSmemBytes = L::SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FITRE_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    check_launch(ctx, name);
}
// Box rows of the operands' maps.
template <int CG, int BN, bool A_MN> constexpr int a_box = A_MN ? 64 : 128;
template <int CG, int BN, bool B_MN, bool TWO> constexpr int b_box = B_MN ? 64 : TWO ? BN / 2 : BN / CG;

}  // namespace
}  // namespace fitre
