// Matrix-product engine of the language-model operators: 16-bit operands, fp32 accumulation on the
// 5th-generation tensor cores.
//   D[m, n] = sum over segments s, k  A_s[m, k] B_s[n, k]
// Either operand may be stored with k contiguous ("K-major") or with its row index contiguous
// ("MN-major": A' or B' in memory); both land in shared memory through tiled TMA in the 128-byte
// swizzle that the tensor core reads, and whatever lies outside a matrix arrives as zeros.
// The loop that issues the loads is the longest chain of the kernel: a 4-D map that cuts the contiguous
// dimension into runs of 64 fetches 128 rows x 128 k with one instruction per operand (against two to
// four smaller ones, 600 -> 552 us for 4096 x 4096 x 24576); blocks at a ragged edge take smaller boxes.
//
// Persistent kernel, warp-specialised:
//   warp 0     one lane issues the TMA loads of a ring of stages (128 k per stage)
//   warp 1     one lane issues tcgen05.mma; accumulators live in TMEM, two of them, so that
//   warps 2-5  read and store one tile (Epi) while the next is being computed.  Each warp gathers 32 rows x 64
//              columns in shared memory and sends them off as one TMA store: full cache lines, edges clipped.
// CG = 2 pairs two SMs on a 256 x BN tile: each CTA loads its 128 rows of A and half of B's rows, so a byte
// of B feeds twice the arithmetic; the even CTA's issuer drives both.  CG = 1 (128 x BN) is for products
// with too few tiles to occupy the pairs; where even those leave SMs idle, a cluster of 2 to 8 CTAs divides a tile's k
// among itself and each CTA adds up and stores a part of the tile, from the others' partial sums in its
// shared memory (1003 x 1000 x 5460: 39 -> 27 us against halving the tiles).  Every wait is bounded; when one runs out, the CTA sets the
// context's error word, lets its copies in flight land, frees its TMEM and returns.
#pragma once

#include "lm_common.cuh"
#include "tma_util.cuh"

namespace fitre {
namespace {

constexpr int G_THREADS = 192;
constexpr int G_KB = 128;   // k per stage: two swizzle rows of 128 bytes

// Which tiles there are and where their operands come from.
struct TileGrid {
    int tilesM, tilesN;   // tiles of one product
    int whole;            // tiles over all products of the batch that are computed whole; those beyond, so few
    int total;            // that they leave half of the last round idle, are computed as two halves each
    int per;              // tiles per product
    int triangle;         // 1: only tiles with column <= row (the product is symmetric)
    int kblocks, nseg;    // stages per segment, segments (map index = segment)
    int split;            // CTAs (a cluster) that share a tile's k; then there are no more tiles than clusters
    int za, zb;           // 1: the batch index is the operand map's third coordinate
    uint32_t idesc, idesc_half;
    int *err;
};

// An operand as the loads see it.  big: runs of 64 elements as a dimension of their own, box 64 x 128 x 2 runs,
// for blocks of 128 elements that end at or before `lim`; edge: box 64 x 128 rows (two loads per block).
struct alignas(64) Operand {
    CUtensorMap big, edge;
    int lim;
};
template <class P>
struct alignas(64) GemmArgs {
    Operand a[2], b[2];
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
__device__ __forceinline__ void tma_runs(uint32_t dst, const CUtensorMap *map, uint32_t bar, int y, int run, int w) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(run), "r"(w)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(y), "r"(run), "r"(w)
            : "memory");
}
// 128 rows x 128 k of an operand, 32 KB: its contiguous dimension is k, or (MN) its rows.
template <int CG, bool MN>
__device__ __forceinline__ void load_operand(uint32_t dst, const Operand &o, uint32_t bar, int row, int k, int z) {
    const int run = MN ? row : k, across = MN ? k : row;   // along and across the contiguous dimension
    if (run + 128 <= o.lim) {
        tma_runs<CG>(dst, &o.big, bar, across, run >> 6, z);
    } else {
        tma_tile<CG>(dst, &o.edge, bar, run, across, z);
        tma_tile<CG>(dst + 16384, &o.edge, bar, run + 64, across, z);
    }
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
// 64 consecutive accumulator columns of this thread's row.
__device__ __forceinline__ void tmem_load64(uint32_t addr, float (&v)[64]) {
    uint32_t r[64];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[h * 32]), "=r"(r[h * 32 + 1]), "=r"(r[h * 32 + 2]), "=r"(r[h * 32 + 3]), "=r"(r[h * 32 + 4]),
              "=r"(r[h * 32 + 5]), "=r"(r[h * 32 + 6]), "=r"(r[h * 32 + 7]), "=r"(r[h * 32 + 8]), "=r"(r[h * 32 + 9]),
              "=r"(r[h * 32 + 10]), "=r"(r[h * 32 + 11]), "=r"(r[h * 32 + 12]), "=r"(r[h * 32 + 13]),
              "=r"(r[h * 32 + 14]), "=r"(r[h * 32 + 15]), "=r"(r[h * 32 + 16]), "=r"(r[h * 32 + 17]),
              "=r"(r[h * 32 + 18]), "=r"(r[h * 32 + 19]), "=r"(r[h * 32 + 20]), "=r"(r[h * 32 + 21]),
              "=r"(r[h * 32 + 22]), "=r"(r[h * 32 + 23]), "=r"(r[h * 32 + 24]), "=r"(r[h * 32 + 25]),
              "=r"(r[h * 32 + 26]), "=r"(r[h * 32 + 27]), "=r"(r[h * 32 + 28]), "=r"(r[h * 32 + 29]),
              "=r"(r[h * 32 + 30]), "=r"(r[h * 32 + 31])
            : "r"(addr + h * 32)
            : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// Where a product's result goes: `map` for TMA stores (box 64 columns x 32 rows) where TMA can write it, else
// `out` directly.
template <class T> struct Output {
    CUtensorMap map;
    T *out;           // NULL: not wanted
    long ld, stride;  // elements between rows, between matrices of a batch
    int rows, cols;
    int tma;
    int passing;      // larger than L2 can keep: its lines are the first to go
};

__device__ __forceinline__ void st_shared16(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void ld_shared16(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
// Two values rounded to a pair of 16-bit elements, and back.
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

// An epilogue warp's two staging buffers of 32 rows x 128 bytes (64 elements), swizzled as TMA reads and writes
// them, and the barrier of its loads.  Shared-memory addresses; `lane` is the row a thread works on.
struct Stager {
    uint32_t base, bar;
    volatile int *gave_up;
    int lane, turn;
    uint32_t phase;
    bool loading;
    uint32_t partial;   // other CTAs' sums for this warp's part of the tile, `parts` blocks of `block` bytes: [columns][32 rows]
    int parts, block;
    // 64 accumulator columns of this thread's row, the first of them column `c` of the tile at `tmem`
    __device__ __forceinline__ void sums(uint32_t tmem, int c, float (&v)[64]) const {
        tmem_load64(tmem + c, v);
        for (int s = 0; s < parts; ++s)
#pragma unroll
            for (int e = 0; e < 64; ++e) {
                float o;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(o) : "r"(partial + s * block + (c + e) * 128 + lane * 4));
                v[e] += o;
            }
    }
    // The next of the two buffers, once its last store has read it.
    __device__ __forceinline__ uint32_t next() {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        __syncwarp();
        turn ^= 1;
        return base + turn * 4096;
    }
    __device__ __forceinline__ uint32_t slot(uint32_t buf, int i) const { return buf + lane * 128 + ((i ^ (lane & 7)) << 4); }
    __device__ __forceinline__ void send(const CUtensorMap *map, uint32_t buf, int x, int y, int z, bool passing) const {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            if (passing) {
                uint64_t policy;
                asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
                asm volatile(
                    "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%2, %3, %4}], [%1], %5;" ::"l"(map),
                    "r"(buf), "r"(x), "r"(y), "r"(z), "l"(policy)
                    : "memory");
            } else {
                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                             "r"(buf), "r"(x), "r"(y), "r"(z)
                             : "memory");
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
    __device__ __forceinline__ void drain() const {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    // Starts loading the same 32 x 64 block of up to two matrices into the two buffers, once both are free; `b` may be
    // NULL.  wait() before reading them.
    __device__ __forceinline__ void load(const CUtensorMap *a, const CUtensorMap *b, int x, int y, int z) {
        loading = true;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // this thread's reads of the buffers come first
        __syncwarp();
        if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            mbar_expect_tx(bar, b ? 8192 : 4096);
            tma_tile<1>(base, a, bar, x, y, z);
            if (b) tma_tile<1>(base + 4096, b, bar, x, y, z);
        }
    }
    __device__ __forceinline__ void wait() {
        if (!mbar_wait_bounded(bar, phase)) *gave_up = 1;
        phase ^= 1;
        loading = false;
    }
    // after a wait elsewhere ran out: a load that was started has to land before the kernel ends
    __device__ __forceinline__ void settle() {
        if (loading) wait();
    }
    // Stores 64 packed values of each lane's row: columns [col, col + 64), rows [row0, row0 + 32).
    template <class T>
    __device__ __forceinline__ void put(const Output<T> &o, int row0, int col, int batch, const uint32_t (&w)[32]) {
        const uint32_t buf = next();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t q[4] = {w[i * 4], w[i * 4 + 1], w[i * 4 + 2], w[i * 4 + 3]};
            st_shared16(slot(buf, i), q);
        }
        if (o.tma) {
            send(&o.map, buf, col, row0, batch, o.passing);
            return;
        }
        // an empty group keeps next()'s count of stores in step
        if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        __syncwarp();
        uint16_t *out = reinterpret_cast<uint16_t *>(o.out) + batch * o.stride;
        for (int r = 0; r < 32 && row0 + r < o.rows; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = h * 32 + lane;
                uint16_t v;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(buf + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2));
                if (col + c < o.cols) out[(long)(row0 + r) * o.ld + col + c] = v;
            }
        __syncwarp();
    }
    template <class T>
    __device__ __forceinline__ void put(const Output<T> &o, int row0, int col, int batch, const float (&v)[64]) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        put(o, row0, col, batch, w);
    }
};

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major: rows 128 bytes apart, groups of 8 rows
// 1024 bytes apart (64 k; the next 64 are a block of their own).  MN-major: blocks of 64 rows x 128 k (16384
// bytes, the leading offset), in each the 8-deep groups of k 1024 bytes apart.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(MN ? (16384 >> 4) : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// The descriptor's step to the i-th group of 16 k: 32 bytes along a swizzled row and, after 64 k, the next block; or
// two 8-deep groups.
template <bool MN> __device__ __forceinline__ uint32_t k_step(int i, int block_bytes) {
    return MN ? (uint32_t)(i * 2048) >> 4 : (uint32_t)((i >> 2) * block_bytes + (i & 3) * 32) >> 4;
}

struct TileAt { int batch, m, n, half; };   // half: -1 whole tile, 0 / 1 its left / right half
__device__ __forceinline__ TileAt tile_at(const TileGrid &g, int t) {
    TileAt r;
    r.half = -1;
    if (t >= g.whole) {
        r.half = (t - g.whole) & 1;
        t = g.whole + ((t - g.whole) >> 1);
    }
    r.batch = t / g.per;
    int i = t - r.batch * g.per;
    if (g.triangle) {
        int row = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
        while (row * (row + 1) / 2 > i) --row;
        while ((row + 1) * (row + 2) / 2 <= i) ++row;
        r.m = row;
        r.n = i - row * (row + 1) / 2;
    } else {
        // bands of 16 tile rows, column by column: the tiles in flight share operands in L2 (bands of 8 and 32 took
        // 1.01 and 1.05 times as long for 8192 x 24576 x 4096)
        const int band = i / (16 * g.tilesN), first = band * 16;
        const int high = min(16, g.tilesM - first);
        i -= band * 16 * g.tilesN;
        r.m = first + i % high;
        r.n = i / high;
    }
    return r;
}

template <int CG, int BN> struct GemmLayout {
    static constexpr int BROWS = BN / CG;                     // rows of B one CTA loads
    static_assert(BROWS == 128, "a stage holds 128 rows of either operand");
    static constexpr int ABYTES = 128 * G_KB * 2, BBYTES = BROWS * G_KB * 2;
    static constexpr int STAGE = ABYTES + BBYTES;
    static constexpr int STAGES = 3;
    static constexpr int STAGING = 4 * 2 * 4096;              // two buffers for each epilogue warp
    static constexpr int SMEM = STAGES * STAGE + STAGING + 1024 + 256;
    static constexpr int TMEM_COLS = 2 * BN;
};

// Epi: { using Params; static constexpr bool kTwoMaps (B's rows come half from map 0, half from map 1);
//        static void store<BN>(const Params &, TileAt, int row0, uint32_t tmem, Stager &) } -- called by the four
// epilogue warps once the tile is computed, and begin<BN> before (to start loads), `row0` = row of the matrix of the warp's first accumulator row, `tmem` = address of its first column.
template <int CG, int BN, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(G_THREADS, 1)
tile_gemm_kernel(const __grid_constant__ GemmArgs<typename Epi::Params> p) {
    using L = GemmLayout<CG, BN>;
    constexpr int ST = L::STAGES;
    extern __shared__ unsigned char smraw[];
    unsigned char *sm = (unsigned char *)(((uintptr_t)smraw + 1023) & ~(uintptr_t)1023);
    unsigned long long *bars = (unsigned long long *)(sm + ST * L::STAGE + L::STAGING);
    // [0, 8) stage full, [8, 16) stage free, [16, 18) accumulator full, [18, 20) accumulator free, [22, 26) epilogue loads
    uint32_t *tmem_slot = (uint32_t *)(bars + 20);
    volatile int *gave_up = (volatile int *)(bars + 21);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const TileGrid &g = p.g;
    const int split = CG == 1 ? g.split : 1, part = split > 1 ? (int)cluster_rank() : 0;
    const int first = blockIdx.x / (CG * split), step = gridDim.x / (CG * split);
    const int all = g.nseg * g.kblocks, it0 = all * part / split, iters = all * (part + 1) / split - it0;

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
        for (int s = 0; s < 4; ++s) mbar_init(smem_u32(bars + 22 + s), 1);
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
    // everything above needs nothing of the kernel before this one in the stream
    wait_for_previous_kernel();
    let_next_kernel_start();

    if (warp == 0 && lane == 0) {
        // ---------------- loads ----------------
        int s = 0, fills = 0;
        uint32_t phase = 1;   // of the free barriers: a fresh barrier passes a wait for the phase before its first
        bool ok = true;
        const uint32_t full0 = smem_u32(bars), free0 = smem_u32(bars + 8), data0 = smem_u32(sm);
        const uint32_t land0 = CG == 2 ? map_to_rank(full0, 0) : full0;   // both CTAs' loads count on the even one's
        const int kblocks = g.kblocks;
        for (int t = first; ok && t < g.total; t += step) {
            const TileAt at = tile_at(g, t);
            const int za = g.za ? at.batch : 0, zb = g.zb ? at.batch : 0;
            const int arow = at.m * (128 * CG) + (int)rank * 128;
            // a half tile uses the first half of the rows of B that each CTA loads
            const int shift = at.half > 0 ? 1 : 0, rows = at.half < 0 ? L::BROWS : L::BROWS / 2;
            const int brow = Epi::kTwoMaps ? at.n * (BN / 2) + shift * (BN / 4)
                                           : at.n * BN + shift * (BN / 2) + (int)rank * rows;
            int seg = it0 / kblocks, kb = it0 - seg * kblocks, left = iters;
            for (; ok && left > 0; ++seg, kb = 0) {
                const Operand &oa = p.a[seg], &ob = p.b[Epi::kTwoMaps ? (int)rank : seg];
                for (int k = kb * G_KB; kb < kblocks && left > 0; ++kb, --left, k += G_KB) {
                    if (!mbar_wait_bounded(free0 + s * 8, phase)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = data0 + s * L::STAGE, sb = sa + L::ABYTES, full = land0 + s * 8;
                    if (rank == 0) mbar_expect_tx(full0 + s * 8, CG * L::STAGE);
                    load_operand<CG, A_MN>(sa, oa, full, arow, k, za);
                    if constexpr (Epi::kTwoMaps && CG == 1) {
                        // gate and up rows side by side in each half of k
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            tma_tile<CG>(sb + h * 16384, &p.b[0].edge, full, k + h * 64, brow, zb);
                            tma_tile<CG>(sb + h * 16384 + 8192, &p.b[1].edge, full, k + h * 64, brow, zb);
                        }
                    } else {
                        load_operand<CG, B_MN>(sb, ob, full, brow, k, zb);
                    }
                    ++fills;
                    if (++s == ST) {
                        s = 0;
                        phase ^= 1;
                    }
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
            if (!mbar_wait_bounded(smem_u32(bars + 18 + buf), (uint32_t)(((n >> 1) & 1) ^ 1))) {
                ok = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + buf * BN, idesc = t >= g.whole ? g.idesc_half : g.idesc;
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
                    mma_f16<CG>(d, da + k_step<A_MN>(k, 128 * 128), db + k_step<B_MN>(k, L::BROWS * 128), idesc,
                                it > 0 || k > 0 ? 1u : 0u);
                mma_commit<CG>(smem_u32(bars + 8 + s));
                if (++s == ST) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (ok) mma_commit<CG>(smem_u32(bars + 16 + buf));
        }
        if (!ok) *gave_up = 1;
    }
    const int quarter = warp & 3;   // the TMEM lanes an epilogue warp may read
    Stager stager{smem_u32(sm + ST * L::STAGE) + quarter * 8192, smem_u32(bars + 22 + quarter), gave_up, lane, 0, 0, false, 0, 0, 0};
    if (warp >= 2 && split == 1) {
        // ---------------- epilogue ----------------
        const uint32_t freed = CG == 2 ? map_to_rank(smem_u32(bars + 18), 0) : smem_u32(bars + 18);
        int n = 0;
        for (int t = first; t < g.total; t += step, ++n) {
            const int buf = n & 1;
            const TileAt at = tile_at(g, t);
            const int row0 = at.m * (128 * CG) + (int)rank * 128 + quarter * 32;
            Epi::template begin<BN>(p.epi, at, row0, stager);
            if (!mbar_wait_bounded(smem_u32(bars + 16 + buf), (uint32_t)((n >> 1) & 1))) {
                *gave_up = 1;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            Epi::template store<BN>(p.epi, at, row0, tmem + buf * BN + ((uint32_t)(quarter * 32) << 16), stager);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(freed + buf * 8);
                else mbar_arrive(freed + buf * 8);
            }
        }
    } else if (split > 1) {
        // ---------------- one tile, its k divided among the cluster ----------------
        bool done = true;
        if (warp >= 2) done = mbar_wait_bounded(smem_u32(bars + 16), 0);
        if (!done) *gave_up = 1;
        __syncwarp();
        cluster_barrier();   // every CTA's stages are free
        // The tile in parts of 32 rows x `span` columns (all of them, or half for 8 CTAs); owner of part (quarter, h): who
        // adds it up.  A CTA's parts lie one behind the other in its shared memory, in each the others' sums in turn.
        const int halves = split == 8 ? 2 : 1, span = BN / halves, block = span * 128;
        const int per = 4 * halves / split;   // parts per CTA
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
        if (warp >= 2) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < BN; c += 64) {
                const int piece = quarter * halves + c / span, owner = piece / per;
                if (owner == part) continue;
                const uint32_t room = smem_u32(sm) + ((piece % per) * (split - 1) + (part < owner ? part : part - 1)) * block;
                const uint32_t to = map_to_rank(room, owner) + lane * 4 + (c % span) * 128;
                float v[64];
                tmem_load64(mine + c, v);
#pragma unroll
                for (int e = 0; e < 64; ++e)
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + e * 128), "f"(v[e]) : "memory");
            }
        }
        __syncwarp();
        cluster_barrier();   // the partial sums have arrived
        if (warp >= 2) {
            TileAt at = tile_at(g, first);
            const int row0 = at.m * 128 + quarter * 32;
            for (int h = 0; h < halves; ++h) {
                const int piece = quarter * halves + h;
                if (piece / per != part) continue;
                if (halves == 2) at.half = h;
                stager.partial = smem_u32(sm) + (piece % per) * (split - 1) * block;
                stager.parts = split - 1;
                stager.block = block;
                Epi::template begin<BN>(p.epi, at, row0, stager);
                Epi::template store<BN>(p.epi, at, row0, mine + h * span, stager);
            }
        }
    }
    if (warp >= 2) {
        stager.drain();
        stager.settle();
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

// A plain product, rounded once: the batch index picks the output.
template <class T>
struct StoreEpi {
    struct Params {
        Output<T> out[2];
    };
    static constexpr bool kTwoMaps = false;
    template <int BN> static __device__ __forceinline__ void begin(const Params &, TileAt, int, Stager &) {}
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row0, uint32_t tmem, Stager &st) {
        const Output<T> &o = p.out[at.batch];
        const int first = at.n * BN + (at.half > 0 ? BN / 2 : 0), width = at.half < 0 ? BN : BN / 2;
        if (row0 >= o.rows) return;
#pragma unroll 1
        for (int c = 0; c < width && first + c < o.cols; c += 64) {
            float v[64];
            st.sums(tmem, c, v);
            st.put(o, row0, first + c, 0, v);
        }
    }
};

// ---- host side ----
enum { G_BF16 = 1, G_F16 = 0 };   // operand formats of the instruction descriptor

inline uint32_t gemm_idesc(int cg, int bn, bool a_mn, bool b_mn, int fmt) {
    return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(128 * cg >> 4) << 24);
}
// A batch of row-major matrices as TMA sees it; box: 64 contiguous elements x `box_rows` rows.  TMA works in units of
// 16 bytes (a store that ends inside one writes all of it), so `cols` is a multiple of 8: scratch matrices are
// padded to one, with zeros, and are given with their padding.
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
// An operand of `rows` x `k`: a batch of matrices, row-major with the k contiguous, or (mn) stored with the rows
// contiguous.  edge_rows: rows of the smaller box.
inline void gemm_operand(Operand *o, bool mn, const void *base, long rows, long k, long batch, long ld, long batch_stride,
                         int fmt, int edge_rows = 128) {
    const long along = mn ? rows : k, across = mn ? k : rows;
    gemm_map(&o->edge, base, along, across, batch, ld, batch_stride, edge_rows, fmt);
    o->lim = (int)(along / 64 * 64);
    if (o->lim < 128) {
        o->lim = 0;
        return;
    }
    cuuint64_t dims[4] = {64, (cuuint64_t)across, (cuuint64_t)(along / 64), (cuuint64_t)batch};
    cuuint64_t strides[3] = {(cuuint64_t)ld * 2, 128, (cuuint64_t)(batch > 1 ? batch_stride : across * ld) * 2};
    cuuint32_t box[4] = {64, 128, 2, 1};
    FITRE_REQUIRE(encode(&o->big, base, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                         fmt == G_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16),
                  FITRE_ERR_CUDA, "tensor map refused");
}
// What TMA can read in place.
inline bool tma_readable(const void *p, long ld) { return aligned16(p) && ld % 8 == 0; }
// An output and, where TMA can write it, its map.
template <class T>
Output<T> gemm_output(void *out, long cols, long rows, long batch, long ld, long stride, int fmt) {
    Output<T> o = {};
    o.out = (T *)out;
    if (!out) return o;
    o.ld = ld, o.stride = stride, o.rows = (int)rows, o.cols = (int)cols;
    o.tma = cols % 8 == 0 && tma_readable(out, ld) && (batch == 1 || stride % 8 == 0);
    o.passing = rows * cols * batch * (long)sizeof(T) > 64l << 20;   // half of L2
    if (o.tma) gemm_map(&o.map, out, cols, rows, batch, ld, stride, 32, fmt);
    return o;
}

// `dependent`: the kernel before it in the stream is this library's and lets this one start its set-up early.
template <int CG, int BN, bool A_MN, bool B_MN, class Epi>
void gemm_launch(fitre_context *ctx, GemmArgs<typename Epi::Params> &args, int M, int N, int batch, bool triangle,
                 long K, int nseg, int fmt, const char *name, bool dependent) {
    using L = GemmLayout<CG, BN>;
    auto kernel = tile_gemm_kernel<CG, BN, A_MN, B_MN, Epi>;
    TileGrid &g = args.g;
    const int bn = Epi::kTwoMaps ? BN / 2 : BN;
    g.tilesM = (M + 128 * CG - 1) / (128 * CG);
    g.tilesN = (N + bn - 1) / bn;
    const long per = triangle ? (long)g.tilesM * (g.tilesM + 1) / 2 : (long)g.tilesM * g.tilesN;
    FITRE_REQUIRE(per * batch < (1l << 30), FITRE_ERR_TOO_LARGE, "too many tiles");
    g.per = (int)per;
    const int room = kLmSms / CG, tiles = (int)per * batch, left = tiles % room;
    // (64 columns are the least an epilogue stores at a time; two maps on one SM load no half tiles)
    g.whole = left > 0 && left <= room / 2 && !(Epi::kTwoMaps && CG == 1) ? tiles - left : tiles;
    // Dividing k by S costs an exchange worth about 5 + S / 2 stages of 0.5 us: for long sums only (five steps of a
    // 1024 x 1024 update, 8 stages a product: 148 us in halves, 196 us divided by 2; 1003 x 1000 x 5460, 44 stages: 39
    // us in halves, 27 us divided by 2).
    const int stages = (int)((K + G_KB - 1) / G_KB) * nseg;
    g.split = 1;
    if (CG == 1) {
        int best = stages;
        for (int s : {2, 4, 8}) {
            const int cost = (stages + s - 1) / s + 5 + s / 2;
            // eight CTAs share a tile by its column halves, which two maps on one SM do not have
            if (tiles * s <= kLmSms && cost < best && !(s == 8 && Epi::kTwoMaps)) best = cost, g.split = s;
        }
        if (g.split > 1) g.whole = tiles;
    }
    g.total = g.whole + 2 * (tiles - g.whole);
    g.triangle = triangle;
    g.kblocks = (int)((K + G_KB - 1) / G_KB);
    g.nseg = nseg;
    g.idesc = gemm_idesc(CG, BN, A_MN, B_MN, fmt);
    g.idesc_half = gemm_idesc(CG, BN / 2, A_MN, B_MN, fmt);
    g.err = (int *)(ctx->dscal + 4000);
    static thread_local int ready = -1;
    if (ready != ctx->device) {
        FITRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
        ready = ctx->device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((g.total < room ? g.total : room) * CG * g.split));
    cfg.blockDim = dim3(G_THREADS);
    cfg.dynamicSmemBytes = L::SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)(CG * g.split);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 2 : 1;
    FITRE_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    check_launch(ctx, name);
}
}  // namespace
}  // namespace fitre
