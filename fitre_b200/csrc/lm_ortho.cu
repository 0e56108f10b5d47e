// Orthogonalised update of a weight matrix by Newton-Schulz products:
//   X = G / (|G|_F + eps);  `steps` times:  A = X X',  B = b A + c A A,  X <- a X + B X
// (from the side of the smaller dimension; X' X and X B where G has more rows than columns), which
// drives all singular values towards 1.  Bound by the tensor cores.
// A and A A are symmetric: only tiles on and below the diagonal are computed and stored twice, which
// saves half of two of the three products.
// The tensor core reads the iterates in fp16, scaled by 2^10: every value is bounded (singular values stay
// below 1.3 with the default coefficients, |B| below 4), so fp16's 11 bits serve all of it with
// headroom of 2^4 above and normal numbers down to 2^-24.  Two parts of the sum a X + B X are kept
// wider, because what is rounded away there comes back amplified:
//   * X is held as an fp16 pair hi + lo.  Rounding X alone would put noise into directions that the
//     update does not have (a gradient of low rank), and each step multiplies them by a, 500-fold over five
//     steps: an error of 3 to 8 % for low-rank updates against 0.1 % with the pair.
//   * B's diagonal is held in fp32 and applied in the epilogue; near singular value 1 it is -2.7 and
//     nearly cancels a, while the off-diagonal part is small.
// Measured on a B200: five steps of 4096 x 8192 bf16 2.18 ms (1.1 PFLOP/s of the halved work, under the power cap), of
// 4 x 513 x 384 fp32 121 us (17 dependent kernels).
// Products accumulate in fp32; the result is rounded to bf16 once, and is within about half a bf16
// rounding of the exact polynomial before that.
#include <cfloat>

#include "lm_gemm.cuh"
#include "lm_simd.cuh"

namespace fitre {
namespace {

constexpr float kScale = 1024.0f;   // 2^10: what the stored iterates are multiplied by

// Sum over the block's 256 threads, in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double q, double *s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = q;
    __syncthreads();
    q = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) q += s[w];
    return q;
}

// Threads of a block that share a row of `chunks` vectors: a power of two from 8 to 256, as its logarithm.
inline int row_share(long chunks) {
    int s = 3;
    while (s < 8 && (1 << s) < chunks) ++s;
    return s;
}
// Sums of squares of each matrix's parts, in fp64 (squares of fp32 values overflow fp32): the blocks of a matrix take
// 256 >> share rows at a time in turn.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
ortho_norm_kernel(const T *in, long ld, long bstride, int rows, int cols, int share, double *partial) {
    let_next_kernel_start();
    __shared__ double s[8];
    const T *m = in + blockIdx.y * bstride;
    const int t = threadIdx.x & ((1 << share) - 1), at = threadIdx.x >> share, step = 256 >> share;
    double q = 0;
    for (int r = blockIdx.x * step + at; r < rows; r += gridDim.x * step)
#pragma unroll 4
        for (int c = t * VEC; c < cols; c += VEC << share) {
            const Vec<T, VEC> x = load_vec<T, VEC>(m + r * ld + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const double v = (double)to_acc<acc_t<T>>(x.v[e]);
                q += v * v;
            }
        }
    q = block_sum(q, s);
    if (threadIdx.x == 0) partial[(long)blockIdx.y * gridDim.x + blockIdx.x] = q;
}

// The first iterate, as a pair of fp16 matrices; zeros in the padding of their rows.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
ortho_scale_kernel(const T *in, long ld, long bstride, int rows, int cols, int share, const double *__restrict__ partial,
                   int parts, double eps, __half *hi, __half *lo, long ldo, long ostride) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ double s[8];
    double q = 0;
    for (int i = threadIdx.x; i < parts; i += 256) q += partial[(long)blockIdx.y * parts + i];
    q = block_sum(q, s);
    // squares that leave fp64's range (elements beyond 1e154): no number rather than zeros
    const double f = q <= DBL_MAX ? (double)kScale / (sqrt(q) + eps) : nan("");
    const T *m = in + blockIdx.y * bstride;
    hi += blockIdx.y * ostride;
    lo += blockIdx.y * ostride;
    const int t = threadIdx.x & ((1 << share) - 1), at = threadIdx.x >> share, step = 256 >> share;
    for (int r = blockIdx.x * step + at; r < rows; r += gridDim.x * step) {
#pragma unroll 2
        for (int c = t * VEC; c < cols; c += VEC << share) {
            const Vec<T, VEC> x = load_vec<T, VEC>(m + r * ld + c);
            Vec<__half, VEC> h, l;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float v = (float)((double)to_acc<acc_t<T>>(x.v[e]) * f);
                h.v[e] = __float2half_rn(v);
                l.v[e] = __float2half_rn(v - __half2float(h.v[e]));
            }
            store_vec<__half, VEC>(hi + r * ldo + c, h);
            store_vec<__half, VEC>(lo + r * ldo + c, l);
        }
        if (cols + t < ldo) hi[r * ldo + cols + t] = lo[r * ldo + cols + t] = __float2half_rn(0.0f);   // fewer than 8
    }
}

// A symmetric product: tile and, off the diagonal, its mirror image.  out = kacc * acc + kin * in; with
// `diag`, the diagonal goes there (unscaled, fp32) and zeros take its place.
struct SymmetricEpi {
    struct Params {
        Output<__half> out;
        CUtensorMap mirror;   // the same matrix, box 32 columns x 64 rows, no swizzle
        CUtensorMap in;       // as out's map
        float *diag;
        float kacc, kin;
        int with_in;
    };
    static constexpr bool kTwoMaps = false;
    template <int BN> static __device__ __forceinline__ void begin(const Params &p, TileAt at, int row0, Stager &st) {
        const int first = at.n * BN + (at.half > 0 ? BN / 2 : 0);
        if (p.with_in && row0 < p.out.rows && first < p.out.rows) st.load(&p.in, nullptr, first, row0, at.batch);
    }
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row0, uint32_t tmem, Stager &st) {
        const int row = row0 + st.lane, n = p.out.rows;
        const int first = at.n * BN + (at.half > 0 ? BN / 2 : 0), width = at.half < 0 ? BN : BN / 2;
        if (row0 >= n) return;
        using P = Simd<float, 2>;
        const P kacc = P::splat(p.kacc), kin = P::splat(p.kin);
#pragma unroll 1
        for (int c = 0; c < width && first + c < n; c += 64) {
            const int col = first + c;
            if (p.with_in && c > 0) st.load(&p.in, nullptr, col, row0, at.batch);
            float acc[64];
            st.sums(tmem, c, acc);
            if (p.with_in) st.wait();
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t q[4] = {0, 0, 0, 0};
                if (p.with_in) ld_shared16(st.slot(st.base, i), q);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = i * 8 + j * 2;
                    const float2 f = unpack_half2(q[j]);
                    const P v = fma(P::of(acc[e], acc[e + 1]), kacc, mul(P::of(f.x, f.y), kin));
                    float x, y;
                    v.split(x, y);
                    w[i * 4 + j] = pack2<__half>(x, y);
                    acc[e] = x;
                    acc[e + 1] = y;
                }
            }
            if (p.diag && row0 < col + 64 && row0 + 32 > col) {   // the diagonal runs through this block
                const int on = row - col;                         // this row's element, if 0..63
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < 64; ++e) d = on == e ? acc[e] : d;
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    w[e] &= on >> 1 == e ? (on & 1 ? 0x0000ffffu : 0xffff0000u) : 0xffffffffu;
                if (row < n && on >= 0 && on < 64) p.diag[(long)at.batch * n + row] = d * (1 / kScale);
            }
            __syncwarp();
            st.put(p.out, row0, col, at.batch, w);
            if (at.m != at.n) {
                // transposed in shared memory: 64 rows (these columns) of 32 (these rows)
                const uint32_t buf = st.next() + st.lane * 2;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(buf + e * 128), "h"((uint16_t)w[e]) : "memory");
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(buf + e * 128 + 64), "h"((uint16_t)(w[e] >> 16)) : "memory");
                }
                st.send(&p.mirror, buf - st.lane * 2, row0, col, at.batch, p.out.passing);
            }
        }
    }
};

// X <- a X + B X:  v = kacc * acc + kout * ((a + d) hi + (a or a + d) lo), acc = (B without its diagonal d) hi.
// The low part takes a alone, which is what acts on directions outside the update, but for the last
// step, where no further step amplifies them and a + d is closer for all others.
// T = __half: v becomes the next pair (lo in place: each warp reads its part before it stores it); else v is the result.
template <class T>
struct IterateEpi {
    struct Params {
        Output<T> out;
        Output<__half> lo;
        CUtensorMap hi;
        const float *diag;
        int cols, small;
        float kacc, kout, a;
        int tall;
    };
    static constexpr bool kTwoMaps = false;
    template <int BN> static __device__ __forceinline__ void begin(const Params &p, TileAt at, int row0, Stager &st) {
        const int first = at.n * BN + (at.half > 0 ? BN / 2 : 0);
        if (row0 < p.out.rows && first < p.out.cols) st.load(&p.hi, &p.lo.map, first, row0, at.batch);
    }
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row0, uint32_t tmem, Stager &st) {
        using P = Simd<float, 2>;
        constexpr bool kLast = !std::is_same<T, __half>::value;
        const int row = row0 + st.lane;
        const int first = at.n * BN + (at.half > 0 ? BN / 2 : 0), width = at.half < 0 ? BN : BN / 2;
        if (row0 >= p.out.rows) return;
        const float *diag = p.diag + (long)at.batch * p.small;
        const float drow = !p.tall && row < p.out.rows ? diag[row] : 0.0f;
        // tall: the diagonal runs along the columns; each lane holds two of the block's 64 and passes them round
        auto along = [&](int col) { return p.tall && col + st.lane < p.cols ? diag[col + st.lane] : 0.0f; };
        float d0 = along(first), d1 = along(first + 32);
        const P kacc = P::splat(p.kacc), kout = P::splat(p.kout), a = P::splat(p.a), minus = P::splat(-1.0f);
#pragma unroll 1
        for (int c = 0; c < width && first + c < p.out.cols; c += 64) {
            const int col = first + c;
            float acc[64];
            st.sums(tmem, c, acc);
            st.wait();
            uint32_t w[32], r[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t h[4], l[4];
                ld_shared16(st.slot(st.base, i), h);
                ld_shared16(st.slot(st.base + 4096, i), l);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = i * 8 + j * 2;
                    const float2 fh = unpack_half2(h[j]), fl = unpack_half2(l[j]);
                    P ad = P::splat(p.a + drow);
                    if (p.tall) {
                        const float d = e < 32 ? d0 : d1;
                        ad = add(a, P::of(__shfl_sync(0xffffffffu, d, e & 31), __shfl_sync(0xffffffffu, d, (e + 1) & 31)));
                    }
                    P x = fma(P::of(fl.x, fl.y), kLast ? ad : a, mul(P::of(fh.x, fh.y), ad));
                    x = fma(P::of(acc[e], acc[e + 1]), kacc, mul(x, kout));
                    float x0, x1;
                    x.split(x0, x1);
                    w[i * 4 + j] = pack2<T>(x0, x1);
                    if (!kLast) {
                        const float2 f = unpack_half2(w[i * 4 + j]);
                        fma(P::of(f.x, f.y), minus, x).split(x0, x1);
                        r[i * 4 + j] = pack2<__half>(x0, x1);
                    }
                }
            }
            d0 = along(col + 64);
            d1 = along(col + 96);
            __syncwarp();
            st.put(p.out, row0, col, at.batch, w);
            if constexpr (!kLast) st.put(p.lo, row0, col, at.batch, r);
            if (c + 64 < width && col + 64 < p.out.cols) st.load(&p.hi, &p.lo.map, col + 64, row0, at.batch);
        }
    }
};

long up8(long n) { return (n + 7) / 8 * 8; }
long up128(long bytes) { return (bytes + 127) / 128 * 128; }

struct Plan {
    int rows, cols, small;   // small: the order of A and B
    int parts;               // blocks that sum one matrix's squares
    int batch;
    bool tall;
    long ldx, xs, lda, as;
    __half *x[2], *lo, *A, *B;
    float *diag;
    double *partial;
    Plan(const OrthoArgs &a) {
        rows = (int)a.rows, cols = (int)a.cols, batch = (int)a.batch;
        tall = rows > cols;
        small = tall ? cols : rows;
        ldx = up8(cols), xs = up128(2 * ldx * rows) / 2;
        lda = up8(small), as = up128(2 * lda * small) / 2;
        parts = 8 * kLmSms / batch < rows ? 8 * kLmSms / batch : rows;
        parts = parts > 0 ? parts : 1;
        char *p = (char *)a.scratch;
        auto take = [&](long bytes) {
            char *q = p;
            p += up128(bytes);
            return q;
        };
        x[0] = (__half *)take(2 * xs * batch);
        x[1] = (__half *)take(2 * xs * batch);
        lo = (__half *)take(2 * xs * batch);
        A = (__half *)take(2 * as * batch);
        B = (__half *)take(2 * as * batch);
        diag = (float *)take(4 * (long)small * batch);
        partial = (double *)take(8 * (long)parts * batch);
        bytes = p - (char *)a.scratch;
    }
    long bytes;
};

void mirror_map(CUtensorMap *map, const __half *base, long n, long batch, long ld, long stride) {
    cuuint64_t dims[3] = {(cuuint64_t)ld, (cuuint64_t)n, (cuuint64_t)batch};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(batch > 1 ? stride : n * ld) * 2};
    cuuint32_t box[3] = {32, 64, 1};
    FITRE_REQUIRE(encode(map, base, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_DATA_TYPE_FLOAT16),
                  FITRE_ERR_CUDA, "tensor map refused");
}

template <int CG, int BN, bool MN>
void symmetric(fitre_context *ctx, const Plan &pl, const __half *x, long K, long rows, long ld, long stride,
               __half *out, const __half *in, float *diag, float kacc, float kin) {
    // MN: the matrix's columns are the product's index
    GemmArgs<SymmetricEpi::Params> g = {};
    gemm_operand(&g.a[0], MN, x, MN ? ld : rows, MN ? rows : ld, pl.batch, ld, stride, G_F16);
    g.b[0] = g.a[0];
    g.g.za = g.g.zb = 1;
    g.epi.out = gemm_output<__half>(out, pl.lda, pl.small, pl.batch, pl.lda, pl.as, G_F16);
    mirror_map(&g.epi.mirror, out, pl.small, pl.batch, pl.lda, pl.as);
    if (in) gemm_map(&g.epi.in, in, pl.lda, pl.small, pl.batch, pl.lda, pl.as, 32, G_F16);
    g.epi.with_in = in != nullptr, g.epi.diag = diag, g.epi.kacc = kacc, g.epi.kin = kin;
    gemm_launch<CG, BN, MN, MN, SymmetricEpi>(ctx, g, pl.small, pl.small, pl.batch, true, K, 1, G_F16,
                                              "ortho_symmetric_kernel", true);
}

template <int CG, int BN, class T>
void iterate(fitre_context *ctx, const Plan &pl, const __half *x, T *out, long ldo, long ostride, float kacc, float kout, float a) {
    GemmArgs<typename IterateEpi<T>::Params> g = {};
    g.g.za = g.g.zb = 1;
    constexpr int fmt = std::is_same<T, __half>::value ? G_F16 : G_BF16;
    g.epi.out = gemm_output<T>(out, fmt == G_F16 ? pl.ldx : pl.cols, pl.rows, pl.batch, ldo, ostride, fmt);
    g.epi.cols = pl.cols;
    g.epi.lo = gemm_output<__half>(pl.lo, pl.ldx, pl.rows, pl.batch, pl.ldx, pl.xs, G_F16);
    gemm_map(&g.epi.hi, x, pl.ldx, pl.rows, pl.batch, pl.ldx, pl.xs, 32, G_F16);
    g.epi.diag = pl.diag, g.epi.small = pl.small, g.epi.kacc = kacc, g.epi.kout = kout, g.epi.a = a, g.epi.tall = pl.tall;
    if (pl.tall) {   // X B: B is symmetric, its rows serve as its columns
        gemm_operand(&g.a[0], false, x, pl.rows, pl.ldx, pl.batch, pl.ldx, pl.xs, G_F16);
        gemm_operand(&g.b[0], false, pl.B, pl.small, pl.lda, pl.batch, pl.lda, pl.as, G_F16);
        gemm_launch<CG, BN, false, false, IterateEpi<T>>(ctx, g, pl.rows, pl.cols, pl.batch, false, pl.small, 1, G_F16,
                                                         "ortho_iterate_kernel", true);
    } else {
        gemm_operand(&g.a[0], false, pl.B, pl.small, pl.lda, pl.batch, pl.lda, pl.as, G_F16);
        gemm_operand(&g.b[0], true, x, pl.ldx, pl.rows, pl.batch, pl.ldx, pl.xs, G_F16);
        gemm_launch<CG, BN, false, true, IterateEpi<T>>(ctx, g, pl.rows, pl.cols, pl.batch, false, pl.small, 1, G_F16,
                                                        "ortho_iterate_kernel", true);
    }
}

template <class T, int VEC>
void start_as(fitre_context *ctx, const OrthoArgs &a, const Plan &pl) {
    const dim3 grid(pl.parts, pl.batch);
    const int share = row_share((pl.cols + VEC - 1) / VEC);
    ortho_norm_kernel<T, VEC><<<grid, 256, 0, ctx->stream>>>((const T *)a.in, a.ldi, a.istride, pl.rows, pl.cols,
                                                             share, pl.partial);
    check_launch(ctx, "ortho_norm_kernel");
    launch_after(ctx->stream, ortho_scale_kernel<T, VEC>, grid, 256, (const T *)a.in, a.ldi, a.istride, pl.rows, pl.cols,
                 share, pl.partial, pl.parts, a.eps, pl.x[0], pl.lo, pl.ldx, pl.xs);
    check_launch(ctx, "ortho_scale_kernel");
}
template <class T>
void start(fitre_context *ctx, const OrthoArgs &a, const Plan &pl) {
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = aligned16(a.in) && pl.cols % VEC == 0 && (a.ldi * (long)sizeof(T)) % 16 == 0 &&
                      (a.istride * (long)sizeof(T)) % 16 == 0;
    wide ? start_as<T, VEC>(ctx, a, pl) : start_as<T, 1>(ctx, a, pl);
}

}  // namespace

long ortho_scratch(long batch, long rows, long cols) {
    OrthoArgs a = {};
    a.batch = batch, a.rows = rows, a.cols = cols;
    return Plan(a).bytes;
}

void orthogonalize(fitre_context *ctx, const OrthoArgs &a) {
    const Plan pl(a);
    switch (a.dtype) {
        case FITRE_DTYPE_F64: start<double>(ctx, a, pl); break;
        case FITRE_DTYPE_F32: start<float>(ctx, a, pl); break;
        case FITRE_DTYPE_BF16: start<__nv_bfloat16>(ctx, a, pl); break;
        default: start<__half>(ctx, a, pl); break;
    }
    // SM pairs where they have tiles enough and sums long enough to outlast the epilogues, which read and write four
    // fp16 matrices here (4 x 2748 x 336: 230 us in pairs, 205 us on single SMs; 4096 x 1024: 294 and 288 us)
    const bool lasting = pl.small > 1024;
    const long side = (pl.small + 255) / 256;
    const bool big = lasting && side * (side + 1) / 2 * pl.batch >= kLmSms / 2 - 16;
    const bool bigx = lasting && (long)((pl.rows + 255) / 256) * ((pl.cols + 255) / 256) * pl.batch >= kLmSms / 2 - 16;
    const long K = pl.tall ? pl.rows : pl.cols;
    for (int s = 0; s < a.steps; ++s) {
        const float ca = (float)a.coef[0], cb = (float)a.coef[1], cc = (float)a.coef[2];
        const __half *x = pl.x[s & 1];
        if (pl.tall) {
            big ? symmetric<2, 256, true>(ctx, pl, x, K, pl.rows, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0)
                : symmetric<1, 128, true>(ctx, pl, x, K, pl.rows, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0);
        } else {
            big ? symmetric<2, 256, false>(ctx, pl, x, K, pl.rows, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0)
                : symmetric<1, 128, false>(ctx, pl, x, K, pl.rows, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0);
        }
        big ? symmetric<2, 256, false>(ctx, pl, pl.A, pl.small, pl.small, pl.lda, pl.as, pl.B, pl.A, pl.diag, cc / kScale, cb)
            : symmetric<1, 128, false>(ctx, pl, pl.A, pl.small, pl.small, pl.lda, pl.as, pl.B, pl.A, pl.diag, cc / kScale, cb);
        if (s + 1 < a.steps) {
            __half *out = pl.x[(s + 1) & 1];
            bigx ? iterate<2, 256, __half>(ctx, pl, x, out, pl.ldx, pl.xs, 1 / kScale, 1.0f, ca)
                 : iterate<1, 128, __half>(ctx, pl, x, out, pl.ldx, pl.xs, 1 / kScale, 1.0f, ca);
        } else {
            const float f = (float)a.scale / kScale;
            bigx ? iterate<2, 256, __nv_bfloat16>(ctx, pl, x, (__nv_bfloat16 *)a.out, a.ldo, a.ostride, f / kScale, f, ca)
                 : iterate<1, 128, __nv_bfloat16>(ctx, pl, x, (__nv_bfloat16 *)a.out, a.ldo, a.ostride, f / kScale, f, ca);
        }
    }
}

}  // namespace fitre
