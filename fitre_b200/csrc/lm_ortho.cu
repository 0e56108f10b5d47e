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
// Products accumulate in fp32; the result is rounded to bf16 once, and is within about half a bf16
// rounding of the exact polynomial before that.
#include "lm_gemm.cuh"

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

// Sums of squares of each matrix's parts, in fp64 (squares of fp32 values overflow fp32): part p holds every
// gridDim.x-th row.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
ortho_norm_kernel(const T *in, long ld, long bstride, int rows, int cols, double *partial) {
    __shared__ double s[8];
    const T *m = in + blockIdx.y * bstride;
    double q = 0;
    for (int r = blockIdx.x; r < rows; r += gridDim.x)
#pragma unroll 4
        for (int c = threadIdx.x * VEC; c < cols; c += 256 * VEC) {
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

// The first iterate, as a pair of fp16 matrices.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
ortho_scale_kernel(const T *in, long ld, long bstride, int rows, int cols, const double *__restrict__ partial, int parts,
                   double eps, __half *hi, __half *lo, long ldo, long ostride) {
    __shared__ double s[8];
    double q = 0;
    for (int i = threadIdx.x; i < parts; i += 256) q += partial[(long)blockIdx.y * parts + i];
    const double f = (double)kScale / (sqrt(block_sum(q, s)) + eps);
    const T *m = in + blockIdx.y * bstride;
    hi += blockIdx.y * ostride;
    lo += blockIdx.y * ostride;
    for (int r = blockIdx.x; r < rows; r += gridDim.x)
#pragma unroll 2
        for (int c = threadIdx.x * VEC; c < cols; c += 256 * VEC) {
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
}

// A symmetric product: tile and, off the diagonal, its mirror image.  out = kacc * acc + kin * in; with
// `diag`, the diagonal goes there (unscaled, fp32) and zeros take its place.
struct SymmetricEpi {
    struct Params {
        __half *out;
        const __half *in;
        float *diag;
        long ld, stride;
        int n;
        float kacc, kin;
    };
    static constexpr bool kTwoMaps = false;
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row, uint32_t tmem) {
        __half *out = p.out + at.batch * p.stride;
        const __half *in = p.in ? p.in + at.batch * p.stride : nullptr;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            const int col = at.n * BN + c;
            if (col >= p.n) break;
            float v[32];
            tmem_load32(tmem + c, v);
            if (row < p.n) {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] *= p.kacc;
                if (in) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (col + e < p.n) v[e] += p.kin * __half2float(in[row * p.ld + col + e]);
                }
                if (p.diag && row >= col && row < col + 32) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (row == col + e) {
                            p.diag[(long)at.batch * p.n + row] = v[e] * (1 / kScale);
                            v[e] = 0.0f;
                        }
                }
                store_row32(out + row * p.ld, col, p.n, true, v);
                if (at.m != at.n) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (col + e < p.n) out[(col + e) * p.ld + row] = __float2half_rn(v[e]);
                }
            }
        }
    }
};

// X <- a X + B X:  v = kacc * acc + kout * ((a + d) hi + (a or a + d) lo), acc = (B without its diagonal d) hi.
// The low part takes a alone, which is what acts on directions outside the update, but for the last
// step, where no further step amplifies them and a + d is closer for all others.
// T = __half: v becomes the next pair (lo in place); else v is the result.
template <class T>
struct IterateEpi {
    struct Params {
        T *out;
        const __half *hi;
        __half *lo;
        const float *diag;
        long ldo, ostride, ldx, xstride;
        int M, N, small;
        float kacc, kout, a;
        bool tall, wide;
    };
    static constexpr bool kTwoMaps = false;
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row, uint32_t tmem) {
        constexpr bool kLast = !std::is_same<T, __half>::value;
        T *out = p.out + at.batch * p.ostride + (long)row * p.ldo;
        const __half *hi = p.hi + at.batch * p.xstride + (long)row * p.ldx;
        __half *lo = p.lo + at.batch * p.xstride + (long)row * p.ldx;
        const float *diag = p.diag + (long)at.batch * p.small;
        const float drow = !p.tall && row < p.M ? diag[row] : 0.0f;
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            const int col = at.n * BN + c;
            if (col >= p.N) break;
            float v[32];
            tmem_load32(tmem + c, v);
            if (row < p.M) {
                // columns beyond N stay inside the row's padding to a multiple of 8
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (col + i * 8 >= p.N) break;
                    const Vec<__half, 8> h = load_vec<__half, 8>(hi + col + i * 8), l = load_vec<__half, 8>(lo + col + i * 8);
                    Vec<__half, 8> nh, nl;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = col + i * 8 + e;
                        const float d = p.tall ? (j < p.N ? diag[j] : 0.0f) : drow;
                        const float x = (p.a + d) * __half2float(h.v[e]) + (kLast ? p.a + d : p.a) * __half2float(l.v[e]);
                        const float w = p.kacc * v[i * 8 + e] + p.kout * x;
                        v[i * 8 + e] = w;
                        nh.v[e] = __float2half_rn(w);
                        nl.v[e] = __float2half_rn(w - __half2float(nh.v[e]));
                    }
                    if (!kLast) {
                        store_vec<__half, 8>((__half *)out + col + i * 8, nh);
                        store_vec<__half, 8>(lo + col + i * 8, nl);
                    }
                }
                if (kLast) store_row32(out, col, p.N, p.wide, v);
            }
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

template <int CG, int BN, bool MN>
void symmetric(fitre_context *ctx, const Plan &pl, const __half *x, long K, long rows, long cols, long ld, long stride,
               __half *out, const __half *in, float *diag, float kacc, float kin) {
    // the matrix is rows x cols in memory; MN: its columns are the product's index
    GemmArgs<SymmetricEpi::Params> g = {};
    gemm_map(&g.a[0], x, cols, rows, pl.batch, ld, stride, a_box<CG, BN, MN>, G_F16);
    gemm_map(&g.b[0], x, cols, rows, pl.batch, ld, stride, b_box<CG, BN, MN, false>, G_F16);
    g.g.za = g.g.zb = 1;
    g.epi = {out, in, diag, pl.lda, pl.as, pl.small, kacc, kin};
    gemm_launch<CG, BN, MN, MN, SymmetricEpi>(ctx, g, pl.small, pl.small, pl.batch, true, K, 1, G_F16,
                                              "ortho_symmetric_kernel");
}

template <int CG, int BN, class T>
void iterate(fitre_context *ctx, const Plan &pl, const __half *x, T *out, long ldo, long ostride, bool wide, float kacc,
             float kout, float a) {
    GemmArgs<typename IterateEpi<T>::Params> g = {};
    g.g.za = g.g.zb = 1;
    g.epi = {out, x, pl.lo, pl.diag, ldo, ostride, pl.ldx, pl.xs, pl.rows, pl.cols, pl.small, kacc, kout, a, pl.tall, wide};
    if (pl.tall) {   // X B: B is symmetric, its rows serve as its columns
        gemm_map(&g.a[0], x, pl.cols, pl.rows, pl.batch, pl.ldx, pl.xs, a_box<CG, BN, false>, G_F16);
        gemm_map(&g.b[0], pl.B, pl.small, pl.small, pl.batch, pl.lda, pl.as, b_box<CG, BN, false, false>, G_F16);
        gemm_launch<CG, BN, false, false, IterateEpi<T>>(ctx, g, pl.rows, pl.cols, pl.batch, false, pl.small, 1, G_F16,
                                                         "ortho_iterate_kernel");
    } else {
        gemm_map(&g.a[0], pl.B, pl.small, pl.small, pl.batch, pl.lda, pl.as, a_box<CG, BN, false>, G_F16);
        gemm_map(&g.b[0], x, pl.cols, pl.rows, pl.batch, pl.ldx, pl.xs, b_box<CG, BN, true, false>, G_F16);
        gemm_launch<CG, BN, false, true, IterateEpi<T>>(ctx, g, pl.rows, pl.cols, pl.batch, false, pl.small, 1, G_F16,
                                                        "ortho_iterate_kernel");
    }
}

template <class T, int VEC>
void start_as(fitre_context *ctx, const OrthoArgs &a, const Plan &pl) {
    const dim3 grid(pl.parts, pl.batch);
    ortho_norm_kernel<T, VEC><<<grid, 256, 0, ctx->stream>>>((const T *)a.in, a.ldi, a.istride, pl.rows, pl.cols,
                                                             pl.partial);
    check_launch(ctx, "ortho_norm_kernel");
    ortho_scale_kernel<T, VEC><<<grid, 256, 0, ctx->stream>>>((const T *)a.in, a.ldi, a.istride, pl.rows, pl.cols,
                                                              pl.partial, pl.parts, a.eps, pl.x[0], pl.lo, pl.ldx, pl.xs);
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
    const long side = (pl.small + 255) / 256;
    const bool big = side * (side + 1) / 2 * pl.batch >= kLmSms / 2 - 16;
    const long cover = (long)((pl.rows + 255) / 256) * ((pl.cols + 255) / 256) * pl.batch;
    const bool bigx = cover >= kLmSms / 2 - 16;
    const long K = pl.tall ? pl.rows : pl.cols;
    for (int s = 0; s < a.steps; ++s) {
        const float ca = (float)a.coef[0], cb = (float)a.coef[1], cc = (float)a.coef[2];
        const __half *x = pl.x[s & 1];
        if (pl.tall) {
            big ? symmetric<2, 256, true>(ctx, pl, x, K, pl.rows, pl.cols, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0)
                : symmetric<1, 128, true>(ctx, pl, x, K, pl.rows, pl.cols, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0);
        } else {
            big ? symmetric<2, 256, false>(ctx, pl, x, K, pl.rows, pl.cols, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0)
                : symmetric<1, 128, false>(ctx, pl, x, K, pl.rows, pl.cols, pl.ldx, pl.xs, pl.A, nullptr, nullptr, 1 / kScale, 0);
        }
        big ? symmetric<2, 256, false>(ctx, pl, pl.A, pl.small, pl.small, pl.small, pl.lda, pl.as, pl.B, pl.A, pl.diag, cc / kScale, cb)
            : symmetric<1, 128, false>(ctx, pl, pl.A, pl.small, pl.small, pl.small, pl.lda, pl.as, pl.B, pl.A, pl.diag, cc / kScale, cb);
        if (s + 1 < a.steps) {
            __half *out = pl.x[(s + 1) & 1];
            bigx ? iterate<2, 256, __half>(ctx, pl, x, out, pl.ldx, pl.xs, true, 1 / kScale, 1.0f, ca)
                 : iterate<1, 128, __half>(ctx, pl, x, out, pl.ldx, pl.xs, true, 1 / kScale, 1.0f, ca);
        } else {
            const float f = (float)a.scale / kScale;
            const bool wide = tma_readable(a.out, a.ldo) && a.ostride % 8 == 0;
            bigx ? iterate<2, 256, __nv_bfloat16>(ctx, pl, x, (__nv_bfloat16 *)a.out, a.ldo, a.ostride, wide, f / kScale, f, ca)
                 : iterate<1, 128, __nv_bfloat16>(ctx, pl, x, (__nv_bfloat16 *)a.out, a.ldo, a.ostride, wide, f / kScale, f, ca);
        }
    }
}

}  // namespace fitre
