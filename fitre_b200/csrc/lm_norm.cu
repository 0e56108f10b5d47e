// Layer norm over the rows of a matrix and its backward pass.
//   y = (x - m) r gamma + beta,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   xh = (x - m) r,  g = dy gamma:  dx = r (g - mean(g) - xh mean(g xh)),
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
// Both passes are bound by HBM, so each element is read once: a row lives in the registers of the G
// threads that share it (16 elements each, 32 to 1024 threads per row chosen by the row's length),
// the mean is subtracted before squaring (two reductions over registers cost nothing next to
// memory), and the following row's loads are issued before this row's reductions wait.  gamma and
// beta are re-read per row: after the first row they come from the SM's L1.  Rows longer than
// 16 x 1024 elements go through a form that re-reads the row (from L2) per pass.
// The weight gradient is summed in a fixed order without atomics: every block keeps the column sums of
// its rows in registers, writes one row of partial sums, and a second kernel adds those rows.
// Sums, mean and reciprocal deviation are fp32 (fp64 for fp64 tensors).
#include "lm_common.cuh"

namespace fitre {
namespace {

constexpr int N_ELEMS = 16;   // elements of a row one thread holds

// Sums `a` and `b` over the G threads of a row; every thread gets the result, added in one fixed
// order.  `slot` alternates between two halves of the buffer so that one barrier per call suffices.
template <int G, class A>
__device__ __forceinline__ void group_sum2(A &a, A &b, A *buf, int &slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (G > 32) {
        constexpr int W = G / 32;
        A *s = buf + slot * 2 * W;
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) {
            s[(threadIdx.x >> 5) * 2] = a;
            s[(threadIdx.x >> 5) * 2 + 1] = b;
        }
        __syncthreads();
        a = 0;
        b = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            a += s[2 * w];
            b += s[2 * w + 1];
        }
    }
}

template <int G> constexpr int norm_threads = G > 32 ? G : 256;   // threads of a block
template <class A> __device__ __forceinline__ A rsqrt_acc(A v);
template <> __device__ __forceinline__ float rsqrt_acc<float>(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double rsqrt_acc<double>(double v) { return 1.0 / sqrt(v); }

template <class T, class W, int VEC, int G>
__global__ void __launch_bounds__(norm_threads<G>, (sizeof(T) == 8 ? 512 : 1024) / norm_threads<G> > 0
                                                         ? (sizeof(T) == 8 ? 512 : 1024) / norm_threads<G>
                                                         : 1)
layer_norm_kernel(const T *x, long ldx, const W *__restrict__ gamma, const W *__restrict__ beta, T *y, long ldy,
                  acc_t<T> *mean, acc_t<T> *rstd, long rows, int cols, double eps) {
    using A = acc_t<T>;
    constexpr int CH = N_ELEMS / VEC;
    constexpr int RPB = norm_threads<G> / G;   // rows a block works on at a time
    __shared__ A buf[G > 32 ? 4 * (G / 32) : 1];
    const int t = threadIdx.x % G;
    const long step = (long)gridDim.x * RPB;
    long row = (long)blockIdx.x * RPB + threadIdx.x / G;
    int slot = 0;
    Vec<T, VEC> next[CH];
    if (row < rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if ((c * G + t) * VEC < cols) next[c] = load_vec<T, VEC>(x + row * ldx + (c * G + t) * VEC);
    }
    for (; row < rows; row += step) {
        A v[N_ELEMS];
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                v[c * VEC + e] = (c * G + t) * VEC < cols ? to_acc<A>(next[c].v[e]) : A(0);
        if (row + step < rows) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if ((c * G + t) * VEC < cols) next[c] = load_vec<T, VEC>(x + (row + step) * ldx + (c * G + t) * VEC);
        }
        A s = 0, unused = 0;
#pragma unroll
        for (int i = 0; i < N_ELEMS; ++i) s += v[i];
        group_sum2<G>(s, unused, buf, slot);
        const A m = s / (A)cols;
        A q = 0;
        unused = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if ((c * G + t) * VEC < cols) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A d = v[c * VEC + e] - m;
                    v[c * VEC + e] = d;
                    q += d * d;
                }
            }
        group_sum2<G>(q, unused, buf, slot);
        const A r = rsqrt_acc<A>(q / (A)cols + (A)eps);
        if (t == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + t) * VEC;
            if (at < cols) {
                Vec<T, VEC> o;
                Vec<W, VEC> g, b;
                if (gamma) g = load_vec<W, VEC>(gamma + at);
                if (beta) b = load_vec<W, VEC>(beta + at);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    A w = v[c * VEC + e] * r;
                    if (gamma) w *= to_acc<A>(g.v[e]);
                    if (beta) w += to_acc<A>(b.v[e]);
                    o.v[e] = from_acc<T>(w);
                }
                store_vec<T, VEC>(y + row * ldy + at, o);
            }
        }
    }
}

// Rows too long for registers: three sweeps over the row, the second and third from L2.
template <class T, class W>
__global__ void __launch_bounds__(1024, 1)
layer_norm_long_kernel(const T *x, long ldx, const W *__restrict__ gamma, const W *__restrict__ beta, T *y, long ldy,
                       acc_t<T> *mean, acc_t<T> *rstd, long rows, int cols, double eps) {
    using A = acc_t<T>;
    __shared__ A buf[4 * 32];
    int slot = 0;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        A s = 0, q = 0, unused = 0;
        for (int i = threadIdx.x; i < cols; i += 1024) s += to_acc<A>(xr[i]);
        group_sum2<1024>(s, unused, buf, slot);
        const A m = s / (A)cols;
        for (int i = threadIdx.x; i < cols; i += 1024) {
            const A d = to_acc<A>(xr[i]) - m;
            q += d * d;
        }
        unused = 0;
        group_sum2<1024>(q, unused, buf, slot);
        const A r = rsqrt_acc<A>(q / (A)cols + (A)eps);
        if (threadIdx.x == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
        for (int i = threadIdx.x; i < cols; i += 1024) {
            A w = (to_acc<A>(xr[i]) - m) * r;
            if (gamma) w *= to_acc<A>(gamma[i]);
            if (beta) w += to_acc<A>(beta[i]);
            y[row * ldy + i] = from_acc<T>(w);
        }
    }
}

template <class T, class W, int VEC, int G>
__global__ void __launch_bounds__(norm_threads<G>, norm_threads<G> <= 256 ? 2 : 1)
layer_norm_backward_kernel(const T *dy, long lddy, const T *x, long ldx, const W *__restrict__ gamma,
                           const acc_t<T> *__restrict__ mean, const acc_t<T> *__restrict__ rstd, T *dx, long lddx,
                           acc_t<T> *partial, long rows, int cols) {
    using A = acc_t<T>;
    constexpr int CH = N_ELEMS / VEC;
    constexpr int THREADS = norm_threads<G>;
    constexpr int RPB = THREADS / G;
    __shared__ A buf[G > 32 ? 4 * (G / 32) : 1];
    const int t = threadIdx.x % G;
    const long step = (long)gridDim.x * RPB;
    long row = (long)blockIdx.x * RPB + threadIdx.x / G;
    int slot = 0;
    A dg[N_ELEMS], db[N_ELEMS];
#pragma unroll
    for (int i = 0; i < N_ELEMS; ++i) dg[i] = db[i] = 0;
    Vec<T, VEC> nx[CH], nd[CH];
    if (row < rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if ((c * G + t) * VEC < cols) {
                nx[c] = load_vec<T, VEC>(x + row * ldx + (c * G + t) * VEC);
                nd[c] = load_vec<T, VEC>(dy + row * lddy + (c * G + t) * VEC);
            }
    }
    for (; row < rows; row += step) {
        const A m = mean[row], r = rstd[row];
        A xh[N_ELEMS], g[N_ELEMS];
        A s1 = 0, s2 = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + t) * VEC;
            if (at < cols) {
                Vec<W, VEC> w;
                if (gamma) w = load_vec<W, VEC>(gamma + at);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = c * VEC + e;
                    const A d = to_acc<A>(nd[c].v[e]);
                    xh[i] = (to_acc<A>(nx[c].v[e]) - m) * r;
                    dg[i] += d * xh[i];
                    db[i] += d;
                    g[i] = gamma ? d * to_acc<A>(w.v[e]) : d;
                    s1 += g[i];
                    s2 += g[i] * xh[i];
                }
            }
        }
        if (row + step < rows) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if ((c * G + t) * VEC < cols) {
                    nx[c] = load_vec<T, VEC>(x + (row + step) * ldx + (c * G + t) * VEC);
                    nd[c] = load_vec<T, VEC>(dy + (row + step) * lddy + (c * G + t) * VEC);
                }
        }
        group_sum2<G>(s1, s2, buf, slot);
        s1 /= (A)cols;
        s2 /= (A)cols;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + t) * VEC;
            if (at < cols) {
                Vec<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int i = c * VEC + e;
                    o.v[e] = from_acc<T>(r * (g[i] - s1 - xh[i] * s2));
                }
                store_vec<T, VEC>(dx + row * lddx + at, o);
            }
        }
    }
    if (!partial) return;
    A *pg = partial + (long)blockIdx.x * 2 * cols, *pb = pg + cols;
    if (G == 32) {
        // the block's warps hold the same columns: added in warp order through shared memory
        __shared__ A sg[G == 32 ? G * N_ELEMS : 1], sb[G == 32 ? G * N_ELEMS : 1];
        for (int w = 0; w < RPB; ++w) {
            if ((int)threadIdx.x / G == w) {
#pragma unroll
                for (int i = 0; i < N_ELEMS; ++i) {
                    A *pgs = sg + i * G + t, *pbs = sb + i * G + t;
                    *pgs = w ? *pgs + dg[i] : dg[i];
                    *pbs = w ? *pbs + db[i] : db[i];
                }
            }
            __syncthreads();
        }
        if ((int)threadIdx.x / G != 0) return;
#pragma unroll
        for (int i = 0; i < N_ELEMS; ++i) {
            dg[i] = sg[i * G + t];
            db[i] = sb[i * G + t];
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int at = (c * G + t) * VEC + e;
            if (at < cols) {
                pg[at] = dg[c * VEC + e];
                pb[at] = db[c * VEC + e];
            }
        }
}

// Column sums for rows too long for registers: a block takes 256 columns and every gridDim.y-th row.
template <class T>
__global__ void __launch_bounds__(256)
layer_norm_columns_kernel(const T *dy, long lddy, const T *x, long ldx, const acc_t<T> *__restrict__ mean,
                          const acc_t<T> *__restrict__ rstd, acc_t<T> *partial, long rows, int cols) {
    using A = acc_t<T>;
    const int at = blockIdx.x * 256 + threadIdx.x;
    if (at >= cols) return;
    A dg = 0, db = 0;
    for (long row = blockIdx.y; row < rows; row += gridDim.y) {
        const A d = to_acc<A>(dy[row * lddy + at]);
        dg += d * ((to_acc<A>(x[row * ldx + at]) - mean[row]) * rstd[row]);
        db += d;
    }
    partial[(long)blockIdx.y * 2 * cols + at] = dg;
    partial[(long)blockIdx.y * 2 * cols + cols + at] = db;
}

template <class T, class W>
__global__ void __launch_bounds__(1024, 1)
layer_norm_backward_long_kernel(const T *dy, long lddy, const T *x, long ldx, const W *__restrict__ gamma,
                                const acc_t<T> *__restrict__ mean, const acc_t<T> *__restrict__ rstd, T *dx,
                                long lddx, long rows, int cols) {
    using A = acc_t<T>;
    __shared__ A buf[4 * 32];
    int slot = 0;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx, *dr = dy + row * lddy;
        const A m = mean[row], r = rstd[row];
        A s1 = 0, s2 = 0;
        for (int i = threadIdx.x; i < cols; i += 1024) {
            const A g = gamma ? to_acc<A>(dr[i]) * to_acc<A>(gamma[i]) : to_acc<A>(dr[i]);
            s1 += g;
            s2 += g * ((to_acc<A>(xr[i]) - m) * r);
        }
        group_sum2<1024>(s1, s2, buf, slot);
        s1 /= (A)cols;
        s2 /= (A)cols;
        for (int i = threadIdx.x; i < cols; i += 1024) {
            const A g = gamma ? to_acc<A>(dr[i]) * to_acc<A>(gamma[i]) : to_acc<A>(dr[i]);
            dx[row * lddx + i] = from_acc<T>(r * (g - s1 - (to_acc<A>(xr[i]) - m) * r * s2));
        }
    }
}

// dgamma / dbeta from the blocks' partial rows: 32 columns per block, 32 row lanes, a fixed tree.
template <class W, class A>
__global__ void __launch_bounds__(1024)
layer_norm_reduce_kernel(const A *__restrict__ partial, int blocks, int cols, W *dgamma, W *dbeta) {
    __shared__ A s[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int at = blockIdx.x * 32 + lane;   // column of [dgamma | dbeta]
    A v = 0;
    if (at < 2 * cols)
        for (int b = w; b < blocks; b += 32) v += partial[(long)b * 2 * cols + at];
    s[w][lane] = v;
    __syncthreads();
    v = s[lane][w];                          // warp w now holds the 32 lanes' sums of column w
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int col = blockIdx.x * 32 + w;
    if (lane == 0 && col < 2 * cols) {
        W *out = col < cols ? dgamma : dbeta;
        if (out) out[col < cols ? col : col - cols] = from_acc<W>(v);
    }
}

int group_for(int cols) {
    for (int g : {32, 128, 256, 512, 1024})
        if (cols <= g * N_ELEMS) return g;
    return 0;
}
int blocks_for(long rows, int g, int threads_per_sm) {
    const int threads = g > 32 ? g : 256;
    const long need = (rows + threads / g - 1) / (threads / g);
    const long room = (long)kLmSms * (threads_per_sm > threads ? threads_per_sm / threads : 1);
    return (int)(need < room ? need : room);
}
constexpr int kBackThreads = 512;        // resident threads per SM of the backward kernel
constexpr int kLongSplit = 64;           // row splits of the column sums of long rows

template <class T, class W, int VEC>
void forward_as(fitre_context *ctx, const NormArgs &a) {
    using A = acc_t<T>;
    const int g = group_for(a.cols);
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const W *gm = (const W *)a.gamma, *bt = (const W *)a.beta;
    A *mean = (A *)a.mean, *rstd = (A *)a.rstd;
    const int blocks = blocks_for(a.rows, g ? g : 1024, sizeof(T) == 8 ? 512 : 1024);
#define NORM_LAUNCH(G)                                                                                       \
    layer_norm_kernel<T, W, VEC, G><<<blocks, norm_threads<G>, 0, ctx->stream>>>(                          \
        x, a.ldx, gm, bt, y, a.ldy, mean, rstd, a.rows, a.cols, a.eps)
    switch (g) {
        case 32: NORM_LAUNCH(32); break;
        case 128: NORM_LAUNCH(128); break;
        case 256: NORM_LAUNCH(256); break;
        case 512: NORM_LAUNCH(512); break;
        case 1024: NORM_LAUNCH(1024); break;
        default:
            layer_norm_long_kernel<T, W><<<blocks, 1024, 0, ctx->stream>>>(x, a.ldx, gm, bt, y, a.ldy, mean, rstd,
                                                                            a.rows, a.cols, a.eps);
            check_launch(ctx, "layer_norm_long_kernel");
            return;
    }
#undef NORM_LAUNCH
    check_launch(ctx, "layer_norm_kernel");
}

template <class T, class W, int VEC>
void backward_as(fitre_context *ctx, const NormArgs &a) {
    using A = acc_t<T>;
    const int g = group_for(a.cols);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    T *dx = (T *)a.dx;
    const W *gm = (const W *)a.gamma;
    const A *mean = (const A *)a.mean, *rstd = (const A *)a.rstd;
    A *partial = a.dgamma || a.dbeta ? (A *)a.scratch : nullptr;
    int blocks = blocks_for(a.rows, g ? g : 1024, kBackThreads);
#define NORM_LAUNCH(G)                                                                                       \
    layer_norm_backward_kernel<T, W, VEC, G><<<blocks, norm_threads<G>, 0, ctx->stream>>>(                 \
        dy, a.lddy, x, a.ldx, gm, mean, rstd, dx, a.lddx, partial, a.rows, a.cols)
    switch (g) {
        case 32: NORM_LAUNCH(32); break;
        case 128: NORM_LAUNCH(128); break;
        case 256: NORM_LAUNCH(256); break;
        case 512: NORM_LAUNCH(512); break;
        case 1024: NORM_LAUNCH(1024); break;
        default: {
            if (partial) {   // before dx, which may overwrite dy or x
                const int split = (int)(a.rows < kLongSplit ? a.rows : kLongSplit);
                layer_norm_columns_kernel<T><<<dim3((a.cols + 255) / 256, split), 256, 0, ctx->stream>>>(
                    dy, a.lddy, x, a.ldx, mean, rstd, partial, a.rows, a.cols);
                check_launch(ctx, "layer_norm_columns_kernel");
                layer_norm_reduce_kernel<W, A><<<(2 * a.cols + 31) / 32, 1024, 0, ctx->stream>>>(
                    partial, split, a.cols, (W *)a.dgamma, (W *)a.dbeta);
                check_launch(ctx, "layer_norm_reduce_kernel");
            }
            layer_norm_backward_long_kernel<T, W><<<blocks, 1024, 0, ctx->stream>>>(dy, a.lddy, x, a.ldx, gm, mean,
                                                                                     rstd, dx, a.lddx, a.rows, a.cols);
            check_launch(ctx, "layer_norm_backward_long_kernel");
            return;
        }
    }
#undef NORM_LAUNCH
    check_launch(ctx, "layer_norm_backward_kernel");
    if (partial) {
        layer_norm_reduce_kernel<W, A><<<(2 * a.cols + 31) / 32, 1024, 0, ctx->stream>>>(
            partial, blocks, a.cols, (W *)a.dgamma, (W *)a.dbeta);
        check_launch(ctx, "layer_norm_reduce_kernel");
    }
}

// The widest access the call's pointers, row strides and width allow.
bool norm_vectorised(const NormArgs &a, int vec) {
    const int e = dtype_bytes(a.dtype);
    if (a.cols % vec) return false;
    for (const void *p : {a.x, a.dy, a.gamma, a.beta, (const void *)a.y, (const void *)a.dx})
        if (p && !aligned16(p)) return false;
    for (long ld : {a.ldx, a.lddy, a.ldy, a.lddx})
        if ((ld * e) % 16) return false;
    return true;
}

template <class T, class W, int VEC>
void norm_typed(fitre_context *ctx, const NormArgs &a, bool back) {
    if (norm_vectorised(a, VEC)) {
        back ? backward_as<T, W, VEC>(ctx, a) : forward_as<T, W, VEC>(ctx, a);
    } else {
        back ? backward_as<T, W, 1>(ctx, a) : forward_as<T, W, 1>(ctx, a);
    }
}

void norm_dispatch(fitre_context *ctx, const NormArgs &a, bool back) {
    const bool wide = a.wtype == FITRE_DTYPE_F32;
    switch (a.dtype) {
        case FITRE_DTYPE_F64: return norm_typed<double, double, 2>(ctx, a, back);
        case FITRE_DTYPE_F32: return norm_typed<float, float, 4>(ctx, a, back);
        case FITRE_DTYPE_BF16:
            return wide ? norm_typed<__nv_bfloat16, float, 8>(ctx, a, back)
                        : norm_typed<__nv_bfloat16, __nv_bfloat16, 8>(ctx, a, back);
        default:
            return wide ? norm_typed<__half, float, 8>(ctx, a, back) : norm_typed<__half, __half, 8>(ctx, a, back);
    }
}

}  // namespace

long layer_norm_backward_scratch(long rows, long cols) {
    const int g = cols <= 1024 * N_ELEMS ? group_for((int)cols) : 0;
    const long parts = g ? blocks_for(rows, g, kBackThreads) : (rows < kLongSplit ? rows : kLongSplit);
    return parts * 2 * cols * (long)sizeof(double);
}
void layer_norm_forward(fitre_context *ctx, const NormArgs &a) { norm_dispatch(ctx, a, false); }
void layer_norm_backward(fitre_context *ctx, const NormArgs &a) { norm_dispatch(ctx, a, true); }

}  // namespace fitre
