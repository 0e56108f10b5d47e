// Layer norm over the rows of a matrix and its backward pass.
//   y = (x - m) r gamma + beta,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   xh = (x - m) r,  g = dy gamma:  dx = r (g - mean(g) - xh mean(g xh)),
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
// Both passes are bound by HBM, so each element is read once: a row lives in the registers of the G
// threads that share it (16 elements each, 32 to 1024 threads per row chosen by the row's length),
// the mean is subtracted before squaring (two reductions over registers cost nothing next to
// memory).  gamma and beta are re-read per row: after the first row they come from the SM's L1.
//   * forward, up to 1024 elements: a warp per row, no barrier;
//   * wider rows on 16-byte boundaries: blocks that stay resident and have their next rows copied into a
//     ring in shared memory by bulk copies, which keep more bytes in flight than registers could;
//   * other rows: the same blocks with element-wise loads into registers, one row ahead;
//   * rows longer than 16 x 1024 elements: a form that re-reads the row (from L2) per pass.
// The weight gradient is summed in a fixed order without atomics: every block keeps the column sums of
// its rows in registers, writes one row of partial sums, and a second kernel adds those rows.
// Sums, mean and reciprocal deviation are fp32 (fp64 for fp64 tensors).
// Measured on a B200 (6.5 TB/s copy): 20011 x 1023 fp32 forward 34 us (4.8 TB/s; element-wise accesses, LSU), gradient of
// 16384 x 4096 bf16 with both sums 78 us (5.2 TB/s; 134 us with the rows in registers, one at a time).
#include "lm_common.cuh"
#include "lm_ring.cuh"
#include "lm_simd.cuh"

namespace fitre {
namespace {

// Elements of a row one thread holds, and the most threads that share a row: fp64 elements take twice the
// registers, of which 1024 threads have 64 each.
constexpr int N_ELEMS = 16;
template <class T> constexpr int n_elems = sizeof(T) == 8 ? 8 : N_ELEMS;
template <class T> constexpr int max_group = sizeof(T) == 8 ? 512 : 1024;

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

// The same for N values at once.
template <int G, int N, class A>
__device__ __forceinline__ void group_sums(A (&v)[N], A *buf, int &slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    constexpr int W = G / 32;
    A *s = buf + slot * N * W;
    slot ^= 1;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[(threadIdx.x >> 5) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += s[w * N + i];
}
template <int G, class A>
__device__ __forceinline__ A group_sum(A a, A *buf, int &slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (G > 32) {
        constexpr int W = G / 32;
        A *s = buf + slot * 2 * W;
        slot ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
        __syncthreads();
        a = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) a += s[w];
    }
    return a;
}

template <int G> constexpr int norm_threads = G > 32 ? G : 256;   // threads of a block
template <class A> __device__ __forceinline__ A rsqrt_acc(A v);
template <> __device__ __forceinline__ float rsqrt_acc<float>(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double rsqrt_acc<double>(double v) { return 1.0 / sqrt(v); }


// The row's elements that one thread of a group holds: chunks c of VEC consecutive elements at (c G + t) VEC,
// as packs of accumulators.
template <class T, int VEC, int G, int CH> struct RowPart {
    using A = acc_t<T>;
    using P = SimdOf<T, VEC>;
    static constexpr int PV = VEC / kPack<VEC>;   // packs in a chunk
    P v[CH][PV];
    int left;                                     // chunk c exists while c * G * VEC < left
    __device__ __forceinline__ RowPart(int cols, int t) : left(cols - t * VEC) {}
    __device__ __forceinline__ bool has(int c) const { return c * G * VEC < left; }
    __device__ __forceinline__ void set(int c, const Vec<T, VEC> &x) { widen(x, v[c]); }
    __device__ __forceinline__ void clear(int c) {
#pragma unroll
        for (int i = 0; i < PV; ++i) v[c][i] = P::splat(A(0));
    }
    __device__ __forceinline__ A sum() const {
        P s = P::splat(A(0));
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < PV; ++i) s = add(s, v[c][i]);
        return s.sum();
    }
    // subtracts the mean; returns the sum of the squares that remain
    __device__ __forceinline__ A centre(A m) {
        const P back = P::splat(-m);
        P q = P::splat(A(0));
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (has(c)) {
#pragma unroll
                for (int i = 0; i < PV; ++i) {
                    v[c][i] = add(v[c][i], back);
                    q = fma(v[c][i], v[c][i], q);
                }
            }
        return q.sum();
    }
    // y = v r gamma + beta, `gamma`, `beta` and `y` at this thread's first element.  AFFINE: both are there.
    // Their loads go out together, four chunks at a time: one after the other they would cost an L1 latency each.
    template <bool AFFINE, class W>
    __device__ __forceinline__ void store(A r, const W *gamma, const W *beta, T *y) const {
        const P scale = P::splat(r);
        constexpr int BATCH = CH < 4 ? CH : 4;
#pragma unroll
        for (int c0 = 0; c0 < CH; c0 += BATCH) {
            Vec<W, VEC> gm[BATCH], bt[BATCH];
            if (AFFINE) {
#pragma unroll
                for (int c = 0; c < BATCH; ++c)
                    if (has(c0 + c)) {
                        gm[c] = load_vec<W, VEC>(gamma + (c0 + c) * G * VEC);
                        bt[c] = load_vec<W, VEC>(beta + (c0 + c) * G * VEC);
                    }
            }
#pragma unroll
            for (int c = 0; c < BATCH; ++c) {
                P o[PV], w[PV], u[PV];
#pragma unroll
                for (int i = 0; i < PV; ++i) o[i] = mul(v[c0 + c][i], scale);
                if (AFFINE) {
                    widen(gm[c], w);
                    widen(bt[c], u);
#pragma unroll
                    for (int i = 0; i < PV; ++i) o[i] = fma(o[i], w[i], u[i]);
                } else if (has(c0 + c)) {
                    if (gamma) {
                        widen(load_vec<W, VEC>(gamma + (c0 + c) * G * VEC), w);
#pragma unroll
                        for (int i = 0; i < PV; ++i) o[i] = mul(o[i], w[i]);
                    }
                    if (beta) {
                        widen(load_vec<W, VEC>(beta + (c0 + c) * G * VEC), u);
#pragma unroll
                        for (int i = 0; i < PV; ++i) o[i] = add(o[i], u[i]);
                    }
                }
                if (has(c0 + c)) store_vec<T, VEC>(y + (c0 + c) * G * VEC, narrowed<T, VEC>(o));
            }
        }
    }
};

// Blocks that stay resident, G threads per row, the next row's elements loaded one row ahead.
template <class T, class W, int VEC, int G, bool AFFINE>
__global__ void __launch_bounds__(G, (sizeof(T) == 8 ? 512 : 1024) / G > 0 ? (sizeof(T) == 8 ? 512 : 1024) / G : 1)
layer_norm_kernel(const T *x, long ldx, const W *__restrict__ gamma, const W *__restrict__ beta, T *y, long ldy,
                  acc_t<T> *mean, acc_t<T> *rstd, long rows, int cols, double eps) {
    using A = acc_t<T>;
    constexpr int CH = n_elems<T> / VEC;
    __shared__ A buf[4 * (G / 32)];
    const int t = threadIdx.x;
    const A over = A(1) / (A)cols;
    int slot = 0;
    x += t * VEC;
    y += t * VEC;
    if (gamma) gamma += t * VEC;
    if (beta) beta += t * VEC;
    RowPart<T, VEC, G, CH> part(cols, t);
    Vec<T, VEC> next[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (part.has(c)) next[c] = load_vec<T, VEC>(x + blockIdx.x * ldx + c * G * VEC);
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long after = row + gridDim.x;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (part.has(c)) part.set(c, next[c]);
            else part.clear(c);
        }
        if (after < rows) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (part.has(c)) next[c] = load_vec<T, VEC>(x + after * ldx + c * G * VEC);
        }
        const A m = group_sum<G>(part.sum(), buf, slot) * over;
        const A r = rsqrt_acc<A>(group_sum<G>(part.centre(m), buf, slot) * over + (A)eps);
        if (t == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
        part.template store<AFFINE>(r, gamma, beta, y + row * ldy);
    }
}

// A warp per row of up to 1024 elements, N (8, 16 or 32) to a lane.
constexpr int N_WIDE = 32;
template <class T, class W, int VEC, int N, bool AFFINE>
__global__ void __launch_bounds__(256, sizeof(T) == 8 ? 2 : 4)
layer_norm_warp_kernel(const T *x, long ldx, const W *__restrict__ gamma, const W *__restrict__ beta, T *y, long ldy,
                       acc_t<T> *mean, acc_t<T> *rstd, long rows, int cols, double eps) {
    using A = acc_t<T>;
    constexpr int CH = N / VEC;
    const int t = threadIdx.x & 31;
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    x += row * ldx + t * VEC;
    RowPart<T, VEC, 32, CH> part(cols, t);
    int slot = 0;
    {
        Vec<T, VEC> raw[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (part.has(c)) raw[c] = load_vec<T, VEC>(x + c * 32 * VEC);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (part.has(c)) part.set(c, raw[c]);
            else part.clear(c);
        }
    }
    const A m = group_sum<32>(part.sum(), (A *)nullptr, slot) / (A)cols;
    const A r = rsqrt_acc<A>(group_sum<32>(part.centre(m), (A *)nullptr, slot) / (A)cols + (A)eps);
    if (t == 0) {
        if (mean) mean[row] = m;
        if (rstd) rstd[row] = r;
    }
    part.template store<AFFINE>(r, gamma ? gamma + t * VEC : gamma, beta ? beta + t * VEC : beta, y + row * ldy + t * VEC);
}

// Rows on 16-byte boundaries through a ring of `stages` rows in shared memory.
template <class T, class W, int VEC, int G, bool AFFINE>
__global__ void __launch_bounds__(G, 1024 / G)
layer_norm_ring_kernel(const T *x, long ldx, const W *__restrict__ gamma, const W *__restrict__ beta, T *y, long ldy,
                       acc_t<T> *mean, acc_t<T> *rstd, long rows, int cols, double eps, int stages, int *err) {
    using A = acc_t<T>;
    constexpr int CH = n_elems<T> / VEC;
    extern __shared__ __align__(16) unsigned char ring_raw[];
    __shared__ unsigned long long bars[kRingMax];
    __shared__ A buf[4 * (G / 32)];
    const int t = threadIdx.x;
    const long step = gridDim.x;
    const A over = A(1) / (A)cols;
    int slot = 0;
    RowRing ring(ring_raw, bars, stages, cols * (int)sizeof(T));
    ring.init();
    if (t == 0)
        for (int i = 0; i < stages; ++i)
            if (blockIdx.x + i * step < rows) ring.fill(i, x + (blockIdx.x + i * step) * ldx);
    y += t * VEC;
    if (gamma) gamma += t * VEC;
    if (beta) beta += t * VEC;
    RowPart<T, VEC, G, CH> part(cols, t);
    for (long row = blockIdx.x; row < rows; row += step) {
        if (!ring.wait()) {
            if (t == 0) atomicExch(err, 1);
            return;
        }
        const T *in = (const T *)ring.data() + t * VEC;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (part.has(c)) part.set(c, load_vec<T, VEC>(in + c * G * VEC));
            else part.clear(c);
        }
        // the sum's barrier also says that every thread has read the stage: the sum is made of what was read
        const A m = group_sum<G>(part.sum(), buf, slot) * over;
        if (t == 0 && row + stages * step < rows) ring.fill(ring.at, x + (row + stages * step) * ldx);
        ring.advance();
        const A r = rsqrt_acc<A>(group_sum<G>(part.centre(m), buf, slot) * over + (A)eps);
        if (t == 0) {
            if (mean) mean[row] = m;
            if (rstd) rstd[row] = r;
        }
        part.template store<AFFINE>(r, gamma, beta, y + row * ldy);
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

// One row of the backward pass as a thread sees it, and its share of the sums over rows.
template <class T, class W, int VEC, int G, int CH> struct BackPart {
    using A = acc_t<T>;
    using P = SimdOf<T, VEC>;
    static constexpr int PV = VEC / kPack<VEC>;
    P dg[CH][PV], db[CH][PV], xh[CH][PV], g[CH][PV];
    Vec<W, VEC> gm[CH];
    int left;
    __device__ __forceinline__ BackPart(int cols, int t, const W *gamma) : left(cols - t * VEC) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int i = 0; i < PV; ++i) dg[c][i] = db[c][i] = P::splat(A(0));
#pragma unroll
            for (int e = 0; e < VEC; ++e) gm[c].v[e] = from_acc<W>(A(1));
            if (gamma && has(c)) gm[c] = load_vec<W, VEC>(gamma + c * G * VEC);
        }
    }
    __device__ __forceinline__ bool has(int c) const { return c * G * VEC < left; }
    // sums of g and g xh over this thread's elements, from functions that give chunk c of x and dy
    template <class X, class D> __device__ __forceinline__ void take(A m, A r, X &&x_at, D &&d_at, A &s1, A &s2) {
        const P scale = P::splat(r), shift = P::splat(-m * r);
        P a = P::splat(A(0)), b = a;
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (has(c)) {
                P d[PV], w[PV];
                widen(x_at(c), xh[c]);
                widen(d_at(c), d);
                widen(gm[c], w);
#pragma unroll
                for (int i = 0; i < PV; ++i) {
                    xh[c][i] = fma(xh[c][i], scale, shift);
                    dg[c][i] = fma(d[i], xh[c][i], dg[c][i]);
                    db[c][i] = add(db[c][i], d[i]);
                    g[c][i] = mul(d[i], w[i]);
                    a = add(a, g[c][i]);
                    b = fma(g[c][i], xh[c][i], b);
                }
            }
        s1 = a.sum();
        s2 = b.sum();
    }
    // dx = r (g - s1 - xh s2)
    __device__ __forceinline__ void store(A r, A s1, A s2, T *dx) const {
        const P scale = P::splat(r), back1 = P::splat(-s1 * r), back2 = P::splat(-s2 * r);
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (has(c)) {
                P o[PV];
#pragma unroll
                for (int i = 0; i < PV; ++i) o[i] = fma(xh[c][i], back2, fma(g[c][i], scale, back1));
                store_vec<T, VEC>(dx + c * G * VEC, narrowed<T, VEC>(o));
            }
    }
    // this thread's columns of the block's partial sums
    __device__ __forceinline__ void flush(A *pg, A *pb) const {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (has(c)) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    pg[c * G * VEC + e] = dg[c][e / kPack<VEC>].get(e % kPack<VEC>);
                    pb[c * G * VEC + e] = db[c][e / kPack<VEC>].get(e % kPack<VEC>);
                }
            }
    }
};

template <class T, class W, int VEC, int G>
__global__ void __launch_bounds__(norm_threads<G>, norm_threads<G> <= 256 ? 2 : 1)
layer_norm_backward_kernel(const T *dy, long lddy, const T *x, long ldx, const W *__restrict__ gamma,
                           const acc_t<T> *__restrict__ mean, const acc_t<T> *__restrict__ rstd, T *dx, long lddx,
                           acc_t<T> *partial, long rows, int cols) {
    using A = acc_t<T>;
    constexpr int CH = n_elems<T> / VEC;
    constexpr int RPB = norm_threads<G> / G;   // rows a block works on at a time
    __shared__ A buf[G > 32 ? 4 * (G / 32) : 1];
    const int t = threadIdx.x % G, group = threadIdx.x / G;
    const long step = (long)gridDim.x * RPB;
    long row = (long)blockIdx.x * RPB + group;
    int slot = 0;
    x += t * VEC;
    dy += t * VEC;
    dx += t * VEC;
    const A over = A(1) / (A)cols;
    BackPart<T, W, VEC, G, CH> part(cols, t, gamma ? gamma + t * VEC : gamma);
    Vec<T, VEC> nx[CH], nd[CH];
    if (row < rows) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (part.has(c)) {
                nx[c] = load_vec<T, VEC>(x + row * ldx + c * G * VEC);
                nd[c] = load_vec<T, VEC>(dy + row * lddy + c * G * VEC);
            }
    }
    for (; row < rows; row += step) {
        const A r = rstd[row];
        A s1, s2;
        part.take(mean[row], r, [&](int c) { return nx[c]; }, [&](int c) { return nd[c]; }, s1, s2);
        if (row + step < rows) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (part.has(c)) {
                    nx[c] = load_vec<T, VEC>(x + (row + step) * ldx + c * G * VEC);
                    nd[c] = load_vec<T, VEC>(dy + (row + step) * lddy + c * G * VEC);
                }
        }
        group_sum2<G>(s1, s2, buf, slot);
        part.store(r, s1 * over, s2 * over, dx + row * lddx);
    }
    if (!partial) return;
    A *pg = partial + (long)blockIdx.x * 2 * cols + t * VEC, *pb = pg + cols;
    if (G > 32) {
        part.flush(pg, pb);
        return;
    }
    // the block's warps hold the same columns: added in warp order through shared memory
    __shared__ A sg[G == 32 ? G * n_elems<T> : 1], sb[G == 32 ? G * n_elems<T> : 1];
    for (int w = 0; w < RPB; ++w) {
        if (group == w) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (part.has(c)) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int i = c * G * VEC + t * VEC + e;
                        const A a = part.dg[c][e / kPack<VEC>].get(e % kPack<VEC>), b = part.db[c][e / kPack<VEC>].get(e % kPack<VEC>);
                        sg[i] = w ? sg[i] + a : a;
                        sb[i] = w ? sb[i] + b : b;
                    }
                }
        }
        __syncthreads();
    }
    pg -= t * VEC;
    pb -= t * VEC;
    for (int i = threadIdx.x; i < cols; i += norm_threads<G>) {
        pg[i] = sg[i];
        pb[i] = sb[i];
    }
}

// Rows on 16-byte boundaries through a ring, R (1 or 2) rows at a time: two rows share one barrier and hide one
// another's latencies.  Elements are read from shared memory twice, for the sums and for dx, so that they need no
// registers while the block waits for the sums.
constexpr int kRingThreads = 512;   // resident threads per SM of the backward kernels
template <class T, class W, int VEC, int G, int R>
__global__ void __launch_bounds__(G, kRingThreads / G > 0 ? kRingThreads / G : 1)
layer_norm_backward_ring_kernel(const T *dy, long lddy, const T *x, long ldx, const W *__restrict__ gamma,
                                const acc_t<T> *__restrict__ mean, const acc_t<T> *__restrict__ rstd, T *dx, long lddx,
                                acc_t<T> *partial, long rows, int cols, int stages, int *err) {
    using A = acc_t<T>;
    using P = SimdOf<T, VEC>;
    constexpr int CH = n_elems<T> / VEC, PV = VEC / kPack<VEC>;
    extern __shared__ __align__(16) unsigned char ring_raw[];
    __shared__ unsigned long long bars[kRingMax];
    __shared__ A buf[4 * R * (G / 32)];
    const int t = threadIdx.x, bytes = cols * (int)sizeof(T);
    const long apart = gridDim.x, step = apart * R;   // between a block's rows, between its groups of rows
    const A over = A(1) / (A)cols;
    int slot = 0, before = stages - 1;
    RowRing ring(ring_raw, bars, stages, 2 * R * bytes);
    ring.init();
    auto count = [&](long row) {   // rows of the group that starts at `row`
        return row >= rows ? 0 : R == 2 && row + apart < rows ? 2 : 1;
    };
    // groups are fetched `stages - 1` ahead: the stage of the group before this one is still being read
    if (t == 0)
        for (int i = 0; i + 1 < stages; ++i) {
            const long r = blockIdx.x + i * step;
            if (count(r)) ring.fill_pairs(i, x, ldx, dy, lddy, r, apart, count(r), bytes);
        }
    dx += t * VEC;
    const int left = cols - t * VEC;   // chunk c exists while c * G * VEC < left
    P dg[CH][PV], db[CH][PV];
    Vec<W, VEC> gm[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < PV; ++i) dg[c][i] = db[c][i] = P::splat(A(0));
#pragma unroll
        for (int e = 0; e < VEC; ++e) gm[c].v[e] = from_acc<W>(A(1));
        if (gamma && c * G * VEC < left) gm[c] = load_vec<W, VEC>(gamma + (c * G + t) * VEC);
    }
    A next_m[R], next_r[R];
    auto statistics = [&](long row) {
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (row + k * apart < rows) {
                next_m[k] = mean[row + k * apart];
                next_r[k] = rstd[row + k * apart];
            }
    };
    statistics(blockIdx.x);
    for (long row = blockIdx.x; row < rows; row += step) {
        const int n = count(row);
        A m[R], r[R], s[2 * R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            m[k] = next_m[k];
            r[k] = next_r[k];
            s[2 * k] = s[2 * k + 1] = 0;
        }
        statistics(row + step);   // travel meanwhile
        if (!ring.wait()) {
            if (t == 0) atomicExch(err, 1);
            return;
        }
        const T *in = (const T *)ring.data() + t * VEC;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (k < n) {
                const T *xs = in + 2 * k * cols, *ds = xs + cols;
                const P scale = P::splat(r[k]), shift = P::splat(-m[k] * r[k]);
                P a = P::splat(A(0)), b = a;
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (c * G * VEC < left) {
                        P xh[PV], d[PV], w[PV];
                        widen(load_vec<T, VEC>(xs + c * G * VEC), xh);
                        widen(load_vec<T, VEC>(ds + c * G * VEC), d);
                        widen(gm[c], w);
#pragma unroll
                        for (int i = 0; i < PV; ++i) {
                            xh[i] = fma(xh[i], scale, shift);
                            dg[c][i] = fma(d[i], xh[i], dg[c][i]);
                            db[c][i] = add(db[c][i], d[i]);
                            const P g = mul(d[i], w[i]);
                            a = add(a, g);
                            b = fma(g, xh[i], b);
                        }
                    }
                s[2 * k] = a.sum();
                s[2 * k + 1] = b.sum();
            }
        group_sums<G>(s, buf, slot);
        // past the sums' barrier no thread reads the stage of the group before this one
        if (t == 0) {
            const long ahead = row + (stages - 1) * step;
            if (count(ahead)) ring.fill_pairs(before, x, ldx, dy, lddy, ahead, apart, count(ahead), bytes);
        }
        before = ring.at;
        ring.advance();
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (k < n) {
                // dx = r (g - s1 - xh s2), s1 and s2 as means
                const T *xs = in + 2 * k * cols, *ds = xs + cols;
                T *to = dx + (row + k * apart) * lddx;
                const P scale = P::splat(r[k]), shift = P::splat(-m[k] * r[k]);
                const P back1 = P::splat(-s[2 * k] * over * r[k]), back2 = P::splat(-s[2 * k + 1] * over * r[k]);
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (c * G * VEC < left) {
                        P xh[PV], d[PV], w[PV];
                        widen(load_vec<T, VEC>(xs + c * G * VEC), xh);
                        widen(load_vec<T, VEC>(ds + c * G * VEC), d);
                        widen(gm[c], w);
#pragma unroll
                        for (int i = 0; i < PV; ++i)
                            d[i] = fma(fma(xh[i], scale, shift), back2, fma(mul(d[i], w[i]), scale, back1));
                        store_vec<T, VEC>(to + c * G * VEC, narrowed<T, VEC>(d));
                    }
            }
    }
    if (!partial) return;
    A *pg = partial + (long)blockIdx.x * 2 * cols + t * VEC, *pb = pg + cols;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (c * G * VEC < left) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                pg[c * G * VEC + e] = dg[c][e / kPack<VEC>].get(e % kPack<VEC>);
                pb[c * G * VEC + e] = db[c][e / kPack<VEC>].get(e % kPack<VEC>);
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
    wait_for_previous_kernel();
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

// Threads per row; 0: too long for registers.
int group_for(int cols, bool f64) {
    for (int g : {32, 128, 256, 512, 1024})
        if (cols <= g * (f64 ? n_elems<double> : N_ELEMS) && (!f64 || g <= max_group<double>)) return g;
    return 0;
}
int blocks_for(long rows, int g, int threads_per_sm) {
    const int threads = g > 32 ? g : 256;
    const long need = (rows + threads / g - 1) / (threads / g);
    const long room = (long)kLmSms * (threads_per_sm > threads ? threads_per_sm / threads : 1);
    return (int)(need < room ? need : room);
}
// Stages of a ring: as many rows as fit the block's share of 200 KB, at least 2 and at most 8 (0: too wide).
int ring_stages(int threads, int threads_per_sm, long bytes) {
    const int blocks = threads_per_sm / threads > 0 ? threads_per_sm / threads : 1;
    const long s = 200 * 1024 / blocks / bytes;
    return s < 2 ? 0 : s > kRingMax ? kRingMax : (int)s;
}
constexpr int kLongSplit = 64;           // row splits of the column sums of long rows
// Lets a kernel use `bytes` of dynamic shared memory (asked for once per device and thread while it is enough).
template <auto kernel> void allow_shared(const fitre_context *ctx, long bytes) {
    static thread_local int device = -1;
    static thread_local long allowed = 0;
    if (device == ctx->device && bytes <= allowed) return;
    FITRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    device = ctx->device;
    allowed = bytes;
}

template <class T, class W, int VEC, bool AFFINE>
void forward_with(fitre_context *ctx, const NormArgs &a) {
    using A = acc_t<T>;
    const int g = group_for(a.cols, sizeof(T) == 8);
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const W *gm = (const W *)a.gamma, *bt = (const W *)a.beta;
    A *mean = (A *)a.mean, *rstd = (A *)a.rstd;
    if (a.cols <= 32 * N_WIDE) {
#define NORM_LAUNCH(N)                                                                                        \
    layer_norm_warp_kernel<T, W, VEC, N, AFFINE><<<(unsigned)((a.rows + 7) / 8), 256, 0, ctx->stream>>>(     \
        x, a.ldx, gm, bt, y, a.ldy, mean, rstd, a.rows, a.cols, a.eps)
        if (a.cols <= 256) NORM_LAUNCH(8);
        else if (a.cols <= 512) NORM_LAUNCH(16);
        else NORM_LAUNCH(32);
#undef NORM_LAUNCH
        check_launch(ctx, "layer_norm_warp_kernel");
        return;
    }
    const int blocks = blocks_for(a.rows, g ? g : 1024, sizeof(T) == 8 ? 512 : 1024);
    const long bytes = (long)a.cols * sizeof(T);
    const int stages = VEC > 1 && g ? ring_stages(g, 1024, bytes) : 0;
    if constexpr (VEC > 1) if (stages) {
        const int room = blocks_for(a.rows, g, 1024);
#define NORM_LAUNCH(G)                                                                                       \
    allow_shared<layer_norm_ring_kernel<T, W, VEC, G, AFFINE>>(ctx, stages * bytes);                                      \
    layer_norm_ring_kernel<T, W, VEC, G, AFFINE><<<room, G, stages * bytes, ctx->stream>>>(                          \
        x, a.ldx, gm, bt, y, a.ldy, mean, rstd, a.rows, a.cols, a.eps, stages, (int *)(ctx->dscal + 4000))
        switch (g) {
            case 128: NORM_LAUNCH(128); break;
            case 256: NORM_LAUNCH(256); break;
            case 512: NORM_LAUNCH(512); break;
            default:
                if constexpr (max_group<T> >= 1024) { NORM_LAUNCH(1024); }
                break;
        }
#undef NORM_LAUNCH
        check_launch(ctx, "layer_norm_ring_kernel");
        return;
    }
#define NORM_LAUNCH(G)                                                                                       \
    layer_norm_kernel<T, W, VEC, G, AFFINE><<<blocks, G, 0, ctx->stream>>>(                          \
        x, a.ldx, gm, bt, y, a.ldy, mean, rstd, a.rows, a.cols, a.eps)
    switch (g) {
        case 128: NORM_LAUNCH(128); break;
        case 256: NORM_LAUNCH(256); break;
        case 512: NORM_LAUNCH(512); break;
        case 1024:
            if constexpr (max_group<T> >= 1024) NORM_LAUNCH(1024);
            break;
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
void forward_as(fitre_context *ctx, const NormArgs &a) {
    a.gamma && a.beta ? forward_with<T, W, VEC, true>(ctx, a) : forward_with<T, W, VEC, false>(ctx, a);
}

template <class T, class W, int VEC>
void backward_as(fitre_context *ctx, const NormArgs &a) {
    using A = acc_t<T>;
    const int g = group_for(a.cols, sizeof(T) == 8);
    const T *x = (const T *)a.x, *dy = (const T *)a.dy;
    T *dx = (T *)a.dx;
    const W *gm = (const W *)a.gamma;
    const A *mean = (const A *)a.mean, *rstd = (const A *)a.rstd;
    A *partial = a.dgamma || a.dbeta ? (A *)a.scratch : nullptr;
    int blocks = blocks_for(a.rows, g ? g : 1024, kRingThreads);
    const long bytes = 2l * a.cols * sizeof(T);
    // two rows at a time where three stages of them fit (not in rows above 8192 elements), else one
    const int two = VEC > 1 && g > 32 && g < 1024 ? ring_stages(g, kRingThreads, 2 * bytes) : 0;
    const int stages = two >= 3 ? two : VEC > 1 && g > 32 ? ring_stages(g, kRingThreads, bytes) : 0;
    if constexpr (VEC > 1) if (stages) {
        blocks = blocks_for(a.rows, g, kRingThreads);
#define NORM_LAUNCH(G, R)                                                                                    \
    do {                                                                                                     \
        allow_shared<layer_norm_backward_ring_kernel<T, W, VEC, G, R>>(ctx, stages * R * bytes);                  \
        layer_norm_backward_ring_kernel<T, W, VEC, G, R><<<blocks, G, stages * R * bytes, ctx->stream>>>(    \
            dy, a.lddy, x, a.ldx, gm, mean, rstd, dx, a.lddx, partial, a.rows, a.cols, stages,               \
            (int *)(ctx->dscal + 4000));                                                                     \
    } while (0)
        if (two >= 3) {
            if (g == 128) NORM_LAUNCH(128, 2);
            else if (g == 256) NORM_LAUNCH(256, 2);
            else NORM_LAUNCH(512, 2);
        } else {
            if (g == 128) NORM_LAUNCH(128, 1);
            else if (g == 256) NORM_LAUNCH(256, 1);
            else if (g == 512) NORM_LAUNCH(512, 1);
            else if constexpr (max_group<T> >= 1024) NORM_LAUNCH(1024, 1);
        }
#undef NORM_LAUNCH
        check_launch(ctx, "layer_norm_backward_ring_kernel");
    }
    if (!stages) {
#define NORM_LAUNCH(G)                                                                                       \
    layer_norm_backward_kernel<T, W, VEC, G><<<blocks, norm_threads<G>, 0, ctx->stream>>>(                 \
        dy, a.lddy, x, a.ldx, gm, mean, rstd, dx, a.lddx, partial, a.rows, a.cols)
    switch (g) {
        case 32: NORM_LAUNCH(32); break;
        case 128: NORM_LAUNCH(128); break;
        case 256: NORM_LAUNCH(256); break;
        case 512: NORM_LAUNCH(512); break;
        case 1024:
            if constexpr (max_group<T> >= 1024) NORM_LAUNCH(1024);
            break;
        default: {
            if (partial) {   // before dx, which may overwrite dy or x
                const int split = (int)(a.rows < kLongSplit ? a.rows : kLongSplit);
                layer_norm_columns_kernel<T><<<dim3((a.cols + 255) / 256, split), 256, 0, ctx->stream>>>(
                    dy, a.lddy, x, a.ldx, mean, rstd, partial, a.rows, a.cols);
                check_launch(ctx, "layer_norm_columns_kernel");
                launch_after(ctx->stream, layer_norm_reduce_kernel<W, A>, dim3((2 * a.cols + 31) / 32), 1024, partial, split,
                             a.cols, (W *)a.dgamma, (W *)a.dbeta);
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
    }
    if (partial) {
        launch_after(ctx->stream, layer_norm_reduce_kernel<W, A>, dim3((2 * a.cols + 31) / 32), 1024, partial, blocks, a.cols,
                     (W *)a.dgamma, (W *)a.dbeta);
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
    // the larger of what fp64 tensors and the others need
    long most = 0;
    for (const bool f64 : {false, true}) {
        const int g = cols <= 1024 * N_ELEMS ? group_for((int)cols, f64) : 0;
        const long parts = g ? blocks_for(rows, g, kRingThreads) : (rows < kLongSplit ? rows : kLongSplit);
        const long bytes = parts * 2 * cols * (f64 ? 8 : 4);
        most = bytes > most ? bytes : most;
    }
    return most;
}
void layer_norm_forward(fitre_context *ctx, const NormArgs &a) { norm_dispatch(ctx, a, false); }
void layer_norm_backward(fitre_context *ctx, const NormArgs &a) { norm_dispatch(ctx, a, true); }

}  // namespace fitre
