// Gated feed-forward block, both projections with the activation and the product in one kernel, and its
// backward pass.
//   g = x Wg', u = x Wu', h = act(g) u                         (x: T x D, Wg and Wu: F x D)
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu,  dWg = dg' x,  dWu = du' x
// Forward: one product whose B tile holds the gate's rows beside the up projection's, so that the two
// accumulators of an output element end up in the same thread's registers: act(g) u costs no memory
// traffic, and the pre-activations are stored only when a backward pass will want them.  Few tokens (a
// serving loop's single token) are bound by one read of the weights and go to a kernel that streams
// them past the tokens held in registers.
// Backward: dg and du are formed once (memory-bound, rounded to the tensors' type because the tensor
// core takes no wider operand next to 16-bit weights), then dx is one product over both halves of the
// concatenated inner dimension, and dWg / dWu one launch over both.
// All sums are fp32; each output is rounded once.
// Measured on a B200: 8192 x 4096 x 12288 bf16 with g and u stored 1089 us from a cool start (1515 TFLOP/s; cuBLAS 1029 us for
// the two projections without activation, product or their stores), 1240 us in a loop under the power cap;
// gradient at 4096 tokens 1187 / 1360 us; one token 37 us (5.4 TB/s of weights).
#include "lm_gemm.cuh"
#include "lm_simd.cuh"

namespace fitre {
namespace {

// 1 / (1 + exp(-g)) to 2^-21 by the fast exponential and reciprocal: outputs have 11 bits at most, and with exact
// division the epilogue would take longer than a short product.
__device__ __forceinline__ float sigmoid(float g) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
__device__ __forceinline__ float act_value(int act, float g) {
    switch (act) {
        case FITRE_CNN_ACT_SWISH: return g * sigmoid(g);
        case FITRE_CNN_ACT_RELU: return fmaxf(g, 0.0f);
        case FITRE_CNN_ACT_SOFTPLUS: return fmaxf(g, 0.0f) + log1pf(__expf(-fabsf(g)));
        default: return g;
    }
}
__device__ __forceinline__ float act_slope(int act, float g) {
    switch (act) {
        case FITRE_CNN_ACT_SWISH: {
            const float s = sigmoid(g);
            return s * (1.0f + g * (1.0f - s));
        }
        case FITRE_CNN_ACT_RELU: return g > 0.0f ? 1.0f : 0.0f;
        case FITRE_CNN_ACT_SOFTPLUS: return sigmoid(g);
        default: return 1.0f;
    }
}

template <class T>
struct GatedEpi {
    struct Params {
        Output<T> h, g, u;
        int act;
    };
    static constexpr bool kTwoMaps = true;
    template <int BN> static __device__ __forceinline__ void begin(const Params &, TileAt, int, Stager &) {}
    template <int BN>
    static __device__ __forceinline__ void store(const Params &p, TileAt at, int row0, uint32_t tmem, Stager &st) {
        // columns: the tile's gates, then as many ups
        const int width = at.half < 0 ? BN / 2 : BN / 4, first = at.n * (BN / 2) + (at.half > 0 ? BN / 4 : 0);
        if (row0 >= p.h.rows) return;
#pragma unroll 1
        for (int c = 0; c < width && first + c < p.h.cols; c += 64) {
            float g[64], u[64];
            st.sums(tmem, c, g);
            st.sums(tmem, width + c, u);
            if (p.g.out) st.put(p.g, row0, first + c, 0, g);
            if (p.u.out) st.put(p.u, row0, first + c, 0, u);
            if (p.act == FITRE_CNN_ACT_SWISH) {   // the choice once, not per element
#pragma unroll
                for (int i = 0; i < 64; ++i) u[i] *= act_value(FITRE_CNN_ACT_SWISH, g[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) u[i] *= act_value(p.act, g[i]);
            }
            st.put(p.h, row0, first + c, 0, u);
        }
    }
};

// Few tokens: a warp takes one hidden unit and streams its two weight rows.
constexpr int V_TOKENS = 4, V_THREADS = 128;   // small blocks: the last ones to finish are few
template <class T, int NT, int VEC>
__global__ void __launch_bounds__(V_THREADS)
gated_few_kernel(const T *__restrict__ x, long ldx, const T *__restrict__ wg, long ldwg, const T *__restrict__ wu,
                 long ldwu, T *h, long ldh, T *g_out, long ldg, T *u_out, long ldu, int D, int F, int act) {
    using P = SimdOf<T, VEC>;
    constexpr int PV = VEC / kPack<VEC>, DEEP = 4;   // loads of each weight row a lane has in flight
    const int lane = threadIdx.x & 31, f = (blockIdx.x * V_THREADS + threadIdx.x) / 32;
    if (f >= F) return;
    P gs[NT], us[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) gs[t] = us[t] = P::splat(0.0f);
    const T *pg = wg + (long)f * ldwg + lane * VEC, *pu = wu + (long)f * ldwu + lane * VEC;
    x += lane * VEC;
    const int left = D - lane * VEC;   // this lane's elements start at multiples of 32 VEC below it
    for (int d0 = 0; d0 < left; d0 += DEEP * 32 * VEC) {
        Vec<T, VEC> a[DEEP], b[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (d0 + i * 32 * VEC < left) {
                a[i] = load_vec<T, VEC>(pg + d0 + i * 32 * VEC);
                b[i] = load_vec<T, VEC>(pu + d0 + i * 32 * VEC);
            }
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (d0 + i * 32 * VEC < left) {
                P av[PV], bv[PV], xv[PV];
                widen(a[i], av);
                widen(b[i], bv);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    widen(load_vec<T, VEC>(x + t * ldx + d0 + i * 32 * VEC), xv);
#pragma unroll
                    for (int j = 0; j < PV; ++j) {
                        gs[t] = fma(av[j], xv[j], gs[t]);
                        us[t] = fma(bv[j], xv[j], us[t]);
                    }
                }
            }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float g = gs[t].sum(), u = us[t].sum();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            g += __shfl_xor_sync(0xffffffffu, g, o);
            u += __shfl_xor_sync(0xffffffffu, u, o);
        }
        if (lane == t) {
            if (g_out) g_out[t * ldg + f] = from_acc<T>(g);
            if (u_out) u_out[t * ldu + f] = from_acc<T>(u);
            h[t * ldh + f] = from_acc<T>(act_value(act, g) * u);
        }
    }
}

// dg and du, side by side in scratch ([2][T][ld], zeros beyond F).
template <class T, int VEC>
__global__ void __launch_bounds__(256)
gated_slopes_kernel(const T *dh, long lddh, const T *g, long ldg, const T *u, long ldu, T *out, long ld, long half,
                    int F, int act) {
    let_next_kernel_start();
    const long row = blockIdx.y;
    const int at = (blockIdx.x * 256 + threadIdx.x) * VEC;
    if (at >= F) {
        if (VEC < 8)
            for (int e = 0; e < VEC; ++e)
                if (at + e < ld) out[row * ld + at + e] = out[half + row * ld + at + e] = from_acc<T>(0.0f);
        return;
    }
    const Vec<T, VEC> a = load_vec<T, VEC>(dh + row * lddh + at), b = load_vec<T, VEC>(g + row * ldg + at),
                      c = load_vec<T, VEC>(u + row * ldu + at);
    Vec<T, VEC> dg, du;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const float d = to_acc<float>(a.v[e]), gv = to_acc<float>(b.v[e]);
        dg.v[e] = from_acc<T>(d * to_acc<float>(c.v[e]) * act_slope(act, gv));
        du.v[e] = from_acc<T>(d * act_value(act, gv));
    }
    store_vec<T, VEC>(out + row * ld + at, dg);
    store_vec<T, VEC>(out + half + row * ld + at, du);
}

// Matrices whose rows TMA cannot read, copied to rows that it can, padded with zeros: a warp per row.
template <class T> struct Copies {
    const T *in[3];
    T *out[3];
    long ld[3], rows[3];
};
template <class T>
__global__ void __launch_bounds__(256)
align_rows_kernel(Copies<T> k, int cols, int ldo) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const int lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const T *in = k.in[blockIdx.y];
    T *out = k.out[blockIdx.y];
    if (row >= k.rows[blockIdx.y]) return;
    in += row * k.ld[blockIdx.y];
    out += row * ldo;
#pragma unroll 4
    for (int c = lane; c < ldo; c += 32) out[c] = c < cols ? in[c] : from_acc<T>(0.0f);
}

long up8(long n) { return (n + 7) / 8 * 8; }
long up128(long bytes) { return (bytes + 127) / 128 * 128; }

// Scratch that the operands' copies take when `width` is no multiple of 8 (rows that start off the 16-byte grid).
long staged_bytes(long tokens, long width, long hidden) {
    if (width % 8 == 0) return 0;
    return up128(2 * tokens * up8(width)) + 2 * up128(2 * hidden * up8(width));
}

template <class T>
struct Operands {
    const T *x, *wg, *wu;
    long ldx, ldwg, ldwu;
};
// The operands as TMA can read them; `room` (bytes) advances past the copies made.
template <class T>
Operands<T> readable(fitre_context *ctx, const GatedArgs &a, char *&room) {
    Operands<T> o{(const T *)a.x, (const T *)a.wg, (const T *)a.wu, a.ldx, a.ldwg, a.ldwu};
    if (a.width % 8 == 0) return o;
    const long ld = up8(a.width);
    Copies<T> k = {{o.x, o.wg, o.wu}, {}, {a.ldx, a.ldwg, a.ldwu}, {a.tokens, a.hidden, a.hidden}};
    for (int i = 0; i < 3; ++i) {
        k.out[i] = (T *)room;
        room += up128(2 * k.rows[i] * ld);
    }
    const long most = a.tokens > a.hidden ? a.tokens : a.hidden;
    launch_after(ctx->stream, align_rows_kernel<T>, dim3((unsigned)((most + 7) / 8), 3), 256, k, (int)a.width, (int)ld);
    check_launch(ctx, "align_rows_kernel");
    o.x = k.out[0], o.wg = k.out[1], o.wu = k.out[2];
    o.ldx = o.ldwg = o.ldwu = ld;
    return o;
}

template <class T> constexpr int fmt_of = sizeof(T) && std::is_same<T, __half>::value ? G_F16 : G_BF16;

template <class T, int CG, int BN>
void forward_tiles(fitre_context *ctx, const GatedArgs &a, const Operands<T> &o) {
    GemmArgs<typename GatedEpi<T>::Params> g = {};
    const int T_ = (int)a.tokens, D = (int)up8(a.width), F = (int)a.hidden;
    gemm_operand(&g.a[0], false, o.x, T_, D, 1, o.ldx, 0, fmt_of<T>);
    gemm_operand(&g.b[0], false, o.wg, F, D, 1, o.ldwg, 0, fmt_of<T>, 64 * CG);
    gemm_operand(&g.b[1], false, o.wu, F, D, 1, o.ldwu, 0, fmt_of<T>, 64 * CG);
    g.epi.h = gemm_output<T>(a.h, F, T_, 1, a.ldh, 0, fmt_of<T>);
    g.epi.g = gemm_output<T>(a.g, F, T_, 1, a.ldg, 0, fmt_of<T>);
    g.epi.u = gemm_output<T>(a.u, F, T_, 1, a.ldu, 0, fmt_of<T>);
    g.epi.act = a.act;
    gemm_launch<CG, BN, false, false, GatedEpi<T>>(ctx, g, T_, F, 1, false, D, 1, fmt_of<T>, "gated_tiles_kernel", a.width % 8 != 0);
}

// Whether a product has tiles enough for the SM pairs' 256-row tiles; below, 128-row tiles on single SMs
// keep more of the GPU busy.
bool pairs_worth(long M, long N, int n_per_tile, int products) {
    return ((M + 255) / 256) * ((N + n_per_tile - 1) / n_per_tile) * products >= kLmSms / 2;
}

template <class T, int NT, int VEC>
void forward_few(fitre_context *ctx, const GatedArgs &a) {
    gated_few_kernel<T, NT, VEC><<<(unsigned)((a.hidden + V_THREADS / 32 - 1) / (V_THREADS / 32)), V_THREADS, 0, ctx->stream>>>(
        (const T *)a.x, a.ldx, (const T *)a.wg, a.ldwg, (const T *)a.wu, a.ldwu, (T *)a.h, a.ldh, (T *)a.g, a.ldg,
        (T *)a.u, a.ldu, (int)a.width, (int)a.hidden, a.act);
    check_launch(ctx, "gated_few_kernel");
}
template <class T, int VEC>
void forward_few_as(fitre_context *ctx, const GatedArgs &a) {
    switch (a.tokens) {
        case 1: return forward_few<T, 1, VEC>(ctx, a);
        case 2: return forward_few<T, 2, VEC>(ctx, a);
        case 3: return forward_few<T, 3, VEC>(ctx, a);
        default: return forward_few<T, 4, VEC>(ctx, a);
    }
}

template <class T>
void forward_as(fitre_context *ctx, const GatedArgs &a) {
    if (a.tokens <= V_TOKENS) {
        const bool wide = a.width % 8 == 0 && tma_readable(a.x, a.ldx) && tma_readable(a.wg, a.ldwg) &&
                          tma_readable(a.wu, a.ldwu);
        wide ? forward_few_as<T, 8>(ctx, a) : forward_few_as<T, 1>(ctx, a);
        return;
    }
    char *room = (char *)a.scratch;
    const Operands<T> o = readable<T>(ctx, a, room);
    if (pairs_worth(a.tokens, a.hidden, 128, 1)) forward_tiles<T, 2, 256>(ctx, a, o);
    else forward_tiles<T, 1, 128>(ctx, a, o);
}

template <class T, int CG, int BN>
void input_gradient(fitre_context *ctx, const GatedArgs &a, const Operands<T> &o, const T *slopes, long ld, long half) {
    GemmArgs<typename StoreEpi<T>::Params> g = {};
    const int T_ = (int)a.tokens, D = (int)a.width, F = (int)a.hidden;
    gemm_operand(&g.a[0], false, slopes, T_, ld, 1, ld, 0, fmt_of<T>);
    gemm_operand(&g.a[1], false, slopes + half, T_, ld, 1, ld, 0, fmt_of<T>);
    gemm_operand(&g.b[0], true, o.wg, up8(D), F, 1, o.ldwg, 0, fmt_of<T>);
    gemm_operand(&g.b[1], true, o.wu, up8(D), F, 1, o.ldwu, 0, fmt_of<T>);
    g.epi.out[0] = gemm_output<T>(a.dx, D, T_, 1, a.lddx, 0, fmt_of<T>);
    gemm_launch<CG, BN, false, true, StoreEpi<T>>(ctx, g, T_, D, 1, false, F, 2, fmt_of<T>, "gated_input_gradient_kernel", true);
}
template <class T, int CG, int BN>
void weight_gradient(fitre_context *ctx, const GatedArgs &a, const Operands<T> &o, const T *slopes, long ld, long half) {
    GemmArgs<typename StoreEpi<T>::Params> g = {};
    const int T_ = (int)a.tokens, D = (int)a.width, F = (int)a.hidden;
    gemm_operand(&g.a[0], true, slopes, ld, T_, 2, ld, half, fmt_of<T>);
    gemm_operand(&g.b[0], true, o.x, up8(D), T_, 1, o.ldx, 0, fmt_of<T>);
    g.g.za = 1;
    g.epi.out[0] = gemm_output<T>(a.dwg, D, F, 1, a.lddwg, 0, fmt_of<T>);
    g.epi.out[1] = gemm_output<T>(a.dwu, D, F, 1, a.lddwu, 0, fmt_of<T>);
    gemm_launch<CG, BN, true, true, StoreEpi<T>>(ctx, g, F, D, 2, false, T_, 1, fmt_of<T>, "gated_weight_gradient_kernel", true);
}

template <class T, int VEC>
void slopes_as(fitre_context *ctx, const GatedArgs &a, T *slopes, long ld, long half) {
    const long most = 65535;   // rows a grid's second dimension can count
    for (long r0 = 0; r0 < a.tokens; r0 += most) {
        const long n = a.tokens - r0 < most ? a.tokens - r0 : most;
        gated_slopes_kernel<T, VEC><<<dim3((unsigned)((ld + 256 * VEC - 1) / (256 * VEC)), (unsigned)n), 256, 0,
                                      ctx->stream>>>(
            (const T *)a.dh + r0 * a.lddh, a.lddh, (const T *)a.g + r0 * a.ldg, a.ldg, (const T *)a.u + r0 * a.ldu,
            a.ldu, slopes + r0 * ld, ld, half, (int)a.hidden, a.act);
        check_launch(ctx, "gated_slopes_kernel");
    }
}

template <class T>
void backward_as(fitre_context *ctx, const GatedArgs &a) {
    const long ld = up8(a.hidden), half = a.tokens * ld;
    T *slopes = (T *)a.scratch;
    char *room = (char *)a.scratch + up128(2 * 2 * half);
    const bool wide = a.hidden % 8 == 0 && tma_readable(a.dh, a.lddh) && tma_readable(a.g, a.ldg) && tma_readable(a.u, a.ldu);
    const bool even = a.hidden % 2 == 0 && ((uintptr_t)a.dh | (uintptr_t)a.g | (uintptr_t)a.u) % 4 == 0 &&
                      (a.lddh | a.ldg | a.ldu) % 2 == 0;
    if (wide) slopes_as<T, 8>(ctx, a, slopes, ld, half);
    else if (even) slopes_as<T, 2>(ctx, a, slopes, ld, half);
    else slopes_as<T, 1>(ctx, a, slopes, ld, half);
    const Operands<T> o = readable<T>(ctx, a, room);
    if (pairs_worth(a.tokens, a.width, 256, 1)) input_gradient<T, 2, 256>(ctx, a, o, slopes, ld, half);
    else input_gradient<T, 1, 128>(ctx, a, o, slopes, ld, half);
    if (pairs_worth(a.hidden, a.width, 256, 2)) weight_gradient<T, 2, 256>(ctx, a, o, slopes, ld, half);
    else weight_gradient<T, 1, 128>(ctx, a, o, slopes, ld, half);
}

}  // namespace

long gated_forward_scratch(long tokens, long width, long hidden) {
    return tokens <= V_TOKENS ? 0 : staged_bytes(tokens, width, hidden);
}
long gated_backward_scratch(long tokens, long width, long hidden) {
    return up128(2 * 2 * tokens * up8(hidden)) + staged_bytes(tokens, width, hidden);
}
bool gated_streams(long tokens) { return tokens <= V_TOKENS; }
bool gated_rows_readable(const void *p, long ld) { return tma_readable(p, ld); }
void gated_forward(fitre_context *ctx, const GatedArgs &a) {
    a.dtype == FITRE_DTYPE_BF16 ? forward_as<__nv_bfloat16>(ctx, a) : forward_as<__half>(ctx, a);
}
void gated_backward(fitre_context *ctx, const GatedArgs &a) {
    a.dtype == FITRE_DTYPE_BF16 ? backward_as<__nv_bfloat16>(ctx, a) : backward_as<__half>(ctx, a);
}

}  // namespace fitre
