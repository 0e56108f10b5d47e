// Log probabilities of given tokens over rows of logits, with the entropy of each row's distribution
// and its largest alternatives, and the gradient with respect to the logits.
//   lse = log sum_j exp x_j,  lp = x_token - lse,  H = lse - sum_j p_j x_j,  p_j = exp(x_j - lse)
//   dx_j = gl (1[j = token] - p_j) - gH p_j (log p_j + H)
// Forward: bound by one read of the logits, next to which one exponential per element is all the
// special-function unit can do, so everything comes out of a single sweep: each thread keeps the running
// maximum m, s = sum exp(x - m) and t = sum exp(x - m)(x - m) (entropy = log s - t / s, free of the
// cancellation that large logits would bring), rescaled only when a batch of loads raises its
// maximum.  The alternatives need no second sweep either: the k-th largest of the threads' maxima is a
// lower bound of the k-th largest element, so only the few threads whose maximum reaches it have their
// elements read again (from L2) and filtered into lists that a warp keeps sorted across its lanes.
// With few rows a cluster of up to 16 blocks shares a row and joins its statistics and lists over
// distributed shared memory; no workspace, no atomics, one launch.
// Backward: one read and one write of the logits, element by element.
#include <cooperative_groups.h>

#include <cfloat>

#include "lm_common.cuh"

namespace cg = cooperative_groups;

namespace fitre {
namespace {

template <class A> struct Num;
template <> struct Num<float> {
    static constexpr float lowest = -FLT_MAX, floor = -1e30f;
    static __device__ __forceinline__ float inf() { return __int_as_float(0x7f800000); }
    // maximum that keeps a NaN (the plain maximum would drop it and with it the row's warning)
    static __device__ __forceinline__ float max_nan(float a, float b) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
        return r;
    }
    static __device__ __forceinline__ float max(float a, float b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float exp_(float d) {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
        return r;
    }
    static __device__ __forceinline__ float log_(float v) { return logf(v); }
};
template <> struct Num<double> {
    static constexpr double lowest = -DBL_MAX, floor = -1e300;
    static __device__ __forceinline__ double inf() { return __longlong_as_double(0x7ff0000000000000ll); }
    static __device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : (a > b ? a : b); }
    static __device__ __forceinline__ double max(double a, double b) { return fmax(a, b); }
    static __device__ __forceinline__ double exp_(double d) { return exp(d); }
    static __device__ __forceinline__ double log_(double v) { return log(v); }
};

// Running statistics of a thread, a warp or a row.
template <class A> struct Stats { A m, s, t; };
template <class A> __device__ __forceinline__ Stats<A> join(const Stats<A> &a, const Stats<A> &b) {
    using N = Num<A>;
    Stats<A> r;
    r.m = N::max(a.m, b.m);
    const A da = N::max_nan(a.m - r.m, N::floor), db = N::max_nan(b.m - r.m, N::floor);
    const A ea = N::exp_(da), eb = N::exp_(db);
    r.s = a.s * ea + b.s * eb;
    r.t = (a.t + da * a.s) * ea + (b.t + db * b.s) * eb;
    return r;
}

// One alternative: larger value first, lower place first among equals.
template <class A> struct Entry { A v; int i; };
template <class A> __device__ __forceinline__ bool better(A v, int i, A w, int j) { return v > w || (v == w && i < j); }

// A warp's sorted list of the k best entries, lane r holding rank r.
template <class A> struct WarpList {
    Entry<A> e;
    int k, lane;
    __device__ __forceinline__ WarpList(int k_, int lane_) : k(k_), lane(lane_) {
        e.v = -Num<A>::inf();
        e.i = 0x7fffffff;
    }
    // every lane offers one entry (or none); called by the whole warp
    __device__ __forceinline__ void offer(bool has, A v, int i) {
        A wv = __shfl_sync(0xffffffffu, e.v, k - 1);
        int wi = __shfl_sync(0xffffffffu, e.i, k - 1);
        unsigned mask = __ballot_sync(0xffffffffu, has && better(v, i, wv, wi));
        while (mask) {
            const int src = __ffs(mask) - 1;
            const A nv = __shfl_sync(0xffffffffu, v, src);
            const int ni = __shfl_sync(0xffffffffu, i, src);
            const int pos = __popc(__ballot_sync(0xffffffffu, lane < k && better(e.v, e.i, nv, ni)));
            const A uv = __shfl_up_sync(0xffffffffu, e.v, 1);
            const int ui = __shfl_up_sync(0xffffffffu, e.i, 1);
            if (lane == pos) {
                e.v = nv;
                e.i = ni;
            } else if (lane > pos) {
                e.v = uv;
                e.i = ui;
            }
            wv = __shfl_sync(0xffffffffu, e.v, k - 1);
            wi = __shfl_sync(0xffffffffu, e.i, k - 1);
            if (lane == src) has = false;
            mask = __ballot_sync(0xffffffffu, has && better(v, i, wv, wi));
        }
    }
};

template <class A> __device__ __forceinline__ A warp_max(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Num<A>::max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

constexpr int L_UNROLL = 4;   // 16-byte loads a thread has in flight

template <class T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, (sizeof(T) == 8 ? 512 : 1024) / THREADS)
token_logprobs_kernel(const T *__restrict__ logits, long ld, const long long *__restrict__ tokens, int vocab, int top,
                      acc_t<T> *logprobs, acc_t<T> *lse_out, acc_t<T> *entropy, acc_t<T> *top_logprobs,
                      long long *top_tokens) {
    using A = acc_t<T>;
    using N = Num<A>;
    constexpr int VEC = 16 / sizeof(T), WARPS = THREADS / 32;
    __shared__ Stats<A> wstat[WARPS];
    __shared__ Stats<A> bstat;                     // this block's part of the row, read by the cluster
    __shared__ A tmax[TOP ? THREADS : 1];
    __shared__ A bound_s;
    __shared__ Entry<A> lists[TOP ? WARPS * kMaxTop : 1], blist[TOP ? kMaxTop : 1];
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const long row = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = logits + row * ld;
    // this block's slice of the row: a head up to the first 16-byte boundary, whole vectors, a tail
    const int lo = (int)((long)vocab * part / parts), hi = (int)((long)vocab * (part + 1) / parts);
    int head = (int)((16 - ((uintptr_t)(x + lo) & 15)) & 15) / (int)sizeof(T);
    head = head < hi - lo ? head : hi - lo;
    const int nvec = (hi - lo - head) / VEC;
    const int vbase = lo + head, tail0 = vbase + nvec * VEC;
    const int edges = head + (hi - tail0);         // fewer than 2 * VEC, at most 14
    const T *xv = x + vbase;

    Stats<A> st{N::lowest, 0, 0};
    if (tid < edges) {
        const int at = tid < head ? lo + tid : tail0 + (tid - head);
        const A v = to_acc<A>(x[at]);
        st.m = N::max(st.m, v);
        const A d = N::max_nan(v - st.m, N::floor);
        st.s = N::exp_(d);
        st.t = st.s * d;
    }
    for (int at = tid; at < nvec; at += THREADS * L_UNROLL) {
        Vec<T, VEC> raw[L_UNROLL];
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u)
            if (at + u * THREADS < nvec) raw[u] = load_vec<T, VEC>(xv + (long)(at + u * THREADS) * VEC);
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u)
            if (at + u * THREADS < nvec) {
                A v[VEC], m = st.m;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    v[e] = to_acc<A>(raw[u].v[e]);
                    m = N::max(m, v[e]);
                }
                if (m > st.m) {
                    const A d = N::max_nan(st.m - m, N::floor), c = N::exp_(d);
                    st.t = (st.t + d * st.s) * c;
                    st.s *= c;
                    st.m = m;
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A d = N::max_nan(v[e] - st.m, N::floor), p = N::exp_(d);
                    st.s += p;
                    st.t += p * d;
                }
            }
    }
    const A mine = st.m > N::lowest ? st.m : -N::inf();   // a lower bound of this thread's maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stats<A> other;
        other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        other.t = __shfl_xor_sync(0xffffffffu, st.t, o);
        st = (lane & o) ? join(other, st) : join(st, other);
    }
    if (lane == 0) wstat[warp] = st;
    if (TOP) tmax[tid] = mine;
    __syncthreads();
    if (tid == 0) {
        Stats<A> r = wstat[0];
        for (int w = 1; w < WARPS; ++w) r = join(r, wstat[w]);
        bstat = r;
    }
    if (TOP) {
        if (warp == WARPS - 1) {
            // the top-th largest of the threads' maxima, by taking the maximum out `top` times
            A v[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v[w] = tmax[w * 32 + lane];
            A b = -N::inf();
            for (int r = 0; r < top; ++r) {
                A best = v[0];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) best = N::max(best, v[w]);
                b = warp_max(best);
                const unsigned who = __ballot_sync(0xffffffffu, best == b);
                if (lane == __ffs(who) - 1) {
                    bool out = false;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w)
                        if (!out && v[w] == b) {
                            v[w] = -N::inf();
                            out = true;
                        }
                }
            }
            if (lane == 0) bound_s = b;
        }
        __syncthreads();
        const A bound = bound_s;
        WarpList<A> list(top, lane);
        if (warp == 0) {
            const bool has = lane < edges;
            const int at = lane < head ? lo + lane : tail0 + (lane - head);
            A v = has ? to_acc<A>(x[at]) : -N::inf();
            if (v != v) v = -N::inf();             // a NaN ranks as -inf
            list.offer(has && v >= bound, v, at);
        }
        int turn = 0;
        for (int w = 0; w < WARPS; ++w) {
            // threads of warp w whose maximum reaches the bound, dealt out to the warps
            unsigned hot = __ballot_sync(0xffffffffu, tmax[w * 32 + lane] >= bound);
            for (; hot; hot &= hot - 1) {
                if (turn++ % WARPS != warp) continue;
                const int owner = w * 32 + __ffs(hot) - 1;
                for (int j0 = 0; owner + j0 * THREADS < nvec; j0 += 32) {
                    const int at = owner + (j0 + lane) * THREADS;
                    const bool in = at < nvec;
                    Vec<T, VEC> raw;
                    if (in) raw = load_vec<T, VEC>(xv + (long)at * VEC);
                    A v[VEC];
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        v[e] = in ? to_acc<A>(raw.v[e]) : -N::inf();
                        if (v[e] != v[e]) v[e] = -N::inf();
                        any = any || (in && v[e] >= bound);
                    }
                    if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) list.offer(in && v[e] >= bound, v[e], vbase + at * VEC + e);
                    }
                }
            }
        }
        if (lane < top) lists[warp * kMaxTop + lane] = list.e;
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < WARPS; ++w) {
                const Entry<A> o = lists[w * kMaxTop + lane];
                list.offer(lane < top && o.i != 0x7fffffff, o.v, o.i);
            }
            if (lane < top) blist[lane] = list.e;
        }
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    if (part == 0 && warp == 0) {
        Stats<A> r = bstat;
        for (int p = 1; p < parts; ++p) r = join(r, *cluster.map_shared_rank(&bstat, p));
        const bool none = r.s == A(0);             // every logit is -inf: no distribution
        const A logs = N::log_(r.s);
        const A lse = none ? -N::inf() : r.m + logs;
        if (lane == 0) {
            if (lse_out) lse_out[row] = lse;
            if (entropy) entropy[row] = none ? A(0) : logs - r.t / r.s;
            if (logprobs) {
                const long long tok = tokens[row];
                A lp = 0;
                if (tok >= vocab) lp = N::inf() - N::inf();
                else if (tok >= 0) lp = none ? -N::inf() : (to_acc<A>(x[tok]) - r.m) - logs;
                logprobs[row] = lp;
            }
        }
        if (TOP) {
            WarpList<A> list(top, lane);
            if (lane < top) list.e = blist[lane];
            for (int p = 1; p < parts; ++p) {
                Entry<A> o{-N::inf(), 0x7fffffff};
                if (lane < top) o = cluster.map_shared_rank(blist, p)[lane];
                list.offer(o.i != 0x7fffffff, o.v, o.i);
            }
            if (lane < top) {
                top_tokens[row * top + lane] = list.e.i;
                top_logprobs[row * top + lane] = none ? -N::inf() : (list.e.v - r.m) - logs;
            }
        }
    }
    if (parts > 1) cluster.sync();                 // the other blocks' shared memory was read above
}

constexpr int B_UNROLL = 4;

template <class T, int THREADS, int VEC>
__global__ void __launch_bounds__(THREADS)
token_logprobs_backward_kernel(const T *logits, long ld, const long long *__restrict__ tokens,
                               const acc_t<T> *__restrict__ lse, const acc_t<T> *__restrict__ entropy,
                               const acc_t<T> *__restrict__ dlogprobs, const acc_t<T> *__restrict__ dentropy, T *dlogits,
                               long ldd, int vocab, int chunks) {
    using A = acc_t<T>;
    using N = Num<A>;
    const long row = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x - row * chunks), tid = threadIdx.x;
    const T *x = logits + row * ld;
    T *dx = dlogits + row * ldd;
    const A z = lse[row];
    const bool none = z == -N::inf();
    const long long tok = dlogprobs ? tokens[row] : -1;
    A gl = dlogprobs && tok >= 0 ? dlogprobs[row] : A(0);
    if (tok >= vocab) gl = N::inf() - N::inf();
    const A gh = dentropy ? dentropy[row] : A(0), h = dentropy ? entropy[row] : A(0);
    const int hot = tok >= 0 && tok < vocab ? (int)tok : -1;
    auto one = [&](A v, int at) {
        const A lp = N::max_nan(v - z, N::floor), p = N::exp_(lp);
        A g = -p * (gl + gh * (lp + h));
        if (p == A(0)) g = gl != gl ? gl : A(0);   // nothing times an overflowing logarithm is nothing
        if (at == hot) g += gl;
        return none ? A(0) : g;
    };
    int head = VEC > 1 ? (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T) : 0;
    head = head < vocab ? head : vocab;
    const int nvec = (vocab - head) / VEC, tail0 = head + nvec * VEC, edges = head + (vocab - tail0);
    if (chunk == 0 && tid < edges) {
        const int at = tid < head ? tid : tail0 + (tid - head);
        dx[at] = from_acc<T>(one(to_acc<A>(x[at]), at));
    }
    const int v0 = chunk * THREADS * B_UNROLL + tid;
    Vec<T, VEC> raw[B_UNROLL];
#pragma unroll
    for (int u = 0; u < B_UNROLL; ++u)
        if (v0 + u * THREADS < nvec) raw[u] = load_vec<T, VEC>(x + head + (long)(v0 + u * THREADS) * VEC);
#pragma unroll
    for (int u = 0; u < B_UNROLL; ++u)
        if (v0 + u * THREADS < nvec) {
            const int at = head + (v0 + u * THREADS) * VEC;
            Vec<T, VEC> o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o.v[e] = from_acc<T>(one(to_acc<A>(raw[u].v[e]), at + e));
            store_vec<T, VEC>(dx + at, o);
        }
}

template <class T, int THREADS, bool TOP>
void launch_logprobs(fitre_context *ctx, const LogProbArgs &a, int parts) {
    using A = acc_t<T>;
    auto kernel = token_logprobs_kernel<T, THREADS, TOP>;
    if (parts > 8) {
        static thread_local int ready = -1;   // a cluster beyond 8 blocks has to be allowed once per device
        if (ready != ctx->device) {
            FITRE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            ready = ctx->device;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FITRE_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const T *)a.logits, a.ld, a.tokens, a.vocab, a.top, (A *)a.logprobs,
                                  (A *)a.lse, (A *)a.entropy, (A *)a.top_logprobs, a.top_tokens));
    check_launch(ctx, "token_logprobs_kernel");
}

// Blocks that share a row: more while the rows alone leave SMs idle, but no slice under 4096 logits.
int parts_for(long rows, int vocab) {
    int parts = 1;
    while (parts < 16 && rows * parts < kLmSms && vocab / (2 * parts) >= 4096) parts *= 2;
    return parts;
}

template <class T>
void logprobs_as(fitre_context *ctx, const LogProbArgs &a) {
    const int parts = parts_for(a.rows, a.vocab);
    const bool narrow = a.vocab <= 4096;   // a short row keeps 64 threads busy, not 256
    if (a.top) {
        narrow ? launch_logprobs<T, 64, true>(ctx, a, parts) : launch_logprobs<T, 256, true>(ctx, a, parts);
    } else {
        narrow ? launch_logprobs<T, 64, false>(ctx, a, parts) : launch_logprobs<T, 256, false>(ctx, a, parts);
    }
}

template <class T, int THREADS, int VEC>
void launch_backward(fitre_context *ctx, const LogProbArgs &a) {
    using A = acc_t<T>;
    const int per = THREADS * B_UNROLL * VEC;
    const int chunks = (a.vocab + per - 1) / per;
    FITRE_REQUIRE(a.rows <= 0x7fffffffl / chunks, FITRE_ERR_TOO_LARGE, "token log probabilities: too many logits");
    token_logprobs_backward_kernel<T, THREADS, VEC><<<(unsigned)(a.rows * chunks), THREADS, 0, ctx->stream>>>(
        (const T *)a.logits, a.ld, a.tokens, (const A *)a.lse, (const A *)a.entropy, (const A *)a.dlogprobs,
        (const A *)a.dentropy, (T *)a.dlogits, a.ldd, a.vocab, chunks);
    check_launch(ctx, "token_logprobs_backward_kernel");
}

template <class T>
void backward_as(fitre_context *ctx, const LogProbArgs &a) {
    constexpr int VEC = 16 / sizeof(T);
    // vectors need every row of both matrices at the same distance from a 16-byte boundary
    const bool same = (((uintptr_t)a.logits ^ (uintptr_t)a.dlogits) & 15) == 0 &&
                      (a.rows == 1 || ((a.ld - a.ldd) * (long)sizeof(T)) % 16 == 0);
    const bool narrow = a.vocab <= 64 * B_UNROLL * VEC;
    if (same) {
        narrow ? launch_backward<T, 64, VEC>(ctx, a) : launch_backward<T, 256, VEC>(ctx, a);
    } else {
        narrow ? launch_backward<T, 64, 1>(ctx, a) : launch_backward<T, 256, 1>(ctx, a);
    }
}

}  // namespace

void token_logprobs(fitre_context *ctx, const LogProbArgs &a) {
    switch (a.dtype) {
        case FITRE_DTYPE_F64: return logprobs_as<double>(ctx, a);
        case FITRE_DTYPE_F32: return logprobs_as<float>(ctx, a);
        case FITRE_DTYPE_BF16: return logprobs_as<__nv_bfloat16>(ctx, a);
        default: return logprobs_as<__half>(ctx, a);
    }
}
void token_logprobs_backward(fitre_context *ctx, const LogProbArgs &a) {
    switch (a.dtype) {
        case FITRE_DTYPE_F64: return backward_as<double>(ctx, a);
        case FITRE_DTYPE_F32: return backward_as<float>(ctx, a);
        case FITRE_DTYPE_BF16: return backward_as<__nv_bfloat16>(ctx, a);
        default: return backward_as<__half>(ctx, a);
    }
}

}  // namespace fitre
