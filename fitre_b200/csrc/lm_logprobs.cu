// Log probabilities of given tokens over rows of logits, with the entropy of each row's distribution
// and its largest alternatives, and the gradient with respect to the logits.
//   lse = log sum_j exp x_j,  lp = x_token - lse,  H = lse - sum_j p_j x_j,  p_j = exp(x_j - lse)
//   dx_j = gl (1[j = token] - p_j) - gH p_j (log p_j + H)
// Forward: bound by one read of the logits, next to which one exponential per element is all the
// special-function unit can do, so everything comes out of a single sweep: each thread keeps a
// reference r, s = sum exp(x - r) and t = sum exp(x - r)(x - r) (entropy = log s - t / s, free of the
// cancellation that large logits would bring).  r follows the running maximum lazily, when a value
// exceeds it by 10: sums of exponentials up to e^10 lose nothing in fp32, and rescaling becomes rare.
// The sweep runs on pairs (packed fp32 arithmetic, 16-bit packed maxima): 4.5 instructions per element
// instead of 8, which would be more than the issue slots one read of memory leaves.  An entry of
// -inf would put 0 * -inf into t; that is noticed per batch of loads, which is then done again with care.
// The alternatives need no second sweep either: the k-th largest of the threads' maxima is a
// lower bound of the k-th largest element, so only the vectors of the few threads whose maximum reaches
// it are read again (from L2) and filtered into lists that each warp keeps sorted across its lanes; lists
// are joined by ranking their entries in one another.
// Many short rows take a warp each instead of a block.
// With few rows a cluster of up to 16 blocks shares a row and joins its statistics and lists over
// distributed shared memory; no workspace, one launch.
// Backward: one read and one write of the logits, element by element.
// Measured on a B200 (6.5 TB/s copy): 4096 x 128000 bf16 without alternatives 165 us (6.4 TB/s), with 8 of them 196 to 215
// us (264 us without the packed sweep and the closer bound); 8 x 128000 with 20 of them 10 us; the gradient
// over 4099 x 50001 140 us (5.9 TB/s; 170 us with scalar arithmetic).
#include <cooperative_groups.h>

#include <cfloat>

#include "lm_common.cuh"
#include "lm_simd.cuh"

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
        e.i = 0x7fffffff;   // none: worse than any entry
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

// The largest value of a warp's lanes.
__device__ __forceinline__ float warp_max(float v) {
    // as integers in the same order: one reduction instruction instead of five exchanges
    const int i = __float_as_int(v);
    const int k = __reduce_max_sync(0xffffffffu, i ^ ((i >> 31) & 0x7fffffff));
    return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float exp2_fast(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// The largest element of a vector; NaN is passed over.
__device__ __forceinline__ float vec_max(const Vec<__nv_bfloat16, 8> &x) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(x.v);
    const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const Vec<__half, 8> &x) {
    const __half2 *p = reinterpret_cast<const __half2 *>(x.v);
    const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const Vec<float, 4> &x) {
    return fmaxf(fmaxf(x.v[0], x.v[1]), fmaxf(x.v[2], x.v[3]));
}
__device__ __forceinline__ double vec_max(const Vec<double, 2> &x) { return fmax(x.v[0], x.v[1]); }

constexpr float kLazy = 10.0f;   // how far values may exceed the reference before it follows

// A thread's statistics and its largest element.
template <class A> struct Running {
    Stats<A> st{Num<A>::lowest, 0, 0};
    A top = -Num<A>::inf();
    // before elements of which `m` is the largest
    __device__ __forceinline__ void follow(A m) {
        using N = Num<A>;
        top = N::max(top, m);
        if (m - st.m > A(kLazy)) {
            const A d = N::max_nan(st.m - m, N::floor), c = N::exp_(d);
            st.t = (st.t + d * st.s) * c;
            st.s *= c;
            st.m = m;
        }
    }
    __device__ __forceinline__ void element(A v) {   // with -inf, NaN and overflowing differences
        using N = Num<A>;
        const A d = N::max_nan(v - st.m, N::floor), p = N::exp_(d);
        st.s += p;
        st.t += p * d;
    }
    // `n` whole vectors; their largest element has been followed
    template <int n, class T, int VEC> __device__ __forceinline__ void vectors(const Vec<T, VEC> *x) {
        bool careful = true;
        if constexpr (sizeof(A) == 4) {
            using P = Simd<float, 2>;
            const P back = P::splat(-st.m), l2e = P::splat(1.4426950408889634f);
            P s = P::splat(0), t = s;
#pragma unroll
            for (int u = 0; u < n; ++u) {
                P v[VEC / 2];
                widen(x[u], v);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    const P d = add(v[i], back);
                    float a, b;
                    mul(d, l2e).split(a, b);
                    const P p = P::of(exp2_fast(a), exp2_fast(b));
                    s = add(s, p);
                    t = fma(p, d, t);
                }
            }
            const float tt = t.sum();
            careful = tt != tt;
            if (!careful) {
                st.s += s.sum();
                st.t += tt;
            }
        }
        if (careful) {
#pragma unroll
            for (int u = 0; u < n; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) element(to_acc<A>(x[u].v[e]));
        }
    }
};

constexpr int kNone = 0x7fffffff;   // place of an entry that is none
// Joins `count` sorted lists (kMaxTop entries each, a power of two of them) into the first, pairs at a time: the
// better of a[i] and b[31 - i] are the 32 best of both as a bitonic sequence, which five exchanges sort.
template <class A> __device__ __forceinline__ void merge_lists(Entry<A> *lists, int count) {
    const int lane = threadIdx.x & 31;
    for (int gap = 1; gap < count; gap *= 2) {
        for (int l = (threadIdx.x >> 5) * 2 * gap; l < count; l += (blockDim.x >> 5) * 2 * gap) {
            Entry<A> e = lists[l * kMaxTop + lane];
            const Entry<A> o = lists[(l + gap) * kMaxTop + 31 - lane];
            if (better(o.v, o.i, e.v, e.i)) e = o;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) {
                Entry<A> p;
                p.v = __shfl_xor_sync(0xffffffffu, e.v, x);
                p.i = __shfl_xor_sync(0xffffffffu, e.i, x);
                if (better(p.v, p.i, e.v, e.i) == ((lane & x) == 0)) e = p;
            }
            lists[l * kMaxTop + lane] = e;
        }
        __syncthreads();
    }
}

constexpr int L_UNROLL = 4;      // 16-byte loads a thread has in flight
constexpr int kMaxParts = 16;    // blocks that may share a row
constexpr int kRoom = 256;       // candidates a block can rank at once

// Resident threads per SM: the sweep fits 64 registers but for fp64, and for fp16, whose conversions take more (4096 x
// 128000 without alternatives: 197 us with 768 threads, 228 us with 1024).
template <class T> constexpr int sweep_threads = sizeof(T) == 8 ? 512 : std::is_same<T, __half>::value ? 768 : 1024;

template <class T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, sweep_threads<T> / THREADS)
token_logprobs_kernel(const T *__restrict__ logits, long ld, const long long *__restrict__ tokens, int vocab, int top,
                      acc_t<T> *logprobs, acc_t<T> *lse_out, acc_t<T> *entropy, acc_t<T> *top_logprobs,
                      long long *top_tokens) {
    using A = acc_t<T>;
    using N = Num<A>;
    constexpr int VEC = 16 / sizeof(T), WARPS = THREADS / 32;
    constexpr int LISTS = WARPS > kMaxParts ? WARPS : kMaxParts;
    __shared__ Stats<A> wstat[WARPS];
    __shared__ Stats<A> bstat;                     // this block's part of the row, read by the cluster
    constexpr int PICK = (kMaxTop + WARPS - 1) / WARPS + 1;   // maxima a warp may put forward
    __shared__ A picks[TOP ? WARPS * PICK : 1];
    __shared__ int hot[TOP ? THREADS : 1], hots, found;
    __shared__ Entry<A> room[TOP ? kRoom : 1], lists[TOP ? LISTS * kMaxTop : 1], blist[TOP ? kMaxTop : 1];
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

    // the given token's logit, fetched while the row is swept: two dependent loads that would end the row otherwise
    A given = 0;
    int state = 0;   // 1: the row has a token, -1: one out of range
    if (logprobs && part == 0 && tid == 0) {
        const long long tok = tokens[row];
        state = tok >= vocab ? -1 : tok >= 0 ? 1 : 0;
        if (state == 1) given = to_acc<A>(x[tok]);
    }

    Running<A> run;
    Vec<T, VEC> raw[2][L_UNROLL];
    int at = tid;
    auto load = [&](Vec<T, VEC> (&to)[L_UNROLL], int from) {
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u) to[u] = load_vec<T, VEC>(xv + (long)(from + u * THREADS) * VEC);
    };
    auto use = [&](const Vec<T, VEC> (&of)[L_UNROLL]) {
        A m = vec_max(of[0]);
#pragma unroll
        for (int u = 1; u < L_UNROLL; ++u) m = N::max(m, vec_max(of[u]));
        run.follow(m);
        run.template vectors<L_UNROLL>(of);
    };
    // whole batches, each one's loads issued before the arithmetic of the one before it
    const int batches = nvec / (THREADS * L_UNROLL);
    constexpr int STEP = THREADS * L_UNROLL;
    if (batches) load(raw[0], at);
    for (int b = 0; b < batches; b += 2) {
        if (b + 1 < batches) load(raw[1], at + STEP);
        use(raw[0]);
        if (b + 1 < batches) {
            if (b + 2 < batches) load(raw[0], at + 2 * STEP);
            use(raw[1]);
        }
        at += 2 * STEP;
    }
    at = tid + batches * STEP;
#pragma unroll
    for (int u = 0; u < L_UNROLL; ++u)
        if (at + u * THREADS < nvec) raw[0][u] = load_vec<T, VEC>(xv + (long)(at + u * THREADS) * VEC);
#pragma unroll
    for (int u = 0; u < L_UNROLL; ++u)
        if (at + u * THREADS < nvec) {
            run.follow(vec_max(raw[0][u]));
            run.template vectors<1>(&raw[0][u]);
        }
    if (tid < edges) {
        const A v = to_acc<A>(x[tid < head ? lo + tid : tail0 + (tid - head)]);
        run.follow(v);
        run.element(v);
    }
    // the warp's statistics: all lanes onto the largest reference, then plain sums
    Stats<A> st{warp_max(run.st.m), 0, 0};
    st = join(st, run.st);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
        st.t += __shfl_xor_sync(0xffffffffu, st.t, o);
    }
    if (lane == 0) wstat[warp] = st;
    if (TOP) {
        // each warp puts forward its largest maxima, one more than an even share of `top`
        A best = run.top;
        const int pick = (top + WARPS - 1) / WARPS + 1;
        for (int q = 0; q < pick; ++q) {
            const A b = warp_max(best);
            const unsigned who = __ballot_sync(0xffffffffu, best == b);
            if (lane == __ffs(who) - 1) best = -N::inf();
            if (lane == 0) picks[warp * pick + q] = b;
        }
        if (tid == 0) hots = found = 0;
        if (tid < kMaxTop) blist[tid] = Entry<A>{-N::inf(), kNone};
    }
    __syncthreads();
    if (warp == WARPS - 1) {
        Stats<A> r{N::lowest, 0, 0};
        if (lane < WARPS) r = wstat[lane];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) {
            Stats<A> other;
            other.m = __shfl_xor_sync(0xffffffffu, r.m, o);
            other.s = __shfl_xor_sync(0xffffffffu, r.s, o);
            other.t = __shfl_xor_sync(0xffffffffu, r.t, o);
            r = (lane & o) ? join(other, r) : join(r, other);
        }
        if (lane == 0) bstat = r;
    }
    if (TOP) {
        // the bound: the top-th largest of what was put forward (every warp finds it for itself)
        const int n = WARPS * ((top + WARPS - 1) / WARPS + 1);
        A bound = -N::inf();
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            const A v = i < n ? picks[i] : -N::inf();
            int rank = i < n ? 0 : n;
            for (int o = 0; o < n; ++o) rank += better(picks[o], o, v, i) ? 1 : 0;
            const unsigned who = __ballot_sync(0xffffffffu, rank == top - 1);
            if (who) bound = __shfl_sync(0xffffffffu, v, __ffs(who) - 1);
        }
        if (run.top >= bound) hot[atomicAdd(&hots, 1)] = tid;   // any order: entries are ranked by value and place
        const bool edge = tid < edges;
        const int edge_at = tid < head ? lo + tid : tail0 + (tid - head);
        A edge_v = edge ? to_acc<A>(x[edge_at]) : -N::inf();
        if (edge_v != edge_v) edge_v = -N::inf();               // a NaN ranks as -inf
        if (edge && edge_v >= bound) room[atomicAdd(&found, 1)] = Entry<A>{edge_v, edge_at};
        __syncthreads();
        // the hot threads' vectors: up to 32 of one thread's, or all of several threads', per warp and step
        const int rounds = (nvec + THREADS - 1) / THREADS, hotn = hots;
        const int wide = rounds >= 32 ? 5 : 32 - __clz(rounds > 1 ? rounds - 1 : 0);   // lanes per thread: 2^wide
        auto each = [&](auto &&use) {
            for (int h0 = warp << (5 - wide); h0 < hotn; h0 += WARPS << (5 - wide)) {
                const int h = h0 + (lane >> wide);
                const int owner = h < hotn ? hot[h] : nvec;
                for (int j0 = 0; j0 < rounds; j0 += 2 << wide) {
                    Vec<T, VEC> raw[2];
                    int vec[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        vec[k] = owner + (j0 + (k << wide) + (lane & ((1 << wide) - 1))) * THREADS;
                        if (vec[k] < nvec) raw[k] = load_vec<T, VEC>(xv + (long)vec[k] * VEC);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const bool worth = vec[k] < nvec && (vec_max(raw[k]) >= bound || bound == -N::inf());
                        if (__any_sync(0xffffffffu, worth))
#pragma unroll
                            for (int e = 0; e < VEC; ++e) {
                                A v = worth ? to_acc<A>(raw[k].v[e]) : -N::inf();
                                if (v != v) v = -N::inf();
                                use(worth && v >= bound, v, vbase + vec[k] * VEC + e);
                            }
                    }
                }
            }
        };
        each([&](bool has, A v, int i) {
            if (has) {
                const int at = atomicAdd(&found, 1);
                if (at < kRoom) room[at] = Entry<A>{v, i};
            }
        });
        __syncthreads();
        if (found <= kRoom) {
            for (int i = tid; i < found; i += THREADS) {
                const Entry<A> e = room[i];
                int rank = 0;
                for (int o = 0; o < found; ++o) rank += better(room[o].v, room[o].i, e.v, e.i) ? 1 : 0;
                if (rank < top) blist[rank] = e;
            }
        } else {
            // too many equal values: sorted lists
            WarpList<A> list(top, lane);
            if (warp == 0) list.offer(edge && edge_v >= bound, edge_v, edge_at);
            each([&](bool has, A v, int i) { list.offer(has, v, i); });
            lists[warp * kMaxTop + lane] = lane < top ? list.e : Entry<A>{-N::inf(), kNone};
            __syncthreads();
            merge_lists(lists, WARPS);
            if (tid < top) blist[tid] = lists[tid];
        }
    }
    if (parts > 1) cluster.sync();
    else __syncthreads();
    if (part == 0) {
        const Entry<A> *final_list = blist;
        if (TOP && parts > 1) {
            for (int i = tid; i < parts * kMaxTop; i += THREADS)
                lists[i] = cluster.map_shared_rank(blist, i / kMaxTop)[i % kMaxTop];
            __syncthreads();
            merge_lists(lists, parts);
            final_list = lists;
        }
        if (warp == 0) {
            Stats<A> r{N::lowest, 0, 0};
            if (lane < parts) r = *cluster.map_shared_rank(&bstat, lane);
#pragma unroll
            for (int o = kMaxParts / 2; o > 0; o >>= 1) {
                Stats<A> other;
                other.m = __shfl_xor_sync(0xffffffffu, r.m, o);
                other.s = __shfl_xor_sync(0xffffffffu, r.s, o);
                other.t = __shfl_xor_sync(0xffffffffu, r.t, o);
                r = (lane & o) ? join(other, r) : join(r, other);
            }
            r.m = __shfl_sync(0xffffffffu, r.m, 0);
            r.s = __shfl_sync(0xffffffffu, r.s, 0);
            r.t = __shfl_sync(0xffffffffu, r.t, 0);
            const bool none = r.s == A(0);         // every logit is -inf: no distribution
            const A logs = N::log_(r.s);
            if (lane == 0) {
                if (lse_out) lse_out[row] = none ? -N::inf() : r.m + logs;
                if (entropy) entropy[row] = none ? A(0) : logs - r.t / r.s;
                if (logprobs) {
                    A lp = 0;
                    if (state < 0) lp = N::inf() - N::inf();
                    else if (state) lp = none ? -N::inf() : (given - r.m) - logs;
                    logprobs[row] = lp;
                }
            }
            if (TOP && lane < top) {
                const Entry<A> e = final_list[lane];
                top_tokens[row * top + lane] = e.i;
                top_logprobs[row * top + lane] = none ? -N::inf() : (e.v - r.m) - logs;
            }
        }
    }
    if (parts > 1) cluster.sync();                 // the other blocks' shared memory was read above
}

// Short rows: a warp per row, no barrier and no shared memory.  The same sweep; the lanes' maxima bound the alternatives.
template <class T, bool TOP>
__global__ void __launch_bounds__(256, sweep_threads<T> / 256)
token_logprobs_warp_kernel(const T *__restrict__ logits, long ld, const long long *__restrict__ tokens, long rows, int vocab,
                           int top, acc_t<T> *logprobs, acc_t<T> *lse_out, acc_t<T> *entropy, acc_t<T> *top_logprobs,
                           long long *top_tokens) {
    using A = acc_t<T>;
    using N = Num<A>;
    constexpr int VEC = 16 / sizeof(T), STEP = 32 * L_UNROLL;
    const int lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const T *x = logits + row * ld;
    int head = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T);
    head = head < vocab ? head : vocab;
    const int nvec = (vocab - head) / VEC, tail0 = head + nvec * VEC, edges = head + (vocab - tail0);
    const T *xv = x + head;
    A given = 0;
    int state = 0;   // 1: the row has a token, -1: one out of range
    if (logprobs && lane == 0) {
        const long long tok = tokens[row];
        state = tok >= vocab ? -1 : tok >= 0 ? 1 : 0;
        if (state == 1) given = to_acc<A>(x[tok]);
    }
    const int edge_at = lane < head ? lane : tail0 + (lane - head);
    A edge_v = -N::inf();
    if (lane < edges) edge_v = to_acc<A>(x[edge_at]);

    Running<A> run;
    int at = lane;
    for (; at - lane + STEP <= nvec; at += STEP) {
        Vec<T, VEC> raw[L_UNROLL];
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u) raw[u] = load_vec<T, VEC>(xv + (long)(at + u * 32) * VEC);
        A m = vec_max(raw[0]);
#pragma unroll
        for (int u = 1; u < L_UNROLL; ++u) m = N::max(m, vec_max(raw[u]));
        run.follow(m);
        run.template vectors<L_UNROLL>(raw);
    }
    {
        Vec<T, VEC> raw[L_UNROLL];
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u)
            if (at + u * 32 < nvec) raw[u] = load_vec<T, VEC>(xv + (long)(at + u * 32) * VEC);
#pragma unroll
        for (int u = 0; u < L_UNROLL; ++u)
            if (at + u * 32 < nvec) {
                run.follow(vec_max(raw[u]));
                run.template vectors<1>(&raw[u]);
            }
    }
    if (lane < edges) {
        run.follow(edge_v);
        run.element(edge_v);
    }
    Stats<A> r{warp_max(run.st.m), 0, 0};
    r = join(r, run.st);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.t += __shfl_xor_sync(0xffffffffu, r.t, o);
    }
    const bool none = r.s == A(0);                 // every logit is -inf: no distribution
    const A logs = N::log_(r.s);
    if (lane == 0) {
        if (lse_out) lse_out[row] = none ? -N::inf() : r.m + logs;
        if (entropy) entropy[row] = none ? A(0) : logs - r.t / r.s;
        if (logprobs) {
            A lp = 0;
            if (state < 0) lp = N::inf() - N::inf();
            else if (state) lp = none ? -N::inf() : (given - r.m) - logs;
            logprobs[row] = lp;
        }
    }
    if (TOP) {
        int rank = 0;
        for (int o = 0; o < 32; ++o) rank += better(__shfl_sync(0xffffffffu, run.top, o), o, run.top, lane) ? 1 : 0;
        const A bound = __shfl_sync(0xffffffffu, run.top, __ffs(__ballot_sync(0xffffffffu, rank == top - 1)) - 1);
        WarpList<A> list(top, lane);
        if (edge_v != edge_v) edge_v = -N::inf();  // a NaN ranks as -inf
        list.offer(lane < edges && edge_v >= bound, edge_v, edge_at);
        for (int v0 = 0; v0 < nvec; v0 += 32) {
            Vec<T, VEC> raw;
            bool worth = v0 + lane < nvec && run.top >= bound;
            if (worth) {
                raw = load_vec<T, VEC>(xv + (long)(v0 + lane) * VEC);
                worth = vec_max(raw) >= bound || bound == -N::inf();
            }
            if (__any_sync(0xffffffffu, worth))
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    A v = worth ? to_acc<A>(raw.v[e]) : -N::inf();
                    if (v != v) v = -N::inf();
                    const bool has = worth && v >= bound;
                    if (__any_sync(0xffffffffu, has)) list.offer(has, v, head + (v0 + lane) * VEC + e);
                }
        }
        if (lane < top) {
            top_tokens[row * top + lane] = list.e.i;
            top_logprobs[row * top + lane] = none ? -N::inf() : (list.e.v - r.m) - logs;
        }
    }
}

template <class T, int THREADS, int VEC, int B_UNROLL>
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
    int head = VEC > 1 ? (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T) : 0;
    head = head < vocab ? head : vocab;
    const int nvec = (vocab - head) / VEC, tail0 = head + nvec * VEC, edges = head + (vocab - tail0);
    // the row's vectors in equal shares, none above THREADS * B_UNROLL
    const int share = (nvec + chunks - 1) / chunks, v0 = chunk * share + tid;
    const int vend = chunk * share + share < nvec ? chunk * share + share : nvec;
    Vec<T, VEC> raw[B_UNROLL];
#pragma unroll
    for (int u = 0; u < B_UNROLL; ++u)
        if (v0 + u * THREADS < vend) raw[u] = load_vec<T, VEC>(x + head + (long)(v0 + u * THREADS) * VEC);
    const A z = lse[row];
    const bool none = z == -N::inf();
    const long long tok = dlogprobs ? tokens[row] : -1;
    A gl = dlogprobs && tok >= 0 ? dlogprobs[row] : A(0);
    if (tok >= vocab) gl = N::inf() - N::inf();
    const A gh = dentropy ? dentropy[row] : A(0), h = dentropy ? entropy[row] : A(0);
    const int hot = tok >= 0 && tok < vocab ? (int)tok : -1;
    // an element with care for -inf, NaN and the given token
    auto one = [&](A v, int at) {
        const A lp = N::max_nan(v - z, N::floor), p = N::exp_(lp);
        A g = -p * (gl + gh * (lp + h));
        if (p == A(0)) g = gl + gh != gl + gh ? gl + gh : A(0);   // nothing times an overflowing logarithm is nothing
        if (at == hot) g += gl;
        return none ? A(0) : g;
    };
    if (chunk == 0 && tid < edges) {
        const int at = tid < head ? tid : tail0 + (tid - head);
        dx[at] = from_acc<T>(one(to_acc<A>(x[at]), at));
    }
#pragma unroll
    for (int u = 0; u < B_UNROLL; ++u)
        if (v0 + u * THREADS < vend) {
            const int at = head + (v0 + u * THREADS) * VEC;
            Vec<T, VEC> o;
            bool careful = true;
            if constexpr (VEC > 1 && sizeof(A) == 4) {
                // pairs: -p (gl + gh (lp + h)) = p (c0 + c1 lp); a sum of the results tells whether one is no number
                using P = Simd<float, 2>;
                const P back = P::splat(-z), l2e = P::splat(1.4426950408889634f), c0 = P::splat(-(gl + gh * h)),
                        c1 = P::splat(-gh);
                P v[VEC / 2], seen = P::splat(0);
                widen(raw[u], v);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    const P lp = add(v[i], back);
                    float a, b;
                    mul(lp, l2e).split(a, b);
                    v[i] = mul(P::of(exp2_fast(a), exp2_fast(b)), fma(c1, lp, c0));
                    seen = add(seen, v[i]);
                }
                const float all = seen.sum();
                careful = all != all || (unsigned)(hot - at) < (unsigned)VEC;
                o = narrowed<T, VEC>(v);
            }
            if (careful) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) o.v[e] = from_acc<T>(one(to_acc<A>(raw[u].v[e]), at + e));
            }
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

template <class T, bool TOP>
void launch_short(fitre_context *ctx, const LogProbArgs &a) {
    using A = acc_t<T>;
    token_logprobs_warp_kernel<T, TOP><<<(unsigned)((a.rows + 7) / 8), 256, 0, ctx->stream>>>(
        (const T *)a.logits, a.ld, a.tokens, a.rows, a.vocab, a.top, (A *)a.logprobs, (A *)a.lse, (A *)a.entropy,
        (A *)a.top_logprobs, a.top_tokens);
    check_launch(ctx, "token_logprobs_warp_kernel");
}

// Blocks that share a row: more while the rows alone leave SMs idle, but no slice under 4096 logits.
int parts_for(long rows, int vocab) {
    int parts = 1;
    while (parts < kMaxParts && rows * parts < kLmSms && vocab / (2 * parts) >= 4096) parts *= 2;
    return parts;
}

// Whether a warp takes a row.  It does where rows are short and enough for 16 warps per SM: what a block spends on its start
// and its barriers is then more than the sweep (150000 x 2000 bf16 without alternatives 174 us, 452 us in blocks; 1000 x
// 8192 9 us either way).  Alternatives are inserted one by one, which blocks do better when rows are longer or there are
// many (top 8: 36621 x 8192 bf16 207 and 264 us, 18310 x 16384 251 and 194 us; top 32: 4000 x 1003 38 us either way).
bool short_rows(const LogProbArgs &a, long row_bytes) {
    return a.rows >= 16 * kLmSms && (a.top ? row_bytes <= 16384 && row_bytes * a.top <= 131072 : row_bytes <= 32768);
}

template <class T>
void logprobs_as(fitre_context *ctx, const LogProbArgs &a) {
    const long row_bytes = (long)a.vocab * sizeof(T);
    if (short_rows(a, row_bytes)) return a.top ? launch_short<T, true>(ctx, a) : launch_short<T, false>(ctx, a);
    const int parts = parts_for(a.rows, a.vocab);
    // 128 threads for short rows, and for longer ones that are more than 256-thread blocks fit the GPU: twice the rows in
    // flight hide the phases behind the sweep (bf16, top 8: 12500 x 32000 203 and 229 us, 6250 x 64000 173 and 175 us, 3125
    // x 128000 178 and 155 us; 300 x 50000 17 us either way)
    const bool narrow = a.vocab <= 4096 || (a.rows > 4 * kLmSms && row_bytes <= 112 * 1024);
    if (a.top) {
        narrow ? launch_logprobs<T, 128, true>(ctx, a, parts) : launch_logprobs<T, 256, true>(ctx, a, parts);
    } else {
        narrow ? launch_logprobs<T, 128, false>(ctx, a, parts) : launch_logprobs<T, 256, false>(ctx, a, parts);
    }
}

template <class T, int THREADS, int VEC, int B_UNROLL>
void launch_backward(fitre_context *ctx, const LogProbArgs &a) {
    using A = acc_t<T>;
    const int per = THREADS * B_UNROLL * VEC;
    const int chunks = (a.vocab + per - 1) / per;
    FITRE_REQUIRE(a.rows <= 0x7fffffffl / chunks, FITRE_ERR_TOO_LARGE, "token log probabilities: too many logits");
    token_logprobs_backward_kernel<T, THREADS, VEC, B_UNROLL><<<(unsigned)(a.rows * chunks), THREADS, 0, ctx->stream>>>(
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
    // small blocks: their shares come out full at more widths (bf16, 64 and 256 threads: 49962 x 4003 130 and 175 us, 19998 x
    // 10001 132 and 160 us, 1562 x 128000 126 and 128 us).  Single elements, 16 to a thread: 6250 x 32000 248 us, 343 us with 4
    // in blocks of 256.
    same ? launch_backward<T, 64, VEC, 4>(ctx, a) : launch_backward<T, 64, 1, 16>(ctx, a);
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
