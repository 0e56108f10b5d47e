// One or two accumulators at a time: pairs of fp32 values go through the packed fp32 instructions, which
// take one issue slot for two operations; fp64 and single elements fall back to scalar code with the
// same interface.
#pragma once

#include "lm_common.cuh"

namespace fitre {
namespace {

template <class A, int N> struct Simd;

template <class A> struct Simd<A, 1> {
    A v;
    static __device__ __forceinline__ Simd splat(A a) { return {a}; }
    __device__ __forceinline__ A sum() const { return v; }
    __device__ __forceinline__ A get(int) const { return v; }
};
template <class A> __device__ __forceinline__ Simd<A, 1> add(Simd<A, 1> a, Simd<A, 1> b) { return {a.v + b.v}; }
template <class A> __device__ __forceinline__ Simd<A, 1> mul(Simd<A, 1> a, Simd<A, 1> b) { return {a.v * b.v}; }
template <class A> __device__ __forceinline__ Simd<A, 1> fma(Simd<A, 1> a, Simd<A, 1> b, Simd<A, 1> c) {
    return {a.v * b.v + c.v};
}

template <> struct Simd<double, 2> {
    double a, b;
    static __device__ __forceinline__ Simd splat(double v) { return {v, v}; }
    static __device__ __forceinline__ Simd of(double x, double y) { return {x, y}; }
    __device__ __forceinline__ double sum() const { return a + b; }
    __device__ __forceinline__ double get(int i) const { return i ? b : a; }
};
__device__ __forceinline__ Simd<double, 2> add(Simd<double, 2> x, Simd<double, 2> y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Simd<double, 2> mul(Simd<double, 2> x, Simd<double, 2> y) { return {x.a * y.a, x.b * y.b}; }
__device__ __forceinline__ Simd<double, 2> fma(Simd<double, 2> x, Simd<double, 2> y, Simd<double, 2> z) {
    return {x.a * y.a + z.a, x.b * y.b + z.b};
}

template <> struct Simd<float, 2> {
    uint64_t v;
    static __device__ __forceinline__ Simd of(float a, float b) {
        Simd r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
        return r;
    }
    static __device__ __forceinline__ Simd splat(float a) { return of(a, a); }
    __device__ __forceinline__ void split(float &a, float &b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
    __device__ __forceinline__ float get(int i) const {
        float a, b;
        split(a, b);
        return i ? b : a;
    }
    __device__ __forceinline__ float sum() const {
        float a, b;
        split(a, b);
        return a + b;
    }
};
__device__ __forceinline__ Simd<float, 2> add(Simd<float, 2> a, Simd<float, 2> b) {
    Simd<float, 2> r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Simd<float, 2> mul(Simd<float, 2> a, Simd<float, 2> b) {
    Simd<float, 2> r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Simd<float, 2> fma(Simd<float, 2> a, Simd<float, 2> b, Simd<float, 2> c) {
    Simd<float, 2> r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// VEC loaded elements as accumulators, VEC / N at a time.
template <int VEC> constexpr int kPack = VEC > 1 ? 2 : 1;
template <class T, int VEC> using SimdOf = Simd<acc_t<T>, kPack<VEC>>;

template <class T> __device__ __forceinline__ void widen(const Vec<T, 1> &x, Simd<acc_t<T>, 1> (&o)[1]) {
    o[0].v = to_acc<acc_t<T>>(x.v[0]);
}
__device__ __forceinline__ void widen(const Vec<double, 2> &x, Simd<double, 2> (&o)[1]) { o[0] = {x.v[0], x.v[1]}; }
__device__ __forceinline__ void widen(const Vec<float, 4> &x, Simd<float, 2> (&o)[2]) {
    o[0] = Simd<float, 2>::of(x.v[0], x.v[1]);
    o[1] = Simd<float, 2>::of(x.v[2], x.v[3]);
}
__device__ __forceinline__ void widen(const Vec<float, 8> &x, Simd<float, 2> (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = Simd<float, 2>::of(x.v[2 * i], x.v[2 * i + 1]);
}
__device__ __forceinline__ void widen(const Vec<__nv_bfloat16, 8> &x, Simd<float, 2> (&o)[4]) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(x.v);   // a bf16 is the upper half of an fp32
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = Simd<float, 2>::of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void widen(const Vec<__half, 8> &x, Simd<float, 2> (&o)[4]) {
    const __half2 *w = reinterpret_cast<const __half2 *>(x.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(w[i]);
        o[i] = Simd<float, 2>::of(f.x, f.y);
    }
}

template <class T> __device__ __forceinline__ Vec<T, 1> narrow(const Simd<acc_t<T>, 1> (&a)[1], Vec<T, 1> *) {
    return {{from_acc<T>(a[0].v)}};
}
__device__ __forceinline__ Vec<double, 2> narrow(const Simd<double, 2> (&a)[1], Vec<double, 2> *) { return {{a[0].a, a[0].b}}; }
__device__ __forceinline__ Vec<float, 4> narrow(const Simd<float, 2> (&a)[2], Vec<float, 4> *) {
    Vec<float, 4> r;
    a[0].split(r.v[0], r.v[1]);
    a[1].split(r.v[2], r.v[3]);
    return r;
}
__device__ __forceinline__ Vec<__nv_bfloat16, 8> narrow(const Simd<float, 2> (&a)[4], Vec<__nv_bfloat16, 8> *) {
    Vec<__nv_bfloat16, 8> r;
    __nv_bfloat162 *w = reinterpret_cast<__nv_bfloat162 *>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x, y;
        a[i].split(x, y);
        w[i] = __floats2bfloat162_rn(x, y);
    }
    return r;
}
__device__ __forceinline__ Vec<__half, 8> narrow(const Simd<float, 2> (&a)[4], Vec<__half, 8> *) {
    Vec<__half, 8> r;
    __half2 *w = reinterpret_cast<__half2 *>(r.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x, y;
        a[i].split(x, y);
        w[i] = __floats2half2_rn(x, y);
    }
    return r;
}
template <class T, int VEC, int M> __device__ __forceinline__ Vec<T, VEC> narrowed(const Simd<acc_t<T>, kPack<VEC>> (&a)[M]) {
    return narrow(a, (Vec<T, VEC> *)nullptr);
}

}  // namespace
}  // namespace fitre
