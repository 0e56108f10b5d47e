// Declarations shared by the language-model operators (layer norm, token log probabilities, gated
// feed-forward block, orthogonalised update): element types, wide loads, conversions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace fitre {

// ---- host entry points of the operators (argument checks happen in lm_api.cpp) ----
struct NormArgs {
    int dtype, wtype;
    const void *x, *dy, *gamma, *beta;
    void *y, *mean, *rstd, *dx, *dgamma, *dbeta;
    long ldx, lddy, ldy, lddx, rows;
    int cols;
    double eps;
    void *scratch;
};
void layer_norm_forward(fitre_context *ctx, const NormArgs &a);
void layer_norm_backward(fitre_context *ctx, const NormArgs &a);
long layer_norm_backward_scratch(long rows, long cols);   // bytes

struct LogProbArgs {
    int dtype;
    const void *logits;
    const long long *tokens;
    void *logprobs, *lse, *entropy, *top_logprobs;
    long long *top_tokens;
    const void *dlogprobs, *dentropy;   // gradient pass: lse and entropy are inputs
    void *dlogits;
    long ld, ldd, rows;
    int vocab, top;
};
constexpr int kMaxTop = 32;   // alternatives per row: one per lane of a warp
void token_logprobs(fitre_context *ctx, const LogProbArgs &a);
void token_logprobs_backward(fitre_context *ctx, const LogProbArgs &a);

struct GatedArgs {
    int dtype, act;
    const void *x, *wg, *wu, *dh;
    void *h, *g, *u;                     // g and u: stored by the forward pass, read by the backward pass
    void *dx, *dwg, *dwu, *scratch;
    long ldx, ldwg, ldwu, lddh, ldh, ldg, ldu, lddx, lddwg, lddwu;
    long tokens, width, hidden;
};
void gated_forward(fitre_context *ctx, const GatedArgs &a);
void gated_backward(fitre_context *ctx, const GatedArgs &a);
long gated_forward_scratch(long tokens, long width, long hidden);    // bytes
long gated_backward_scratch(long tokens, long width, long hidden);
bool gated_rows_readable(const void *p, long ld);
bool gated_streams(long tokens);   // so few tokens that the forward pass reads its operands in any layout

struct OrthoArgs {
    int dtype, steps;
    const void *in;
    void *out, *scratch;
    long ldi, istride, ldo, ostride, batch, rows, cols;
    double coef[3], scale, eps;
};
void orthogonalize(fitre_context *ctx, const OrthoArgs &a);
long ortho_scratch(long batch, long rows, long cols);

constexpr int kLmSms = 148;   // streaming multiprocessors of a B200

namespace {

template <class T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };
template <class T> using acc_t = typename Acc<T>::type;

template <class A, class T> __device__ __forceinline__ A to_acc(T v) { return (A)v; }
template <> __device__ __forceinline__ float to_acc<float, __nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_acc<float, __half>(__half v) { return __half2float(v); }
template <class T, class A> __device__ __forceinline__ T from_acc(A v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16, float>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_acc<__half, float>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, moved with the widest load their size allows (16 bytes at most).
template <class T, int VEC> struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Vec { T v[VEC]; };

template <class T, int VEC> __device__ __forceinline__ Vec<T, VEC> load_vec(const T *p) {
    return *reinterpret_cast<const Vec<T, VEC> *>(p);
}
template <class T, int VEC> __device__ __forceinline__ void store_vec(T *p, const Vec<T, VEC> &v) {
    *reinterpret_cast<Vec<T, VEC> *>(p) = v;
}

// A kernel that follows another of this library in the same call may start while that one drains: it has to
// wait here before it touches memory.  Without the launch attribute (launch_after below) both are no-ops.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <class... P, class... A>
void launch_after(cudaStream_t stream, void (*kernel)(P...), dim3 grid, int threads, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    FITRE_CUDA(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline int dtype_bytes(int dtype) { return dtype == FITRE_DTYPE_F64 ? 8 : dtype == FITRE_DTYPE_F32 ? 4 : 2; }

}  // namespace
}  // namespace fitre
