// extern "C" surface of the language-model operators: argument checks, then the launches of
// lm_norm.cu, lm_logprobs.cu and lm_gemm.cu on the context's stream.  No call waits for the GPU.
#include <cmath>
#include <initializer_list>

#include "lm_common.cuh"

using namespace fitre;

namespace {

// Runs `f` on the context's device, gives the caller's device back, and turns every exception into
// a status.
template <class F>
int on_context(fitre_context *ctx, F &&f) {
    if (!ctx) return FITRE_ERR_BAD_ARG;
    int before = -1;
    int status = FITRE_OK;
    try {
        FITRE_CUDA(cudaGetDevice(&before));
        if (before != ctx->device) FITRE_CUDA(cudaSetDevice(ctx->device));
        f();
    } catch (const Error &e) {
        status = e.code;
        try { ctx->err = e.what(); } catch (...) {}
    } catch (const std::exception &e) {
        status = FITRE_ERR_CUDA;
        try { ctx->err = e.what(); } catch (...) {}
    } catch (...) {
        status = FITRE_ERR_CUDA;
    }
    if (before >= 0 && before != ctx->device) cudaSetDevice(before);
    return status;
}

void need(bool ok, const char *what) { FITRE_REQUIRE(ok, FITRE_ERR_BAD_ARG, what); }

void need_type(int dtype) {
    FITRE_REQUIRE(dtype == FITRE_DTYPE_F64 || dtype == FITRE_DTYPE_F32 || dtype == FITRE_DTYPE_BF16 ||
                      dtype == FITRE_DTYPE_F16,
                  FITRE_ERR_UNSUPPORTED, "unknown element type");
}
constexpr long kMaxElements = 1l << 40;   // bound of a matrix extent, so that byte offsets stay in 63 bits
// A matrix of rows x cols elements whose rows start `ld` elements apart.
void need_matrix(const void *p, long ld, long rows, long cols, int dtype, const char *what) {
    const std::string name(what);
    FITRE_REQUIRE(p != nullptr, FITRE_ERR_BAD_ARG, name + " is NULL");
    FITRE_REQUIRE((uintptr_t)p % dtype_bytes(dtype) == 0, FITRE_ERR_BAD_ARG, name + " is not aligned to its elements");
    FITRE_REQUIRE(rows <= 1 || ld >= cols, FITRE_ERR_BAD_ARG, name + ": rows overlap (stride below the width)");
    FITRE_REQUIRE(ld >= 0 && ld < kMaxElements && (rows <= 1 || ld <= kMaxElements / rows), FITRE_ERR_TOO_LARGE,
                  name + " spans too many elements");
}
void need_vector(const void *p, int dtype, const char *what) {
    const std::string name(what);
    FITRE_REQUIRE(!p || (uintptr_t)p % dtype_bytes(dtype) == 0, FITRE_ERR_BAD_ARG,
                  name + " is not aligned to its elements");
}
// statistics are fp64 next to fp64 tensors, else fp32
int stat_type(int dtype) { return dtype == FITRE_DTYPE_F64 ? FITRE_DTYPE_F64 : FITRE_DTYPE_F32; }
long as_doubles(long bytes) { return (bytes + 7) / 8; }

void need_norm_shape(int dtype, int wtype, long rows, long cols) {
    need_type(dtype);
    FITRE_REQUIRE(wtype == dtype || (wtype == FITRE_DTYPE_F32 && dtype != FITRE_DTYPE_F64), FITRE_ERR_UNSUPPORTED,
                  "layer norm: weights are of the tensor's type, or fp32 next to a 16-bit one");
    need(rows >= 0 && cols >= 1, "layer norm: rows >= 0 and cols >= 1");
    FITRE_REQUIRE(cols <= (1l << 28) && rows <= (1l << 40), FITRE_ERR_TOO_LARGE, "layer norm: too large");
}
void need_token_shape(int dtype, long rows, long vocab) {
    need_type(dtype);
    need(rows >= 0 && vocab >= 1, "token log probabilities: rows >= 0 and vocab >= 1");
    FITRE_REQUIRE(vocab <= (1l << 28) && rows <= (1l << 27), FITRE_ERR_TOO_LARGE,
                  "token log probabilities: at most 2^28 entries and 2^27 rows");
}

}  // namespace

extern "C" {

int fitre_layer_norm_forward(fitre_context *ctx, int dtype, int wtype, const void *x, long ldx, const void *gamma,
                             const void *beta, void *y, long ldy, void *mean, void *rstd, long rows, long cols,
                             real eps) {
    return on_context(ctx, [&] {
        need_norm_shape(dtype, wtype, rows, cols);
        need(std::isfinite(eps) && eps >= 0, "layer norm: eps must be finite and not negative");
        if (rows == 0) return;
        need_matrix(x, ldx, rows, cols, dtype, "x");
        need_matrix(y, ldy, rows, cols, dtype, "y");
        need_vector(gamma, wtype, "gamma");
        need_vector(beta, wtype, "beta");
        need_vector(mean, stat_type(dtype), "mean");
        need_vector(rstd, stat_type(dtype), "rstd");
        NormArgs a = {};
        a.dtype = dtype, a.wtype = wtype, a.x = x, a.ldx = ldx, a.gamma = gamma, a.beta = beta, a.y = y, a.ldy = ldy;
        a.mean = mean, a.rstd = rstd, a.rows = rows, a.cols = (int)cols, a.eps = eps;
        layer_norm_forward(ctx, a);
    });
}

long fitre_layer_norm_backward_mem_required(long rows, long cols) {
    if (rows <= 0 || cols <= 0 || cols > (1l << 28)) return 0;
    return as_doubles(layer_norm_backward_scratch(rows, cols));
}

int fitre_layer_norm_backward(fitre_context *ctx, int dtype, int wtype, const void *dy, long lddy, const void *x,
                              long ldx, const void *gamma, const void *mean, const void *rstd, void *dx, long lddx,
                              void *dgamma, void *dbeta, long rows, long cols, real *devPtr) {
    return on_context(ctx, [&] {
        need_norm_shape(dtype, wtype, rows, cols);
        need_vector(dgamma, wtype, "dgamma");
        need_vector(dbeta, wtype, "dbeta");
        if (rows == 0) {   // the sum over no rows
            if (dgamma) FITRE_CUDA(cudaMemsetAsync(dgamma, 0, cols * dtype_bytes(wtype), ctx->stream));
            if (dbeta) FITRE_CUDA(cudaMemsetAsync(dbeta, 0, cols * dtype_bytes(wtype), ctx->stream));
            return;
        }
        need_matrix(dy, lddy, rows, cols, dtype, "dy");
        need_matrix(x, ldx, rows, cols, dtype, "x");
        need_matrix(dx, lddx, rows, cols, dtype, "dx");
        need(mean && rstd, "layer norm backward: mean and rstd of the forward pass are needed");
        need_vector(gamma, wtype, "gamma");
        need_vector(mean, stat_type(dtype), "mean");
        need_vector(rstd, stat_type(dtype), "rstd");
        if (dgamma || dbeta) {
            need(devPtr && aligned16(devPtr), "layer norm backward: devPtr is NULL or not 16-byte aligned");
            require_scratch(ctx, fitre_layer_norm_backward_mem_required(rows, cols), "layer norm backward");
        }
        NormArgs a = {};
        a.dtype = dtype, a.wtype = wtype, a.dy = dy, a.lddy = lddy, a.x = x, a.ldx = ldx, a.gamma = gamma;
        a.mean = (void *)mean, a.rstd = (void *)rstd, a.dx = dx, a.lddx = lddx, a.dgamma = dgamma, a.dbeta = dbeta;
        a.rows = rows, a.cols = (int)cols, a.scratch = devPtr;
        layer_norm_backward(ctx, a);
    });
}

int fitre_token_logprobs(fitre_context *ctx, int dtype, const void *logits, long ld, const long long *tokens,
                         long rows, long vocab, void *logprobs, void *lse, void *entropy, int top,
                         void *topLogprobs, long long *topTokens) {
    return on_context(ctx, [&] {
        need_token_shape(dtype, rows, vocab);
        need(top >= 0 && top <= vocab, "token log probabilities: 0 <= top <= vocab");
        FITRE_REQUIRE(top <= kMaxTop, FITRE_ERR_TOO_LARGE, "token log probabilities: at most 32 alternatives");
        if (rows == 0) return;
        need_matrix(logits, ld, rows, vocab, dtype, "logits");
        need(!logprobs || tokens, "token log probabilities: tokens is NULL");
        need(logprobs || lse || entropy || top, "token log probabilities: no output asked for");
        need(!top || (topLogprobs && topTokens), "token log probabilities: top needs topLogprobs and topTokens");
        need((uintptr_t)tokens % 8 == 0 && (uintptr_t)topTokens % 8 == 0, "tokens are not aligned to 8 bytes");
        need_vector(logprobs, stat_type(dtype), "logprobs");
        need_vector(lse, stat_type(dtype), "lse");
        need_vector(entropy, stat_type(dtype), "entropy");
        need_vector(topLogprobs, stat_type(dtype), "topLogprobs");
        LogProbArgs a = {};
        a.dtype = dtype, a.logits = logits, a.ld = ld, a.tokens = tokens, a.rows = rows, a.vocab = (int)vocab;
        a.logprobs = logprobs, a.lse = lse, a.entropy = entropy, a.top = top, a.top_logprobs = topLogprobs;
        a.top_tokens = topTokens;
        token_logprobs(ctx, a);
    });
}

int fitre_token_logprobs_backward(fitre_context *ctx, int dtype, const void *logits, long ld, const long long *tokens,
                                  const void *lse, const void *entropy, const void *dLogprobs, const void *dEntropy,
                                  void *dLogits, long ldd, long rows, long vocab) {
    return on_context(ctx, [&] {
        need_token_shape(dtype, rows, vocab);
        if (rows == 0) return;
        need_matrix(logits, ld, rows, vocab, dtype, "logits");
        need_matrix(dLogits, ldd, rows, vocab, dtype, "dLogits");
        need(lse != nullptr, "token log probabilities backward: lse of the forward pass is needed");
        need(dLogprobs || dEntropy, "token log probabilities backward: no incoming gradient");
        need(!dLogprobs || (tokens && (uintptr_t)tokens % 8 == 0), "tokens is NULL or not aligned to 8 bytes");
        need(!dEntropy || entropy, "token log probabilities backward: dEntropy needs the forward pass's entropy");
        for (const void *p : {lse, entropy, dLogprobs, dEntropy}) need_vector(p, stat_type(dtype), "a row vector");
        LogProbArgs a = {};
        a.dtype = dtype, a.logits = logits, a.ld = ld, a.tokens = tokens, a.rows = rows, a.vocab = (int)vocab;
        a.lse = (void *)lse, a.entropy = (void *)entropy, a.dlogprobs = dLogprobs, a.dentropy = dEntropy;
        a.dlogits = dLogits, a.ldd = ldd;
        token_logprobs_backward(ctx, a);
    });
}

}  // extern "C"
