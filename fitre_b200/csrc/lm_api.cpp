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
    FITRE_REQUIRE(cols <= (1l << 28) && rows <= (1l << 33), FITRE_ERR_TOO_LARGE,
                  "layer norm: at most 2^33 rows of 2^28 elements");
}
void need_token_shape(int dtype, long rows, long vocab) {
    need_type(dtype);
    need(rows >= 0 && vocab >= 1, "token log probabilities: rows >= 0 and vocab >= 1");
    FITRE_REQUIRE(vocab <= (1l << 28) && rows <= (1l << 27), FITRE_ERR_TOO_LARGE,
                  "token log probabilities: at most 2^28 entries and 2^27 rows");
}

// Checks the matrices of the gated block; `stored`: g and u are needed.
void need_gated_shape(int dtype, int act, long tokens, long width, long hidden) {
    FITRE_REQUIRE(dtype == FITRE_DTYPE_BF16 || dtype == FITRE_DTYPE_F16, FITRE_ERR_UNSUPPORTED,
                  "gated block: bf16 or fp16 tensors");
    FITRE_REQUIRE(act == FITRE_CNN_ACT_NONE || act == FITRE_CNN_ACT_SOFTPLUS || act == FITRE_CNN_ACT_RELU ||
                      act == FITRE_CNN_ACT_SWISH,
                  FITRE_ERR_UNSUPPORTED, "gated block: activation outside the path");
    need(tokens >= 0 && width >= 1 && hidden >= 1, "gated block: tokens >= 0, width >= 1 and hidden >= 1");
    FITRE_REQUIRE(tokens <= (1l << 24) && width <= (1l << 20) && hidden <= (1l << 20), FITRE_ERR_TOO_LARGE,
                  "gated block: too large");
}
// The stride of a matrix of one row never matters; one that TMA takes.
void settle_stride(long &ld, long rows, long cols) {
    if (rows <= 1) ld = (cols + 7) / 8 * 8;
}
// Operands of the tensor-core products with a width that is a multiple of 8 are read in place.
void need_readable(const void *p, long ld, long width, const char *what) {
    FITRE_REQUIRE(width % 8 != 0 || gated_rows_readable(p, ld), FITRE_ERR_UNSUPPORTED,
                  std::string(what) + ": rows have to start on 16-byte boundaries when the width is a multiple of 8");
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

long fitre_gated_forward_mem_required(long tokens, long width, long hidden) {
    if (tokens <= 0 || width <= 0 || hidden <= 0 || tokens > (1l << 24) || width > (1l << 20) || hidden > (1l << 20))
        return 0;
    return as_doubles(gated_forward_scratch(tokens, width, hidden));
}

int fitre_gated_forward(fitre_context *ctx, int dtype, int act, const void *x, long ldx, const void *wGate, long ldwg,
                        const void *wUp, long ldwu, void *h, long ldh, void *gate, long ldg, void *up, long ldu,
                        long tokens, long width, long hidden, real *devPtr) {
    return on_context(ctx, [&] {
        need_gated_shape(dtype, act, tokens, width, hidden);
        if (tokens == 0) return;
        need_matrix(x, ldx, tokens, width, dtype, "x");
        need_matrix(wGate, ldwg, hidden, width, dtype, "wGate");
        need_matrix(wUp, ldwu, hidden, width, dtype, "wUp");
        need_matrix(h, ldh, tokens, hidden, dtype, "h");
        if (gate) need_matrix(gate, ldg, tokens, hidden, dtype, "gate");
        if (up) need_matrix(up, ldu, tokens, hidden, dtype, "up");
        settle_stride(ldx, tokens, width), settle_stride(ldwg, hidden, width), settle_stride(ldwu, hidden, width);
        settle_stride(ldh, tokens, hidden), settle_stride(ldg, tokens, hidden), settle_stride(ldu, tokens, hidden);
        if (!gated_streams(tokens)) {
            need_readable(x, ldx, width, "x");
            need_readable(wGate, ldwg, width, "wGate");
            need_readable(wUp, ldwu, width, "wUp");
        }
        const long scratch = fitre_gated_forward_mem_required(tokens, width, hidden);
        if (scratch) {
            need(devPtr && aligned16(devPtr), "gated block: devPtr is NULL or not 16-byte aligned");
            require_scratch(ctx, scratch, "gated block");
        }
        GatedArgs a = {};
        a.dtype = dtype, a.act = act, a.x = x, a.ldx = ldx, a.wg = wGate, a.ldwg = ldwg, a.wu = wUp, a.ldwu = ldwu;
        a.h = h, a.ldh = ldh, a.g = gate, a.ldg = ldg, a.u = up, a.ldu = ldu;
        a.tokens = tokens, a.width = width, a.hidden = hidden, a.scratch = devPtr;
        gated_forward(ctx, a);
    });
}

long fitre_gated_backward_mem_required(long tokens, long width, long hidden) {
    if (tokens <= 0 || width <= 0 || hidden <= 0 || tokens > (1l << 24) || width > (1l << 20) || hidden > (1l << 20))
        return 0;
    return as_doubles(gated_backward_scratch(tokens, width, hidden));
}

int fitre_gated_backward(fitre_context *ctx, int dtype, int act, const void *dh, long lddh, const void *x, long ldx,
                         const void *wGate, long ldwg, const void *wUp, long ldwu, const void *gate, long ldg,
                         const void *up, long ldu, void *dx, long lddx, void *dwGate, long lddwg, void *dwUp,
                         long lddwu, long tokens, long width, long hidden, real *devPtr) {
    return on_context(ctx, [&] {
        need_gated_shape(dtype, act, tokens, width, hidden);
        need_matrix(dwGate, lddwg, hidden, width, dtype, "dwGate");
        need_matrix(dwUp, lddwu, hidden, width, dtype, "dwUp");
        if (tokens == 0) {   // the sum over no tokens
            const long row = width * dtype_bytes(dtype);
            FITRE_CUDA(cudaMemset2DAsync(dwGate, (hidden > 1 ? lddwg : width) * dtype_bytes(dtype), 0, row, hidden, ctx->stream));
            FITRE_CUDA(cudaMemset2DAsync(dwUp, (hidden > 1 ? lddwu : width) * dtype_bytes(dtype), 0, row, hidden, ctx->stream));
            return;
        }
        need_matrix(dh, lddh, tokens, hidden, dtype, "dh");
        need_matrix(x, ldx, tokens, width, dtype, "x");
        need_matrix(wGate, ldwg, hidden, width, dtype, "wGate");
        need_matrix(wUp, ldwu, hidden, width, dtype, "wUp");
        need_matrix(gate, ldg, tokens, hidden, dtype, "gate");
        need_matrix(up, ldu, tokens, hidden, dtype, "up");
        need_matrix(dx, lddx, tokens, width, dtype, "dx");
        settle_stride(ldx, tokens, width), settle_stride(ldwg, hidden, width), settle_stride(ldwu, hidden, width);
        settle_stride(lddh, tokens, hidden), settle_stride(ldg, tokens, hidden), settle_stride(ldu, tokens, hidden);
        settle_stride(lddx, tokens, width), settle_stride(lddwg, hidden, width), settle_stride(lddwu, hidden, width);
        need_readable(x, ldx, width, "x");
        need_readable(wGate, ldwg, width, "wGate");
        need_readable(wUp, ldwu, width, "wUp");
        need(devPtr && aligned16(devPtr), "gated block backward: devPtr is NULL or not 16-byte aligned");
        require_scratch(ctx, fitre_gated_backward_mem_required(tokens, width, hidden), "gated block backward");
        GatedArgs a = {};
        a.dtype = dtype, a.act = act, a.dh = dh, a.lddh = lddh, a.x = x, a.ldx = ldx, a.wg = wGate, a.ldwg = ldwg;
        a.wu = wUp, a.ldwu = ldwu, a.g = (void *)gate, a.ldg = ldg, a.u = (void *)up, a.ldu = ldu;
        a.dx = dx, a.lddx = lddx, a.dwg = dwGate, a.lddwg = lddwg, a.dwu = dwUp, a.lddwu = lddwu;
        a.tokens = tokens, a.width = width, a.hidden = hidden, a.scratch = devPtr;
        gated_backward(ctx, a);
    });
}

long fitre_orthogonalize_mem_required(long batch, long rows, long cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || batch > 65535 || rows > (1l << 17) || cols > (1l << 17)) return 0;
    return as_doubles(ortho_scratch(batch, rows, cols));
}

int fitre_orthogonalize_update(fitre_context *ctx, int dtype, const void *update, long ldu, long strideu, void *out,
                               long ldo, long strideo, long batch, long rows, long cols, int steps,
                               const real *coefficients_host, real scale, real eps, real *devPtr) {
    return on_context(ctx, [&] {
        need_type(dtype);
        need(batch >= 0 && rows >= 1 && cols >= 1, "orthogonalised update: batch >= 0, rows >= 1 and cols >= 1");
        need(steps >= 1 && steps <= 100, "orthogonalised update: 1 to 100 steps");
        need(std::isfinite(scale) && std::isfinite(eps) && eps >= 0, "orthogonalised update: scale or eps not finite");
        FITRE_REQUIRE(batch <= 65535 && rows <= (1l << 17) && cols <= (1l << 17), FITRE_ERR_TOO_LARGE,
                      "orthogonalised update: at most 65535 matrices of 131072 rows and columns");
        static const real usual[3] = {3.4445, -4.7750, 2.0315};
        const real *coef = coefficients_host ? coefficients_host : usual;
        need(std::isfinite(coef[0]) && std::isfinite(coef[1]) && std::isfinite(coef[2]),
             "orthogonalised update: coefficients not finite");
        if (batch == 0) return;
        settle_stride(ldu, rows, cols), settle_stride(ldo, rows, cols);
        need_matrix(update, ldu, rows, cols, dtype, "update");
        need_matrix(out, ldo, rows, cols, FITRE_DTYPE_BF16, "out");
        const long spanu = rows > 1 ? (rows - 1) * ldu + cols : cols, spano = rows > 1 ? (rows - 1) * ldo + cols : cols;
        need(batch == 1 || (strideu >= spanu && strideo >= spano), "orthogonalised update: matrices overlap");
        FITRE_REQUIRE(batch == 1 || (strideu < kMaxElements && strideo < kMaxElements), FITRE_ERR_TOO_LARGE,
                      "orthogonalised update: spans too many elements");
        need(devPtr && aligned16(devPtr), "orthogonalised update: devPtr is NULL or not 16-byte aligned");
        require_scratch(ctx, fitre_orthogonalize_mem_required(batch, rows, cols), "orthogonalised update");
        OrthoArgs a = {};
        a.dtype = dtype, a.in = update, a.ldi = ldu, a.istride = batch > 1 ? strideu : 0, a.out = out, a.ldo = ldo;
        a.ostride = batch > 1 ? strideo : 0, a.batch = batch, a.rows = rows, a.cols = cols, a.steps = steps;
        for (int i = 0; i < 3; ++i) a.coef[i] = coef[i];
        a.scale = scale, a.eps = eps, a.scratch = devPtr;
        orthogonalize(ctx, a);
    });
}

int fitre_synchronize(fitre_context *ctx) {
    return on_context(ctx, [&] { check_device_error(ctx); });
}

}  // extern "C"
