"""Orthogonalised update against the same polynomial in 64 bits, and as one training step with the other
language-model operators."""
import types

import pytest
import torch

import lm_util as U
from fitre_b200 import _structs as S
from fitre_b200 import api

gpu = pytest.mark.gpu
SWISH = S.CNN_ACT_SWISH
DEFAULT = (3.4445, -4.7750, 2.0315)


def polynomial(g, steps=5, coef=DEFAULT, eps=1e-7):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    a, b, c = coef
    for _ in range(steps):
        y = x @ x.mT
        x = a * x + (b * y + c * (y @ y)) @ x
    return x.mT if tall else x


def update(batch, rows, cols, kind, dtype, seed=3):
    g = U.gen(seed + rows + cols)
    k = max(1, min(rows, cols) // 16)
    low = torch.randn(batch, rows, k, generator=g, device="cuda", dtype=torch.float64) @ torch.randn(
        batch, k, cols, generator=g, device="cuda", dtype=torch.float64)
    full = torch.randn(batch, rows, cols, generator=g, device="cuda", dtype=torch.float64)
    return {"full": full, "low": low, "mixed": full + 3 * low / k ** 0.5}[kind].mul(0.01).to(dtype)


def run(g, steps=5, how="dense", **kw):
    batch, rows, cols = g.shape if g.dim() == 3 else (1, *g.shape)
    out = torch.full_like(g, 9.0, dtype=torch.bfloat16)
    ws = torch.empty(api.orthogonalizeMemRequired(batch, rows, cols), device="cuda", dtype=torch.float64)
    api.orthogonalizeUpdate(U.ctx(), g, out, ws, steps, **kw)
    U.ctx().synchronize()
    return out


# The result's norm-wise error: bf16's own rounding (2^-8 / sqrt 3 at most in the mean square) and that of the
# iteration.  The latter: every product rounds its operands to fp16 (2^-11 / sqrt 3 in the mean square), with weights
# that the steps' terms a, b s^2, c s^4 (at most 3.4, 5.7, 2.9) put on them; with the low part and the diagonal held
# apart, what a step adds is below 4 of those roundings, and what five steps add, independent of one another and
# amplified by slopes of at most 1.7 once the singular values are of order one, below 4 sqrt(1 + 2.9 + 2.9 + ...) < 12:
# 12 * 2^-11 / sqrt 3 = 3.4e-3 beside 2.3e-3, in sum of squares 4.1e-3.  Matrices of a few entries average nothing:
# twice that.
BOUND = 4.1e-3


@gpu
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 40), (1, 17, 5), (3, 8, 8), (1, 64, 64), (2, 100, 260), (1, 129, 128),
                                   (5, 513, 384), (1, 1000, 77), (2, 384, 1001), (1, 1024, 1024), (1, 300, 4000), (2, 3000, 200),
                                   (2, 2304, 2560), (2, 2600, 2304)], ids=str)
@pytest.mark.parametrize("kind", ["full", "low", "mixed"])
def test_against_the_polynomial(shape, kind):
    dtype = {"full": torch.float32, "low": torch.bfloat16, "mixed": torch.float64}[kind]
    g = update(*shape, kind, dtype)
    for steps in (1, 5):
        want = polynomial(g, steps)
        got = run(g, steps).double()
        err = (got - want).norm() / want.norm()
        assert err < (BOUND if min(shape[1:]) >= 64 else 2 * BOUND), (steps, float(err))
    # singular values of the result: the quintic's fixed band
    if kind == "full" and shape[1] != shape[2] and min(shape[1:]) <= 384:
        sv = torch.linalg.svdvals(got)
        assert sv.max() < 1.25 and sv.min() > 0.3


@gpu
@pytest.mark.parametrize("dtype", list(U.TYPES))
def test_layouts_types_and_parameters(dtype):
    g = update(3, 70, 50, "full", U.TYPES[dtype])
    plain = run(g)
    # a view with gaps between rows and between matrices, off every boundary
    buf = torch.zeros(3, 75, 53, device="cuda", dtype=g.dtype)
    view = buf[:, 2:72, 1:51]
    view.copy_(g)
    obuf = torch.full((3, 75, 61), 7.0, device="cuda", dtype=torch.bfloat16)
    oview = obuf[:, 2:72, 5:55]
    ws = torch.empty(api.orthogonalizeMemRequired(3, 70, 50), device="cuda", dtype=torch.float64)
    api.orthogonalizeUpdate(U.ctx(), view, oview, ws)
    assert torch.equal(oview, plain)
    obuf[:, 2:72, 5:55] = 7.0
    assert (obuf == 7.0).all()
    # one of the batch alone, and in place
    assert torch.equal(run(g[1]), plain[1])
    if g.dtype == torch.bfloat16:
        same = g.clone()
        api.orthogonalizeUpdate(U.ctx(), same, same, ws)
        assert torch.equal(same, plain)
    # scale, coefficients, eps
    want = polynomial(g, 3, (2.0, -1.5, 0.5), 0.1) * 0.2
    got = run(g, 3, coefficients=(2.0, -1.5, 0.5), scale=0.2, eps=0.1).double()
    assert (got - want).norm() / want.norm() < BOUND


@gpu
def test_special_matrices():
    c = U.ctx()
    g = torch.zeros(4, 20, 30, device="cuda")
    g[1] = U.randn(U.gen(1), 20, 30) * 1e25          # squares beyond fp32
    g[2] = U.randn(U.gen(2), 20, 30) * 1e-30         # far below eps: vanishes as the formula says
    g[3, 2, 3] = float("nan")
    out = run(g)
    assert not out[0].any()
    want = polynomial(g[1])
    assert (out[1].double() - want).norm() / want.norm() < 2 * BOUND
    assert out[2].abs().max() < 1e-15
    assert torch.isnan(out[3]).all()
    out = run(g, eps=0.0)
    assert torch.isnan(out[0]).all()                 # 0 / 0 without eps
    want = polynomial(g[2], eps=0.0)
    assert (out[2].double() - want).norm() / want.norm() < 2 * BOUND
    api.orthogonalizeUpdate(c, g[:0], out[:0], None)


@gpu
def test_the_range_of_fp64():
    g = torch.stack([U.randn(U.gen(3), 20, 30).double().cuda() * f for f in (1e200, 1e150, 1e-150, 1e-200)])
    out = run(g, eps=0.0)
    assert torch.isnan(out[0]).all()                 # the sum of squares overflows
    for i in (1, 2):
        want = polynomial(g[i], eps=0.0)
        assert (out[i].double() - want).norm() / want.norm() < 2 * BOUND
    assert not run(g)[3].any()                       # far below eps


@gpu
def test_same_bits_on_a_stream_and_in_a_graph():
    g = update(2, 300, 520, "mixed", torch.float32)
    first = run(g)
    stream = torch.cuda.Stream()
    c = U.ctx(stream)
    out = torch.zeros_like(first)
    ws = torch.empty(api.orthogonalizeMemRequired(2, 300, 520), device="cuda", dtype=torch.float64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        api.orthogonalizeUpdate(c, g, out, ws)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def refused(status, f, *args, **kw):
    with pytest.raises(api.FitreError) as e:
        f(*args, **kw)
    assert e.value.status == status


def test_refusals_without_a_device():
    c = types.SimpleNamespace(device=0, h=None, lib=None)
    x = torch.zeros(4, 8)
    refused(S.ERR_BAD_ARG, api.orthogonalizeUpdate, c, x, x.bfloat16(), None)
    refused(S.ERR_UNSUPPORTED, api.orthogonalizeUpdate, c, x, x, None)
    refused(S.ERR_UNSUPPORTED, api.orthogonalizeUpdate, c, x.int(), x, None)
    refused(S.ERR_BAD_ARG, api.orthogonalizeUpdate, c, x, x[:2].bfloat16(), None)
    from fitre_b200 import _lib
    L = _lib.load()
    assert L.fitre_orthogonalize_update(None, 1, None, 8, 0, None, 8, 0, 1, 4, 8, 5, None, 1.0, 1e-7, None) == S.ERR_BAD_ARG
    assert L.fitre_synchronize(None) == S.ERR_BAD_ARG
    assert api.orthogonalizeMemRequired(0, 4, 4) == 0 and api.orthogonalizeMemRequired(1, 2 ** 20, 4) == 0
    assert api.orthogonalizeMemRequired(2, 100, 300) >= 2 * (3 * 100 * 300 + 2 * 100 * 100) // 4


@gpu
def test_refusals():
    c = U.ctx()
    x = torch.ones(4, 8, device="cuda")
    o = torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(api.orthogonalizeMemRequired(1, 4, 8), device="cuda", dtype=torch.float64)
    f = api.orthogonalizeUpdate
    refused(S.ERR_BAD_ARG, f, c, x, o, ws, 0)
    refused(S.ERR_BAD_ARG, f, c, x, o, ws, 5, (1.0, float("inf"), 0.0))
    refused(S.ERR_BAD_ARG, f, c, x, o, ws, 5, None, float("nan"))
    refused(S.ERR_BAD_ARG, f, c, x, o, ws, 5, None, 1.0, -1.0)
    refused(S.ERR_WORKSPACE, f, c, x, o, None)
    refused(S.ERR_WORKSPACE, f, c, x, o, ws[:3])
    refused(S.ERR_BAD_ARG, f, c, x.t(), o.t(), ws)
    refused(S.ERR_BAD_ARG, f, c, x[0], o[0], ws)
    refused(S.ERR_BAD_ARG, f, c, x[None].expand(2, 4, 8), o[None].expand(2, 4, 8),
            torch.empty(api.orthogonalizeMemRequired(2, 4, 8), device="cuda", dtype=torch.float64))


@gpu
def test_one_training_step():
    """norm -> gated block -> projection -> token log probabilities, their gradients back through all of it, and
    the orthogonalised update of both weights, against the same step in 64 bits by automatic differentiation."""
    t, d, f, v = 96, 128, 320, 500
    dt = torch.bfloat16
    g = U.gen(11)
    c = U.ctx()
    x = U.randn(g, t, d, dtype=dt)
    gamma, beta = (1 + U.randn(g, d, scale=0.1)).to(dt), U.randn(g, d, scale=0.1, dtype=dt)
    wg, wu = (U.randn(g, f, d, scale=d ** -0.5, dtype=dt) for _ in range(2))
    proj = U.randn(g, v, f, scale=2 * f ** -0.5, dtype=dt)
    tokens = torch.randint(0, v, (t,), generator=g, device="cuda")
    tokens[5] = -1
    new = lambda *s, dtype=dt: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
    y, mean, rstd = new(t, d), new(t, dtype=torch.float32), new(t, dtype=torch.float32)
    api.layerNormForward(c, x, gamma, beta, y, mean, rstd)
    h, gate, up = new(t, f), new(t, f), new(t, f)
    api.gatedForward(c, y, wg, wu, h, gate, up)
    logits = h @ proj.T
    lp, lse, ent = (new(t, dtype=torch.float32) for _ in range(3))
    api.tokenLogProbs(c, logits, tokens, lp, lse, ent)
    weight = -torch.ones(t, device="cuda") / t
    bonus = torch.full((t,), -0.01 / t, device="cuda")
    dlogits = new(t, v)
    api.tokenLogProbsBackward(c, logits, tokens, lse, ent, weight, bonus, dlogits)
    dh = dlogits @ proj
    dy, dwg, dwu = new(t, d), new(f, d), new(f, d)
    api.gatedBackward(c, dh, y, wg, wu, gate, up, dy, dwg, dwu, SWISH,
                      torch.empty(api.gatedBackwardMemRequired(t, d, f), device="cuda", dtype=torch.float64))
    dx, dgamma, dbeta = new(t, d), new(d), new(d)
    api.layerNormBackward(c, dy, x, gamma, mean, rstd, dx, dgamma, dbeta,
                          torch.empty(api.layerNormBackwardMemRequired(t, d), device="cuda", dtype=torch.float64))
    both, steps = torch.stack((dwg, dwu)), new(2, f, d)
    api.orthogonalizeUpdate(c, both, steps, torch.empty(api.orthogonalizeMemRequired(2, f, d), device="cuda",
                                                       dtype=torch.float64))
    c.synchronize()

    leaves = [p.double().requires_grad_() for p in (x, gamma, beta, wg, wu)]
    X, G, B, Wg, Wu = leaves
    Y = torch.nn.functional.layer_norm(X, (d,), G, B, 1e-5)
    H = torch.nn.functional.silu(Y @ Wg.T) * (Y @ Wu.T)
    LP = torch.log_softmax(H @ proj.double().T, 1)
    picked = LP.gather(1, tokens.clamp_min(0)[:, None])[:, 0].masked_fill(tokens < 0, 0)
    entropy = -(LP.exp() * LP).sum(1)
    loss = (picked * weight.double()).sum() + (entropy * bonus.double()).sum()
    loss.backward()
    got = (lp.double() * weight.double()).sum() + (ent.double() * bonus.double()).sum()
    # every tensor between the operators is rounded to bf16 (2^-8): the loss moves by a few of those, the gradients
    # by the roundings of the six tensors behind them, 2^-8 / sqrt 3 each, amplified a few times by the soft-max
    assert abs(got - loss) < 0.01 * abs(loss)
    for mine, p in ((dx, X), (dgamma, G), (dbeta, B), (dwg, Wg), (dwu, Wu)):
        assert (mine.double() - p.grad).norm() < 0.05 * p.grad.norm()
    # the update of the gradients that the step itself formed
    for mine, grad in zip(steps, (dwg, dwu)):
        want = polynomial(grad)
        assert (mine.double() - want).norm() < BOUND * want.norm()



@gpu
def test_products_on_two_streams_at_once():
    """The tensor-core kernels take whole SMs and wait within their clusters only: two streams interleave freely."""
    gs = [update(2, 300, 520, "mixed", torch.float32, s) for s in (1, 2)]
    alone = [run(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    ctxs = [U.ctx(s) for s in streams]
    outs = [torch.zeros_like(a) for a in alone]
    scratch = [torch.empty(api.orthogonalizeMemRequired(2, 300, 520), device="cuda", dtype=torch.float64) for _ in gs]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, g, o, w in zip(ctxs, gs, outs, scratch):
            api.orthogonalizeUpdate(c, g, o, w)
    for c in ctxs:
        c.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))


@gpu
def test_offsets_beyond_32_bits():
    g = update(2, 70, 96, "full", torch.bfloat16)
    apart = 1 << 31
    far = torch.empty(apart + 70 * 96, device="cuda", dtype=torch.bfloat16).as_strided((2, 70, 96), (apart, 96, 1))
    far.copy_(g)
    want = run(g)
    ws = torch.empty(api.orthogonalizeMemRequired(2, 70, 96), device="cuda", dtype=torch.float64)
    api.orthogonalizeUpdate(U.ctx(), far, far, ws)
    U.ctx().synchronize()
    assert torch.equal(far, want)
