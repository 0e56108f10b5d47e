"""Layer norm forward and backward against the formulas in 64 bits."""
import types

import pytest
import torch

import lm_util as U
from fitre_b200 import _structs as S
from fitre_b200 import api

gpu = pytest.mark.gpu
SHAPES = [(1, 1), (3, 7), (5, 32), (4, 512), (9, 513), (2, 1000), (3, 2048), (600, 2049), (7, 4096), (2, 8191),
          (3, 8192), (2, 16384), (2, 16385), (70, 20011), (1501, 96), (4001, 257), (2001, 1536), (1300, 4096), (901, 8192),
          (451, 9176)]


def reference(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    y = (x - mean) * rstd
    y = y * gamma.double() if gamma is not None else y
    return (y + beta.double() if beta is not None else y), mean[:, 0], rstd[:, 0]


def inputs(shape, dtype, wide, seed=1):
    g = U.gen(seed)
    rows, cols = shape
    x = U.randn(g, rows, cols) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda")) + U.randn(g, rows, 1)
    w = torch.float32 if wide else dtype
    return x.to(dtype), (1 + U.randn(g, cols, scale=0.2)).to(w), U.randn(g, cols, scale=0.2, dtype=w), g


def backward_reference(dy, x, gamma, mean, rstd):
    dy, x, m, r = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - m) * r
    g = dy * gamma.double() if gamma is not None else dy
    s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - s1 - xh * s2)
    # magnitudes that entered each result
    xa = (x.abs() + m.abs()) * r
    mdx = r * (g.abs() + g.abs().mean(1, keepdim=True) + xa * ((g.abs() * xa).mean(1, keepdim=True)))
    return dx, (dy * xh).sum(0), dy.sum(0), mdx, (dy.abs() * xa).sum(0), dy.abs().sum(0)


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16", "bf16 wide", "f16 wide"])
def test_forward_and_backward(shape, kind):
    dtype, wide = U.TYPES[kind.split()[0]], "wide" in kind
    u, half = U.unit(dtype), U.half_step(dtype)
    rows, cols = shape
    x, gamma, beta, g = inputs(shape, dtype, wide)
    for how in ("dense", "strided", "odd"):
        xv, y = U.laid_out(x, how), U.laid_out(torch.zeros_like(x), how)
        mean, rstd = (torch.zeros(rows, device="cuda", dtype=U.stat(dtype)) for _ in range(2))
        api.layerNormForward(U.ctx(), xv, gamma, beta, y, mean, rstd, 1e-5)
        ref, m, r = reference(x, gamma, beta, 1e-5)
        xa = x.double().abs()
        am = xa.mean(1)
        # mean: one sum.  rstd: the deviations carry the mean's error, their squares one more sum
        U.close(mean, m, 64 * u * am)
        rel = 64 * u * (1 + am * r)
        U.close(rstd, r, rel * r)
        mag = gamma.double().abs() * ((xa + am[:, None]) * r[:, None]) * (1 + 2 * (am * r)[:, None])
        U.close(y, ref, half * ref.abs() + 64 * u * (2 * mag + beta.double().abs()) + U.tiny(dtype))
        assert U.gaps_untouched(y)
        # backward, from the statistics just computed
        dy = U.randn(g, rows, cols, dtype=dtype)
        dyv, dx = U.laid_out(dy, how), U.laid_out(torch.zeros_like(x), how)
        dg, db = torch.full_like(gamma, 9.0), torch.full_like(gamma, 9.0)
        ws = torch.empty(api.layerNormBackwardMemRequired(rows, cols), device="cuda", dtype=torch.float64)
        api.layerNormBackward(U.ctx(), dyv, xv, gamma, mean, rstd, dx, dg, db, ws)
        rdx, rdg, rdb, mdx, mdg, mdb = backward_reference(dy, x, gamma, mean, rstd)
        U.close(dx, rdx, half * rdx.abs() + 64 * u * mdx + U.tiny(dtype))
        assert U.gaps_untouched(dx)
        hw = U.half_step(gamma.dtype)
        # chains of the sums over rows: <= rows / 100 + 64 terms with these shapes
        k = (128 + rows / 100) * u
        U.close(dg, rdg, hw * rdg.abs() + k * mdg + U.tiny(gamma.dtype))
        U.close(db, rdb, hw * rdb.abs() + k * mdb + U.tiny(gamma.dtype))


@gpu
@pytest.mark.parametrize("shape", [(5, 40), (33, 1023), (3, 16400)], ids=str)
def test_optional_arguments_and_in_place(shape):
    x, gamma, beta, g = inputs(shape, torch.float32, False, 3)
    rows, cols = shape
    c = U.ctx()
    y = torch.empty_like(x)
    api.layerNormForward(c, x, None, None, y)
    ref = reference(x, None, None, 1e-5)[0]
    U.close(y, ref, 1e-4)
    api.layerNormForward(c, x, gamma, None, y)
    U.close(y, reference(x, gamma, None, 1e-5)[0], 1e-4)
    api.layerNormForward(c, x, None, beta, y)
    U.close(y, reference(x, None, beta, 1e-5)[0], 1e-4)
    mean, rstd = (torch.empty(rows, device="cuda") for _ in range(2))
    api.layerNormForward(c, x, gamma, beta, y, mean, rstd)
    same = x.clone()
    api.layerNormForward(c, same, gamma, beta, same)
    assert torch.equal(same, y)
    # the gradient alone, without gamma, with one of the two sums, and over its own inputs
    dy, dx = U.randn(g, rows, cols), torch.empty_like(x)
    ws = torch.empty(api.layerNormBackwardMemRequired(rows, cols), device="cuda", dtype=torch.float64)
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    api.layerNormBackward(c, dy, x, gamma, mean, rstd, dx, dg, db, ws)
    only, one = torch.empty_like(x), torch.empty_like(gamma)
    api.layerNormBackward(c, dy, x, gamma, mean, rstd, only)
    assert torch.equal(only, dx)
    api.layerNormBackward(c, dy, x, gamma, mean, rstd, only, one, None, ws)
    assert torch.equal(one, dg)
    api.layerNormBackward(c, dy, x, gamma, mean, rstd, only, None, one, ws)
    assert torch.equal(one, db)
    for at in (0, 1):
        pair = [dy.clone(), x.clone()]
        api.layerNormBackward(c, pair[0], pair[1], gamma, mean, rstd, pair[at], dg, db, ws)
        assert torch.equal(pair[at], dx) and torch.equal(db, one)
    api.layerNormBackward(c, dy, x, None, mean, rstd, dx)
    U.close(dx, backward_reference(dy, x, None, mean, rstd)[0], 1e-4)


@gpu
def test_special_rows():
    c = U.ctx()
    x = torch.zeros(4, 48, device="cuda")
    x[0] = 5.0                       # no variance
    x[1] = 1e4 + torch.arange(48, device="cuda") * 1e-2   # a large offset: the squares are of differences
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    y, mean, rstd = torch.empty_like(x), torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    api.layerNormForward(c, x, None, None, y, mean, rstd, 1e-5)
    assert torch.equal(y[0], torch.zeros(48, device="cuda")) and abs(rstd[0].item() - 1e-5 ** -0.5) < 1e-3
    want = reference(x[1:2], None, None, 1e-5)[0]
    # inputs near 1e4 are exact; the mean is off by 64 u 1e4 at most, the deviations are of order 0.1
    U.close(y[1:2], want, 64 * 2.0 ** -24 * 1e4 / 0.13 * 2)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()


@gpu
def test_no_rows():
    c = U.ctx()
    e = torch.empty(0, 24, device="cuda")
    s = torch.empty(0, device="cuda")
    gamma = torch.ones(24, device="cuda")
    api.layerNormForward(c, e, gamma, gamma, e.clone(), s, s)
    dg, db = torch.full((24,), 3.0, device="cuda"), torch.full((24,), 3.0, device="cuda")
    api.layerNormBackward(c, e, e, gamma, s, s, e.clone(), dg, db, None)
    assert not dg.any() and not db.any()


@gpu
def test_gradient_matches_differences():
    g = U.gen(5)
    x, dy = U.randn(g, 3, 37, dtype=torch.float64), U.randn(g, 3, 37, dtype=torch.float64)
    gamma, beta = U.randn(g, 37, dtype=torch.float64), U.randn(g, 37, dtype=torch.float64)
    c = U.ctx()
    y, mean, rstd = torch.empty_like(x), *(torch.empty(3, device="cuda", dtype=torch.float64) for _ in range(2))

    def value(x_, gamma_, beta_):
        api.layerNormForward(c, x_, gamma_, beta_, y, mean, rstd, 1e-5)
        return (y * dy).sum().item()

    value(x, gamma, beta)
    dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
    ws = torch.empty(api.layerNormBackwardMemRequired(3, 37), device="cuda", dtype=torch.float64)
    api.layerNormBackward(c, dy, x, gamma, mean.clone(), rstd.clone(), dx, dg, db, ws)
    h = 1e-5   # central differences: error h^2 f''' / 6 ~ 1e-9, rounding 1e-15 |f| / h ~ 1e-9
    for which, grad in ((0, dx), (1, dg), (2, db)):
        args = [x, gamma, beta]
        d = U.randn(g, *args[which].shape, dtype=torch.float64)
        plus, minus = list(args), list(args)
        plus[which], minus[which] = args[which] + h * d, args[which] - h * d
        slope = (value(*plus) - value(*minus)) / (2 * h)
        assert abs(slope - (grad * d).sum().item()) < 1e-6 * (1 + abs(slope))


@gpu
def test_same_bits_on_a_stream_and_in_a_graph():
    x, gamma, beta, g = inputs((777, 1024), torch.bfloat16, False, 8)
    dy = U.randn(g, 777, 1024, dtype=torch.bfloat16)
    ws = torch.empty(api.layerNormBackwardMemRequired(777, 1024), device="cuda", dtype=torch.float64)

    def run(c, out):
        api.layerNormForward(c, x, gamma, beta, out[0], out[1], out[2])
        api.layerNormBackward(c, dy, x, gamma, out[1], out[2], out[3], out[4], out[5], ws)

    def fresh():
        f = torch.float32
        return [torch.zeros_like(x), torch.zeros(777, device="cuda", dtype=f), torch.zeros(777, device="cuda", dtype=f),
                torch.zeros_like(x), torch.zeros_like(gamma), torch.zeros_like(gamma)]

    first, second = fresh(), fresh()
    run(U.ctx(), first)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    c = U.ctx(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(c, second)
    for _ in range(2):
        for t in second:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, second))


def refused(status, f, *args, **kw):
    with pytest.raises(api.FitreError) as e:
        f(*args, **kw)
    assert e.value.status == status


def test_refusals_without_a_device():
    """The host-side checks come before anything touches the GPU."""
    c = types.SimpleNamespace(device=0, h=None, lib=None)
    x = torch.zeros(4, 8)
    refused(S.ERR_BAD_ARG, api.layerNormForward, c, x, None, None, x)          # not on the device
    refused(S.ERR_UNSUPPORTED, api.layerNormForward, c, x.to(torch.int32), None, None, x)
    from fitre_b200 import _lib
    L = _lib.load()
    assert L.fitre_layer_norm_forward(None, 1, 1, None, 8, None, None, None, 8, None, None, 4, 8, 1e-5) == S.ERR_BAD_ARG
    assert L.fitre_layer_norm_backward(None, 1, 1, None, 8, None, 8, None, None, None, None, 8, None, None, 4, 8,
                                       None) == S.ERR_BAD_ARG
    assert api.layerNormBackwardMemRequired(0, 8) == 0 and api.layerNormBackwardMemRequired(-1, 8) == 0
    for rows, cols in ((1, 1), (100, 300), (10 ** 6, 4096), (5, 10 ** 5)):
        assert api.layerNormBackwardMemRequired(rows, cols) >= 2 * cols


@gpu
def test_refusals():
    c = U.ctx()
    x = torch.zeros(4, 8, device="cuda")
    w, s = torch.ones(8, device="cuda"), torch.zeros(4, device="cuda")
    f, b = api.layerNormForward, api.layerNormBackward
    ws = torch.empty(api.layerNormBackwardMemRequired(4, 8), device="cuda", dtype=torch.float64)
    refused(S.ERR_BAD_ARG, f, c, x, w, w, x[:, :7])
    refused(S.ERR_BAD_ARG, f, c, x, w, w, x.half())
    refused(S.ERR_BAD_ARG, f, c, x.t(), w[:4], w[:4], x.t())
    refused(S.ERR_BAD_ARG, f, c, x[0], w, w, x[0])
    refused(S.ERR_BAD_ARG, f, c, x, w[:7], w, x)
    refused(S.ERR_BAD_ARG, f, c, x[:1].expand(4, 8), w, w, x)     # rows on top of one another
    refused(S.ERR_UNSUPPORTED, f, c, x, w.double(), w, x)
    refused(S.ERR_BAD_ARG, f, c, x, w, w, x, s.double())
    refused(S.ERR_BAD_ARG, f, c, x, w, w, x, s, s, float("nan"))
    refused(S.ERR_BAD_ARG, f, c, x, w, w, x, s, s, -1.0)
    refused(S.ERR_BAD_ARG, f, c, x[:, :0], None, None, x[:, :0])
    refused(S.ERR_BAD_ARG, b, c, x, x, w, None, s, x)
    refused(S.ERR_WORKSPACE, b, c, x, x, w, s, s, x, w.clone(), None, None)
    refused(S.ERR_WORKSPACE, b, c, x, x, w, s, s, x, w.clone(), None, ws[:1])
    c.set_scratch_limit(1)
    try:
        refused(S.ERR_WORKSPACE, b, c, x, x, w, s, s, x, w.clone(), None, ws)
    finally:
        c.set_scratch_limit(0)
    api.layerNormForward(c, x, w, w, x)                            # the context stays usable


@gpu
def test_offsets_beyond_32_bits():
    """Rows far apart: the last ones lie more than 2^31 elements from the first."""
    rows, cols, ld = 33000, 64, 70000
    g = U.gen(12)
    base = torch.empty(rows * ld, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((rows, cols), (ld, 1))
    x.copy_(U.randn(g, rows, cols, dtype=torch.bfloat16))
    dense = x.contiguous()
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    c = U.ctx()
    outs = []
    for t in (x, dense):
        y, mean, rstd = torch.empty_like(dense), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        api.layerNormForward(c, t, w, w, y, mean, rstd)
        dx, dg, db = torch.empty_like(dense), torch.empty_like(w), torch.empty_like(w)
        ws = torch.empty(api.layerNormBackwardMemRequired(rows, cols), device="cuda", dtype=torch.float64)
        api.layerNormBackward(c, dense, t, w, mean, rstd, dx, dg, db, ws)
        outs.append((y, mean, rstd, dx, dg, db))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    api.layerNormForward(c, x, w, w, x)                   # written there, too
    assert torch.equal(x, outs[0][0])
