"""Gated feed-forward block, forward and backward, against the formulas in 64 bits."""
import types

import pytest
import torch

import lm_util as U
from fitre_b200 import _structs as S
from fitre_b200 import api

gpu = pytest.mark.gpu
SWISH, RELU, SOFTPLUS, NONE = S.CNN_ACT_SWISH, S.CNN_ACT_RELU, S.CNN_ACT_SOFTPLUS, S.CNN_ACT_NONE
# tokens, width, hidden: streaming kernel (up to 4 tokens), single-SM tiles, SM pairs, ragged edges, every
# alignment class, one of everything
SHAPES = [(1, 1, 1), (1, 8, 3), (1, 520, 100), (2, 4096, 333), (3, 77, 40), (4, 1000, 129), (5, 8, 1), (5, 64, 64),
          (7, 65, 9), (128, 128, 64), (129, 72, 257), (300, 1000, 650), (513, 200, 2730), (1003, 333, 511),
          (2048, 512, 1280), (2100, 264, 1400)]


def activation(act, g):
    """act and its derivative"""
    if act == RELU:
        return g.clamp_min(0), (g > 0).double()
    if act == SOFTPLUS:
        return torch.logaddexp(g, torch.zeros_like(g)), torch.sigmoid(g)
    if act == NONE:
        return g, torch.ones_like(g)
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s))


def data(shape, dtype, seed=1):
    t, d, f = shape
    g = U.gen(seed + t + d + f)
    x = U.randn(g, t, d, dtype=dtype)
    wg, wu = (U.randn(g, f, d, dtype=dtype, scale=d ** -0.5) for _ in range(2))
    return x, wg, wu, g


def scratch(n):
    return torch.empty(n, device="cuda", dtype=torch.float64) if n else None


def sum_units(k):
    """Units of u in a tensor-core sum of k products relative to the sum of their magnitudes: one addition per
    16 products, each of which may truncate (2 u) instead of rounding, and the 16 inside (2 u each)."""
    return 2 * (k / 16 + 32)


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_forward_and_backward(shape, kind):
    dtype = U.TYPES[kind]
    t, d, f = shape
    x, wg, wu, gen = data(shape, dtype)
    u, half, tiny, c = 2.0 ** -24, U.half_step(dtype), U.tiny(dtype), U.ctx()
    xd, gd, ud = x.double(), wg.double(), wu.double()
    g64, u64 = xd @ gd.T, xd @ ud.T
    mg, mu = xd.abs() @ gd.abs().T, xd.abs() @ ud.abs().T
    eg, eu = sum_units(d) * u * mg, sum_units(d) * u * mu
    for act, how in ((SWISH, "dense"), (RELU, "strided"), (SOFTPLUS, "odd"), (NONE, "dense")):
        odd_ok = d % 8 != 0 or t <= 4      # rows off the 16-byte grid: small token counts or odd widths only
        lay = how if how != "odd" or odd_ok else "strided"
        xv, gv, uv = (U.laid_out(m, lay) for m in (x, wg, wu))
        h, go, uo = (U.laid_out(torch.full((t, f), 9.0, device="cuda", dtype=dtype), how) for _ in range(3))
        api.gatedForward(c, xv, gv, uv, h, go, uo, act, scratch(api.gatedForwardMemRequired(t, d, f)))
        c.synchronize()
        U.close(go, g64, half * g64.abs() + eg + tiny)
        U.close(uo, u64, half * u64.abs() + eu + tiny)
        a, da = activation(act, g64)
        want = a * u64
        # the activation's own arithmetic: exp to 2^-21 and a few roundings; slopes are below 1.1; a softplus or
        # Swish value near zero is a difference of numbers of order one only for softplus (absolute 2^-22)
        ea = 1.1 * eg + a.abs() * (16 + 4 * g64.abs()) * u + (2.0 ** -21 * torch.exp(-g64.abs()) if act == SOFTPLUS else 0)
        U.close(h, want, half * want.abs() + ea * u64.abs() + (a.abs() + ea) * eu + tiny)
        assert all(U.gaps_untouched(m) for m in (h, go, uo))
        only = U.laid_out(torch.full((t, f), 9.0, device="cuda", dtype=dtype), how)
        api.gatedForward(c, xv, gv, uv, only, None, None, act, scratch(api.gatedForwardMemRequired(t, d, f)))
        assert torch.equal(only, h)

        # backward from the stored tensors
        dh = U.randn(gen, t, f, dtype=dtype)
        dhv = U.laid_out(dh, how)
        dx = U.laid_out(torch.full((t, d), 9.0, device="cuda", dtype=dtype), how)
        dwg, dwu = (U.laid_out(torch.full((f, d), 9.0, device="cuda", dtype=dtype), how) for _ in range(2))
        if d % 8 == 0 and lay == "odd":
            xv, gv, uv = (U.laid_out(m, "strided") for m in (x, wg, wu))   # the backward pass reads tiles at any size
        api.gatedBackward(c, dhv, xv, gv, uv, go, uo, dx, dwg, dwu, act, scratch(api.gatedBackwardMemRequired(t, d, f)))
        c.synchronize()
        gs, us = go.double(), uo.double()
        a, da = activation(act, gs)
        dg, du = dh.double() * us * da, dh.double() * a
        # dg and du are rounded to the type once (and carry the activation's arithmetic)
        slack = half + (32 + 8 * gs.abs()) * u
        edg = dg.abs() * slack + tiny + (dh.double() * us).abs() * 2.0 ** -20
        edu = du.abs() * slack + tiny + (dh.double().abs() * 2.0 ** -21 if act == SOFTPLUS else 0)
        want = dg @ gd + du @ ud
        mag = dg.abs() @ gd.abs() + du.abs() @ ud.abs()
        U.close(dx, want, half * want.abs() + edg @ gd.abs() + edu @ ud.abs() + sum_units(2 * f) * u * mag + tiny)
        for out, s, e in ((dwg, dg, edg), (dwu, du, edu)):
            want = s.T @ xd
            U.close(out, want, half * want.abs() + e.T @ xd.abs() + sum_units(t) * u * (s.abs().T @ xd.abs()) + tiny)
            if want.numel() > 1000 and t > 16:
                # independent roundings: the error's norm is far below the bound above, two half steps at most
                assert (out.double() - want).norm() <= 2 * half * want.norm()
        assert all(U.gaps_untouched(m) for m in (dx, dwg, dwu))


@gpu
def test_extreme_preactivations():
    """Large positive and negative gates: Swish goes to g or to 0, never to NaN."""
    x = torch.eye(8, device="cuda", dtype=torch.bfloat16)
    gate = torch.tensor([-3e38, -1e4, -200.0, -90.0, 90.0, 200.0, 1e4, 1e30], device="cuda").to(torch.bfloat16)
    wg = torch.diag(gate)
    wu = torch.ones(8, 8, device="cuda", dtype=torch.bfloat16)
    h, g, u = (torch.empty(8, 8, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    c = U.ctx()
    for act in (SWISH, RELU, SOFTPLUS):
        api.gatedForward(c, x, wg, wu, h, g, u, act)
        on = h.diagonal().double()
        want = gate.double().clamp_min(0)
        assert torch.isfinite(h).all() and ((on - want).abs() <= 1e-30 + 2.0 ** -8 * want).all()
        dx, dwg, dwu = (torch.empty(8, 8, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        api.gatedBackward(c, torch.ones_like(h), x, wg, wu, g, u, dx, dwg, dwu, act,
                          scratch(api.gatedBackwardMemRequired(8, 8, 8)))
        assert torch.isfinite(dwg).all() and torch.isfinite(dwu).all()
        slope = (gate > 0).double()
        assert ((dwg.diagonal().double() - slope).abs() < 1e-6).all()


@gpu
def test_no_tokens():
    c = U.ctx()
    e = torch.empty(0, 16, device="cuda", dtype=torch.float16)
    w = torch.ones(24, 16, device="cuda", dtype=torch.float16)
    h = torch.empty(0, 24, device="cuda", dtype=torch.float16)
    api.gatedForward(c, e, w, w, h)
    dwg, dwu = U.laid_out(w, "odd"), w.clone()
    api.gatedBackward(c, h, e, w, w, h, h, e, dwg, dwu)
    assert not dwg.any() and not dwu.any() and U.gaps_untouched(dwg)


@gpu
def test_gradient_matches_differences():
    """Directional derivatives of sum(h * r) by differences large enough for fp16 outputs: h is linear in wUp,
    and smooth in wGate."""
    t, d, f = 24, 64, 40
    x, wg, wu, gen = data((t, d, f), torch.float16, 5)
    r = U.randn(gen, t, f, dtype=torch.float16)
    c = U.ctx()
    h, g, u = (torch.empty(t, f, device="cuda", dtype=torch.float16) for _ in range(3))

    def value(x_, g_, u_):
        api.gatedForward(c, x_, g_, u_, h, g, u)
        return (h.double() * r.double()).sum().item()

    value(x, wg, wu)
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    api.gatedBackward(c, r, x, wg, wu, g.clone(), u.clone(), dx, dwg, dwu, SWISH,
                      scratch(api.gatedBackwardMemRequired(t, d, f)))
    for which, grad in ((0, dx), (1, dwg), (2, dwu)):
        args = [x, wg, wu]
        step = 2.0 ** -4 * grad.double() / grad.double().norm()          # along the gradient: the largest slope
        plus, minus = list(args), list(args)
        plus[which], minus[which] = (args[which].double() + step).half(), (args[which].double() - step).half()
        moved = plus[which].double() - minus[which].double()             # what the rounded steps really are
        predicted = (grad.double() * moved).sum().item()
        # h's roundings: 2^-11 of values of order one, random signs over t * f values and two evaluations:
        # below 2^-11 * sqrt(2 * 960) * 4 = 0.09 of a change of 2^-3 * |grad|; third derivatives: step^2
        got = value(*plus) - value(*minus)
        assert abs(got - predicted) < 0.09 + 0.02 * abs(predicted), (which, got, predicted)


@gpu
def test_same_bits_on_a_stream_and_in_a_graph():
    t, d, f = 700, 333, 520
    x, wg, wu, gen = data((t, d, f), torch.bfloat16, 9)
    dh = U.randn(gen, t, f, dtype=torch.bfloat16)
    ws = scratch(max(api.gatedForwardMemRequired(t, d, f), api.gatedBackwardMemRequired(t, d, f)))

    def fresh():
        new = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        return [new(t, f), new(t, f), new(t, f), new(t, d), new(f, d), new(f, d)]

    def run(c, o):
        api.gatedForward(c, x, wg, wu, o[0], o[1], o[2], SWISH, ws)
        api.gatedBackward(c, dh, x, wg, wu, o[1], o[2], o[3], o[4], o[5], SWISH, ws)

    first, second = fresh(), fresh()
    run(U.ctx(), first)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    c = U.ctx(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(c, second)
    for _ in range(2):
        for o in second:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, second))
    c.synchronize()


def refused(status, f, *args, **kw):
    with pytest.raises(api.FitreError) as e:
        f(*args, **kw)
    assert e.value.status == status


def test_refusals_without_a_device():
    c = types.SimpleNamespace(device=0, h=None, lib=None)
    x = torch.zeros(8, 16, dtype=torch.bfloat16)
    refused(S.ERR_BAD_ARG, api.gatedForward, c, x, x, x, x)
    refused(S.ERR_UNSUPPORTED, api.gatedBackward, c, x, x.int(), x, x, x, x, x, x, x)
    from fitre_b200 import _lib
    L = _lib.load()
    assert L.fitre_gated_forward(None, 2, 14, *[None, 8] * 6, 4, 8, 8, None) == S.ERR_BAD_ARG
    assert L.fitre_gated_backward(None, 2, 14, *[None, 8] * 9, 4, 8, 8, None) == S.ERR_BAD_ARG
    assert api.gatedForwardMemRequired(4, 333, 10) == 0 and api.gatedForwardMemRequired(100, 1000, 10) == 0
    assert api.gatedForwardMemRequired(100, 333, 10) >= (100 + 20) * 336 // 4
    assert api.gatedBackwardMemRequired(100, 64, 333) >= 2 * 100 * 336 // 4
    assert api.gatedBackwardMemRequired(-1, 64, 333) == 0 and api.gatedBackwardMemRequired(1, 2 ** 40, 3) == 0


@gpu
def test_refusals():
    c = U.ctx()
    new = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, w, h = new(8, 16), new(24, 16), new(8, 24)
    ws = scratch(api.gatedBackwardMemRequired(8, 16, 24))
    f, b = api.gatedForward, api.gatedBackward
    refused(S.ERR_UNSUPPORTED, f, c, x.float(), w.float(), w.float(), h.float())
    refused(S.ERR_UNSUPPORTED, f, c, x, w, w, h, act=S.CNN_ACT_ELU)
    refused(S.ERR_BAD_ARG, f, c, x, w[:, :8], w, h)
    refused(S.ERR_BAD_ARG, f, c, x, w, w[:20], h)
    refused(S.ERR_BAD_ARG, f, c, x, w, w, h[:, :20])
    refused(S.ERR_BAD_ARG, f, c, x, w.half(), w, h)
    refused(S.ERR_BAD_ARG, f, c, x, w, w, h, new(8, 20))
    refused(S.ERR_UNSUPPORTED, f, c, U.laid_out(x, "odd"), w, w, h)
    refused(S.ERR_WORKSPACE, f, c, new(8, 15), new(24, 15), new(24, 15), h)
    refused(S.ERR_BAD_ARG, b, c, h, x, w, w, h, h, x.t(), w, w, devPtr=ws)
    refused(S.ERR_WORKSPACE, b, c, h, x, w, w, h, h, x.clone(), w.clone(), w.clone(), devPtr=None)
    refused(S.ERR_WORKSPACE, b, c, h, x, w, w, h, h, x.clone(), w.clone(), w.clone(), devPtr=ws[:4])
    f(c, x, w, w, h)
    c.synchronize()


@gpu
def test_offsets_beyond_32_bits():
    t, d, f, ld = 33000, 64, 72, 70000
    x, wg, wu, gen = data((t, d, f), torch.bfloat16, 2)
    far = torch.empty(t * ld, device="cuda", dtype=torch.bfloat16).as_strided((t, d), (ld, 1))
    far.copy_(x)
    c = U.ctx()
    results = []
    for view in (far, x):
        h, g, u = (torch.empty(t, f, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        api.gatedForward(c, view, wg, wu, h, g, u)
        dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
        api.gatedBackward(c, h, view, wg, wu, g, u, dx, dwg, dwu, SWISH, scratch(api.gatedBackwardMemRequired(t, d, f)))
        results.append((h, g, u, dx, dwg, dwu))
    c.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))
    ws = scratch(api.gatedBackwardMemRequired(t, d, f))
    api.gatedBackward(c, results[0][0], x, wg, wu, *results[0][1:3], far, torch.empty_like(wg), torch.empty_like(wu), SWISH, ws)
    assert torch.equal(far, results[0][3])
