"""Token log probabilities, entropy, alternatives and the logits' gradient against 64 bits."""
import types

import pytest
import torch

import lm_util as U
from fitre_b200 import _structs as S
from fitre_b200 import api

gpu = pytest.mark.gpu
INF = float("inf")
SHAPES = [(1, 1), (2, 5), (3, 33), (1, 4097), (300, 130), (2, 8193), (1, 50001), (5, 32000), (160, 5000), (1, 131072),
          (2, 256000), (200, 70001), (1500, 4096)]


def reference(x, tokens, top):
    x = x.double()
    m = x.amax(1, keepdim=True)
    p = torch.exp(x - m)
    z = p.sum(1, keepdim=True)
    logs = torch.log(z)
    lse = (m + logs)[:, 0]
    d = torch.where(p > 0, x - m, 0.0)
    ed = (p * d).sum(1) / z[:, 0]
    ent = logs[:, 0] - ed
    lp = torch.where(tokens >= 0, ((x - m) - logs).gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return lse, ent, lp, ((x - m) - logs).gather(1, order), order, -ed


def outputs(rows, top, dtype):
    s = U.stat(dtype)
    new = [torch.full((rows,), 9.0, device="cuda", dtype=s) for _ in range(3)]
    if top:
        new += [torch.full((rows, top), 9.0, device="cuda", dtype=s),
                torch.full((rows, top), -5, device="cuda", dtype=torch.int64)]
    else:
        new += [None, None]
    return new


def chain(vocab, u, spread):
    """Longest chain of additions of a thread (at least 64 threads share a row), the 2^-22 of the fast
    exponential, and its argument's rounding, in units of the arithmetic."""
    return u * (vocab / 64 + 64 + 4 * spread)


def check(x, tokens, out, dtype, top):
    lse, ent, lp, tv, ti, ed = reference(x, tokens, max(top, 1))
    u = U.unit(dtype)
    k = chain(x.shape[1], u, 104) * (1 + ed)
    U.close(out[1], lse, k + 4 * u * lse.abs())
    U.close(out[2], ent, 2 * k + 4 * u * ent.abs())
    U.close(out[0], lp, k + 8 * u * (lp.abs() + lse.abs()))
    if top:
        assert torch.equal(out[4], ti)
        U.close(out[3], tv, k[:, None] + 8 * u * (tv.abs() + lse.abs()[:, None]))


@gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
def test_forward(shape, kind):
    dtype = U.TYPES[kind]
    rows, vocab = shape
    g = U.gen(vocab)
    x = U.randn(g, rows, vocab, dtype=dtype, scale=3.0)   # 16-bit types: many equal values
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens[rows // 2] = vocab - 1
    if rows > 2:
        tokens[1] = -1
    for top in sorted({0, 1, min(8, vocab), min(32, vocab)}):
        for how in ("dense", "strided", "odd"):
            xv = U.laid_out(x, how)
            out = outputs(rows, top, dtype)
            api.tokenLogProbs(U.ctx(), xv, tokens, *out)
            check(x, tokens, out, dtype, top)


@gpu
@pytest.mark.parametrize("shape", [(2400, 1), (2401, 5), (2500, 33), (2368, 255), (3001, 1024), (2371, 2049), (2400, 4097),
                                   (2390, 8192), (2368, 16001), (600, 30003)], ids=str)
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
def test_many_short_rows(shape, kind):
    # a warp per row adds chains of vocab / 32 elements, in pairs (fp64: up to 4096 elements, singly): within `chain`
    dtype = U.TYPES[kind]
    rows, vocab = shape
    g = U.gen(rows + vocab)
    x = U.randn(g, rows, vocab, dtype=dtype, scale=3.0)
    x[5, vocab // 2:] = -INF
    x[7] = torch.finfo(dtype).min
    x[8, 0] = 50.0
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens[5] = 0
    tokens[rows // 2] = vocab - 1
    tokens[1] = -1
    if vocab == 1:
        x[5] = 1.0
    for top in sorted({0, 1, *(min(t, max(1, vocab // 2)) for t in (3, 8, 32))}):
        for how in ("dense", "strided", "odd"):
            out = outputs(rows, top, dtype)
            api.tokenLogProbs(U.ctx(), U.laid_out(x, how), tokens, *out)
            check(x, tokens, out, dtype, top)


@gpu
@pytest.mark.parametrize("vocab", [40, 1000, 7000])
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
def test_many_short_rows_without_a_distribution(vocab, kind):
    dtype = U.TYPES[kind]
    rows = 2400
    x = U.randn(U.gen(vocab), rows, vocab, dtype=dtype)
    tokens = torch.full((rows,), 3, device="cuda")
    x[0] = -INF
    x[1, 6] = float("nan")
    x[2, vocab - 1] = INF
    tokens[3] = vocab
    x[4] = 0.0                                                 # ties: the lower index first
    x[5] = -INF
    x[5, 9] = -1.0
    for top in (0, 2, min(8, vocab)):
        out = outputs(rows, top, dtype)
        api.tokenLogProbs(U.ctx(), x, tokens, *out)
        lp, lse, ent = (o[:6].tolist() for o in out[:3])
        assert lse[0] == -INF and lp[0] == -INF and ent[0] == 0
        assert all(v != v for i in (1, 2) for v in (lp[i], lse[i], ent[i]))
        assert lp[3] != lp[3] and lse[3] == lse[3]
        assert lse[5] == -1.0 and ent[5] == 0 and lp[5] == -INF
        if top:
            order = list(range(top))
            assert out[4][0].tolist() == order and (out[3][0] == -INF).all()
            assert out[4][4].tolist() == order
            assert 6 not in out[4][1].tolist()
            assert out[4][2, 0] == vocab - 1
            assert out[4][5].tolist() == [9] + order[:-1] and (out[3][5, 1:] == -INF).all()
        rest = slice(6, None)
        check(x[rest], tokens[rest], [None if o is None else o[rest] for o in out], dtype, top)


@gpu
@pytest.mark.parametrize("vocab", [64, 999, 40000])
def test_ties_order_and_extremes(vocab):
    dtype = torch.float32
    x = torch.zeros(6, vocab, device="cuda")
    x[1] = torch.arange(vocab, device="cuda") / vocab                 # rising: the maximum moves all the time
    x[2] = -x[1]
    x[3] = torch.finfo(dtype).min                                      # masked with the lowest value throughout
    x[4] = torch.finfo(dtype).min
    x[4, vocab // 3] = 1.0
    x[5] = 1e30
    x[5, 7] = 1.00001e30
    x[0, 5] = -0.0
    tokens = torch.tensor([3, vocab - 1, 0, 1, vocab // 3, 7], device="cuda")
    out = outputs(6, 32, dtype)
    api.tokenLogProbs(U.ctx(), x, tokens, *out)
    check(x, tokens, out, dtype, 32)


@gpu
@pytest.mark.parametrize("vocab", [50, 1000, 70000])
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16"])
def test_infinities_and_nan(vocab, kind):
    dtype = U.TYPES[kind]
    g = U.gen(2)
    x = U.randn(g, 7, vocab, dtype=dtype)
    x[0, vocab // 2:] = -INF              # half masked
    x[1] = -INF
    x[1, 4] = -2.0                        # one entry left
    x[2] = -INF                           # nothing left
    x[3, 9] = float("nan")
    x[4, 11] = INF
    x[5, :vocab - 3] = -INF               # fewer than `top` left
    tokens = torch.tensor([0, 4, 4, 0, 0, vocab - 1, vocab], device="cuda")   # the last one is out of range
    out = outputs(7, 8, dtype)
    api.tokenLogProbs(U.ctx(), x, tokens, *out)
    lp, lse, ent, tv, ti = out
    keep = [0, 1, 5]
    check(x[keep], tokens[keep], [o[keep] for o in out], dtype, 8)
    assert lse[2] == -INF and lp[2] == -INF and ent[2] == 0
    assert ti[2].tolist() == list(range(8)) and (tv[2] == -INF).all()
    for r in (3, 4):
        assert torch.isnan(lse[r]) or r == 4
        assert torch.isnan(ent[r]) and torch.isnan(lp[r])
    assert 9 not in ti[3].tolist() and ti[4, 0] == 11
    assert torch.isnan(lp[6]) and torch.isfinite(lse[6])
    # the gradient of the same rows
    s = U.stat(dtype)
    dl, de = torch.ones(7, device="cuda", dtype=s), torch.full((7,), 0.5, device="cuda", dtype=s)
    dx = torch.full_like(x, 9.0)
    api.tokenLogProbsBackward(U.ctx(), x, tokens, lse, ent, dl, de, dx)
    assert not dx[2].any()
    assert torch.isfinite(dx[keep]).all() and not dx[0, vocab // 2:].any() and dx[1].abs().max() < 1e-5
    assert torch.isnan(dx[3]).all() and torch.isnan(dx[6]).all()


def gradient_reference(x, tokens, lse, ent, dl, de):
    lp = x.double() - lse.double()[:, None]
    p = torch.exp(lp)
    gl = torch.where(tokens >= 0, dl.double(), 0.0)[:, None] if dl is not None else torch.zeros_like(lp[:, :1])
    hot = torch.zeros_like(p).scatter_(1, tokens.clamp_min(0)[:, None], 1.0)
    g = gl * (hot - p)
    mag = gl.abs() * (hot + p)
    if de is not None:
        term = p * (torch.where(p > 0, lp, 0.0) + ent.double()[:, None])
        g = g - de.double()[:, None] * term
        mag = mag + de.double().abs()[:, None] * p * (torch.where(p > 0, lp, 0.0).abs() + ent.double().abs()[:, None])
    return g, mag * (16 + 4 * torch.where(p > 0, lp, 0.0).abs())


@gpu
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (40, 2000), (5, 8192), (9, 50001), (2, 256000)], ids=str)
@pytest.mark.parametrize("kind", ["f64", "f32", "bf16", "f16"])
def test_backward(shape, kind):
    dtype = U.TYPES[kind]
    rows, vocab = shape
    g = U.gen(vocab + 1)
    x = U.randn(g, rows, vocab, dtype=dtype, scale=3.0)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens[0] = vocab - 1
    if rows > 2:
        tokens[1] = -1
    s = U.stat(dtype)
    lse = torch.logsumexp(x.double(), 1).to(s)
    ent = torch.special.entr(torch.softmax(x.double(), 1)).sum(1).to(s)
    dl, de = U.randn(g, rows, dtype=s), U.randn(g, rows, dtype=s)
    for a, b in ((dl, None), (None, de), (dl, de)):
        want, mag = gradient_reference(x, tokens, lse, ent, a, b)
        tol = U.half_step(dtype) * want.abs() + U.unit(dtype) * mag + U.tiny(dtype)
        for how, other in (("dense", "dense"), ("strided", "strided"), ("odd", "odd"), ("dense", "odd")):
            dx = U.laid_out(torch.full_like(x, 9.0), other)
            api.tokenLogProbsBackward(U.ctx(), U.laid_out(x, how), tokens, lse, ent if b is not None else None, a, b, dx)
            U.close(dx, want, tol)
            assert U.gaps_untouched(dx)
        same = x.clone()
        api.tokenLogProbsBackward(U.ctx(), same, tokens, lse, ent, a, b, same)
        U.close(same, want, tol)


@gpu
def test_gradient_matches_differences():
    g = U.gen(4)
    x = U.randn(g, 3, 41, dtype=torch.float64)
    tokens = torch.tensor([2, -1, 40], device="cuda")
    dl, de = U.randn(g, 3, dtype=torch.float64), U.randn(g, 3, dtype=torch.float64)
    lp, lse, ent, _, _ = outputs(3, 0, torch.float64)

    def value(x_):
        api.tokenLogProbs(U.ctx(), x_, tokens, lp, lse, ent)
        return (dl * lp + de * ent).sum().item()

    value(x)
    dx = torch.empty_like(x)
    api.tokenLogProbsBackward(U.ctx(), x, tokens, lse.clone(), ent.clone(), dl, de, dx)
    for _ in range(3):
        d = U.randn(g, 3, 41, dtype=torch.float64)
        slope = (value(x + 1e-5 * d) - value(x - 1e-5 * d)) / 2e-5   # error of the quotient ~ 1e-9
        assert abs(slope - (dx * d).sum().item()) < 1e-7 * (1 + abs(slope))


@gpu
def test_same_bits_on_a_stream_and_in_a_graph():
    g = U.gen(6)
    cases = [(3, 90000), (200, 1000)]
    xs = [U.randn(g, *s, dtype=torch.bfloat16, scale=3.0) for s in cases]
    toks = [torch.randint(0, s[1], (s[0],), generator=g, device="cuda") for s in cases]
    first = [outputs(s[0], 16, torch.bfloat16) for s in cases]
    second = [outputs(s[0], 16, torch.bfloat16) for s in cases]
    for x, t, o in zip(xs, toks, first):
        api.tokenLogProbs(U.ctx(), x, t, *o)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    c = U.ctx(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for x, t, o in zip(xs, toks, second):
            api.tokenLogProbs(c, x, t, *o)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def refused(status, f, *args, **kw):
    with pytest.raises(api.FitreError) as e:
        f(*args, **kw)
    assert e.value.status == status


def test_refusals_without_a_device():
    c = types.SimpleNamespace(device=0, h=None, lib=None)
    x = torch.zeros(4, 8)
    refused(S.ERR_BAD_ARG, api.tokenLogProbs, c, x, None, torch.zeros(4))
    refused(S.ERR_UNSUPPORTED, api.tokenLogProbs, c, x.long(), None, torch.zeros(4))
    refused(S.ERR_BAD_ARG, api.tokenLogProbsBackward, c, x, None, None, None, None, None, x)
    from fitre_b200 import _lib
    L = _lib.load()
    assert L.fitre_token_logprobs(None, 1, None, 8, None, 4, 8, None, None, None, 0, None, None) == S.ERR_BAD_ARG
    assert L.fitre_token_logprobs_backward(None, 1, None, 8, None, None, None, None, None, None, 8, 4, 8) == S.ERR_BAD_ARG


@gpu
def test_refusals_and_no_rows():
    c = U.ctx()
    x = torch.zeros(4, 40, device="cuda")
    t = torch.zeros(4, device="cuda", dtype=torch.int64)
    s = torch.zeros(4, device="cuda")
    f, b = api.tokenLogProbs, api.tokenLogProbsBackward
    refused(S.ERR_BAD_ARG, f, c, x, None, s)
    refused(S.ERR_BAD_ARG, f, c, x, t)
    refused(S.ERR_BAD_ARG, f, c, x, t.int(), s)
    refused(S.ERR_BAD_ARG, f, c, x, t[:3], s)
    refused(S.ERR_BAD_ARG, f, c, x, t, s.double())
    refused(S.ERR_BAD_ARG, f, c, x, t, s, s, s, torch.zeros(4, 3, device="cuda"))
    refused(S.ERR_BAD_ARG, f, c, x, t, s, s, s, torch.zeros(4, 2, device="cuda"),
            torch.zeros(4, 3, device="cuda", dtype=torch.int64))
    refused(S.ERR_TOO_LARGE, f, c, x, t, s, s, s, torch.zeros(4, 33, device="cuda"),
            torch.zeros(4, 33, device="cuda", dtype=torch.int64))
    refused(S.ERR_BAD_ARG, f, c, x[:, :5], t, s, s, s, torch.zeros(4, 6, device="cuda"),
            torch.zeros(4, 6, device="cuda", dtype=torch.int64))
    refused(S.ERR_BAD_ARG, b, c, x, t, None, None, s, None, x)
    refused(S.ERR_BAD_ARG, b, c, x, t, s, None, None, s, x)
    refused(S.ERR_BAD_ARG, b, c, x, t, s, s, None, None, x)
    refused(S.ERR_BAD_ARG, b, c, x, None, s, s, s, None, x)
    refused(S.ERR_BAD_ARG, b, c, x, t, s, s, s, None, x[:, :39])
    f(c, x[:0], t[:0], s[:0])
    b(c, x[:0], t[:0], s[:0], None, s[:0], None, x[:0])


@gpu
def test_two_streams_at_once():
    """Contexts of their own on two streams: nothing is shared between them."""
    g = U.gen(9)
    xs = [U.randn(g, 120, 30000, dtype=torch.bfloat16, scale=3.0) for _ in range(2)]
    tok = torch.zeros(120, device="cuda", dtype=torch.int64)
    alone = [outputs(120, 8, torch.bfloat16) for _ in xs]
    for x, o in zip(xs, alone):
        api.tokenLogProbs(U.ctx(), x, tok, *o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    ctxs = [U.ctx(s) for s in streams]
    both = [outputs(120, 8, torch.bfloat16) for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, x, o in zip(ctxs, xs, both):
            api.tokenLogProbs(c, x, tok, *o)
    for c in ctxs:
        c.synchronize()
    for a, b in zip(alone, both):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_offsets_beyond_32_bits():
    rows, vocab, ld = 33000, 200, 70000
    g = U.gen(13)
    base = torch.empty(rows * ld, device="cuda", dtype=torch.bfloat16)
    x = base.as_strided((rows, vocab), (ld, 1))
    x.copy_(U.randn(g, rows, vocab, dtype=torch.bfloat16, scale=3.0))
    dense = x.contiguous()
    tok = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    one = torch.ones(rows, device="cuda")
    results = []
    for t in (x, dense):
        out = outputs(rows, 4, torch.bfloat16)
        api.tokenLogProbs(U.ctx(), t, tok, *out)
        dx = torch.empty_like(dense)
        api.tokenLogProbsBackward(U.ctx(), t, tok, out[1], out[2], one, one, dx)
        results.append(out + [dx])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    api.tokenLogProbsBackward(U.ctx(), x, tok, results[0][1], results[0][2], one, one, x)
    assert torch.equal(x, results[0][-1])
