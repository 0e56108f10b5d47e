"""What is measured of the language-model operators: layer norm, token log probabilities, the gated
feed-forward block and the orthogonalised update.  Each case is one pass of one operator; `run`
computes it in elementary torch operations (own = False) or through fitre_b200.api (own = True)."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "f64": 8}
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # the framework's default quintic
SWISH, RELU, SOFTPLUS = 14, 13, 11            # the framework's activation numbers


def listed():
    return [
        # the rows of one decoding step for a few requests: latency
        {"name": "layer norm, few rows", "op": "norm", "rows": 8, "cols": 1024, "type": "f16"},
        # a single-precision run with an unaligned width
        {"name": "layer norm, odd width", "op": "norm", "rows": 20011, "cols": 1023, "type": "f32"},
        # the backward pass of a training step
        {"name": "layer norm gradient", "op": "norm_back", "rows": 16384, "cols": 4096, "type": "bf16"},
        # scoring the tokens that a few requests have just drawn
        {"name": "log probs, few rows", "op": "logp", "rows": 8, "vocab": 128000, "type": "bf16", "top": 20,
         "padded": 0},
        # scoring whole responses, with alternatives
        {"name": "log probs, many rows", "op": "logp", "rows": 4096, "vocab": 128000, "type": "bf16", "top": 8,
         "padded": 0},
        # loss gradient over an odd vocabulary
        {"name": "log prob gradient, odd", "op": "logp_back", "rows": 4099, "vocab": 50001, "type": "bf16",
         "entropy": True, "padded": 0},
        # one token of a serving loop
        {"name": "gated block, one token", "op": "gated", "tokens": 1, "width": 4096, "hidden": 12288,
         "type": "bf16", "act": SWISH, "saved": False},
        # a batch of a training step, pre-activations kept for the backward pass
        {"name": "gated block, batch", "op": "gated", "tokens": 8192, "width": 4096, "hidden": 12288,
         "type": "bf16", "act": SWISH, "saved": True},
        # its backward pass
        {"name": "gated block gradient", "op": "gated_back", "tokens": 4096, "width": 4096, "hidden": 12288,
         "type": "bf16", "act": SWISH},
        # a ragged batch of a small model
        {"name": "gated block gradient, odd", "op": "gated_back", "tokens": 1003, "width": 1000, "hidden": 2730,
         "type": "f16", "act": SWISH},
        # the attention projections of a small model's layers, updated together
        {"name": "orthogonalise, small", "op": "ortho", "batch": 4, "rows": 513, "cols": 384, "type": "f32",
         "steps": 5},
        # one wide layer of a large model
        {"name": "orthogonalise, large", "op": "ortho", "batch": 1, "rows": 4096, "cols": 8192, "type": "bf16",
         "steps": 5},
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v += rng.choice((0, 0, 0, 1)) if v < hi else 0
    r = rng.choice((1, 8, 64))
    return max(lo, min(hi, v // r * r if v >= r else v))


def draw(rng):
    op = rng.choice(("norm", "norm_back", "logp", "logp_back", "gated", "gated_back", "ortho"))
    if op in ("norm", "norm_back"):
        cols = _log(rng, 16, 16384)
        rows = _log(rng, 1, max(1, min(65536, (1 << 26) // cols)))
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(("bf16", "f16", "f32", "f64"))}
    if op in ("logp", "logp_back"):
        vocab = _log(rng, 64, 256000)
        rows = _log(rng, 1, max(1, min(16384, (1 << 28) // vocab)))
        case = {"op": op, "rows": rows, "vocab": vocab, "type": rng.choice(("bf16", "f16", "f32", "f64")),
                "padded": rng.choice((0, 0, 7))}
        if op == "logp":
            case["top"] = rng.choice((0, 1, 5, 20, 32))
        else:
            case["entropy"] = rng.choice((False, True))
        return case
    if op in ("gated", "gated_back"):
        width, hidden = _log(rng, 64, 4096), _log(rng, 64, 12288)
        case = {"op": op, "tokens": _log(rng, 1, 4096), "width": width, "hidden": hidden,
                "type": rng.choice(("bf16", "f16")), "act": rng.choice((SWISH, SWISH, RELU, SOFTPLUS))}
        if op == "gated":
            case["saved"] = rng.choice((False, True))
        return case
    rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
    batch = _log(rng, 1, max(1, min(16, (1 << 24) // (rows * cols))))
    return {"op": op, "batch": batch, "rows": rows, "cols": cols, "type": rng.choice(("bf16", "f16", "f32", "f64")),
            "steps": rng.choice((3, 5, 5))}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    state = dict(case)
    op, dt = case["op"], TYPES[case["type"]]
    make = torch.float64 if case["type"] == "f64" else torch.float32

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=make) * scale

    def new(*shape, dtype=dt):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    stat = make
    if op in ("norm", "norm_back"):
        n, c = case["rows"], case["cols"]
        x = normal(n, c) * (0.5 + torch.rand(n, 1, generator=g, device="cuda", dtype=make)) + normal(n, 1, scale=0.5)
        state["x"] = x.to(dt)
        state["gamma"] = (1 + normal(c, scale=0.1)).to(dt)
        state["beta"] = normal(c, scale=0.1).to(dt)
        state["eps"] = 1e-5
        if op == "norm":
            state["y"], state["mean"], state["rstd"] = new(n, c), new(n, dtype=stat), new(n, dtype=stat)
        else:
            x = state["x"].double()
            mean = x.mean(1)
            state["mean"] = mean.to(stat)
            state["rstd"] = (x.var(1, unbiased=False) + 1e-5).rsqrt().to(stat)
            state["dy"] = normal(n, c).to(dt)
            state["dx"], state["dgamma"], state["dbeta"] = new(n, c), new(c), new(c)
    elif op in ("logp", "logp_back"):
        n, v = case["rows"], case["vocab"]
        x = normal(n, v, scale=2.5)
        x += 6.0 * (torch.rand(n, v, generator=g, device="cuda") < 4.0 / v)   # a few likely tokens
        if case["padded"]:
            x[:, v - case["padded"]:] = -math.inf                              # a vocabulary padded for alignment
        state["logits"] = x.to(dt)
        tokens = torch.randint(0, v - case["padded"], (n,), generator=g, device="cuda")
        if n > 16:
            tokens[torch.rand(n, generator=g, device="cuda") < 0.05] = -1     # rows of padding
        state["tokens"] = tokens
        if op == "logp":
            k = case["top"]
            state["out"] = [new(n, dtype=stat) for _ in range(3)]
            state["out"] += [new(n, k, dtype=stat), new(n, k, dtype=torch.int64)] if k else [None, None]
        else:
            lse, ent = [], []
            for part in state["logits"].split(512):
                lp = torch.log_softmax(part.double(), 1)
                lse.append((part[:, :1].double() - lp[:, :1])[:, 0])
                ent.append(-(lp.exp() * lp.clamp_min(-1e4)).sum(1))
            state["lse"], state["ent"] = torch.cat(lse).to(stat), torch.cat(ent).to(stat)
            state["dlogp"] = normal(n).to(stat)
            state["dent"] = normal(n, scale=0.1).to(stat) if case["entropy"] else None
            state["dlogits"] = new(n, v)
    elif op in ("gated", "gated_back"):
        t, d, f = case["tokens"], case["width"], case["hidden"]
        state["x"] = normal(t, d).to(dt)
        state["wg"] = normal(f, d, scale=d ** -0.5).to(dt)
        state["wu"] = normal(f, d, scale=d ** -0.5).to(dt)
        if op == "gated":
            state["h"] = new(t, f)
            state["g"], state["u"] = (new(t, f), new(t, f)) if case["saved"] else (None, None)
        else:
            state["g"], state["u"] = state["x"] @ state["wg"].T, state["x"] @ state["wu"].T
            state["dh"] = normal(t, f).to(dt)
            state["dx"], state["dwg"], state["dwu"] = new(t, d), new(f, d), new(f, d)
    else:
        b, r, c = case["batch"], case["rows"], case["cols"]
        # a gradient: a few strong directions over a broad floor, as sums of outer products are
        k = max(1, min(r, c) // 8)
        u = normal(b, r, c) + 3.0 * (normal(b, r, k) @ normal(b, k, c)) / math.sqrt(k)
        state["update"] = (0.02 * u).to(dt)
        state["out"] = new(b, r, c, dtype=torch.bfloat16)
    if own:
        from fitre_b200 import api
        state["ctx"] = api.Context(torch.cuda.current_device())
        state["ws"] = None
        if op == "norm_back":
            need = api.layerNormBackwardMemRequired(case["rows"], case["cols"])
        elif op == "gated":
            need = api.gatedForwardMemRequired(case["tokens"], case["width"], case["hidden"])
        elif op == "gated_back":
            need = api.gatedBackwardMemRequired(case["tokens"], case["width"], case["hidden"])
        elif op == "ortho":
            need = api.orthogonalizeMemRequired(case["batch"], case["rows"], case["cols"])
        else:
            need = 0
        if need:
            state["ws"] = torch.empty(need, device="cuda", dtype=torch.float64)
    return state


def _activate(act, g):
    """act(g) and act'(g)."""
    if act == RELU:
        return g.clamp_min(0), (g > 0).to(g.dtype)
    s = 1 / (1 + torch.exp(-g))
    if act == SOFTPLUS:
        return g.clamp_min(0) + torch.log1p(torch.exp(-g.abs())), s
    return g * s, s * (1 + g * (1 - s))


def _top(x, k):
    """The k largest of each row and their places; among equal ones the lowest place first."""
    n = x.shape[1]
    if x.dtype == torch.float64:
        v, at = torch.sort(x, dim=1, descending=True, stable=True)
        return v[:, :k], at[:, :k]
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    key = bits * (1 << 32) + (0x7FFFFFFF - torch.arange(n, device=x.device))
    at = 0x7FFFFFFF - (torch.topk(key, k, dim=1).values & 0x7FFFFFFF)
    return x.gather(1, at), at


def _plain(s):
    op, dt = s["op"], TYPES[s["type"]]
    wide = torch.float64 if s["type"] == "f64" else torch.float32
    if op == "norm":
        x = s["x"].to(wide)
        mean = x.mean(1, keepdim=True)
        xc = x - mean
        rstd = (xc.square().mean(1, keepdim=True) + s["eps"]).rsqrt()
        y = xc * rstd * s["gamma"].to(wide) + s["beta"].to(wide)
        return {"y": y.to(dt), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "norm_back":
        x, dy = s["x"].to(wide), s["dy"].to(wide)
        xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["gamma"].to(wide)
        dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return {"dx": dx.to(dt), "dgamma": (dy * xh).sum(0).to(dt), "dbeta": dy.sum(0).to(dt)}
    if op == "logp":
        x = s["logits"].to(wide)
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - m)
        z = e.sum(1, keepdim=True)
        lse = (m + torch.log(z))[:, 0]
        tok = s["tokens"]
        lp = torch.where(tok >= 0, x.gather(1, tok.clamp_min(0)[:, None])[:, 0] - lse, 0.0)
        shifted = torch.where(e > 0, x - m, 0.0)
        ent = torch.log(z)[:, 0] - (e * shifted).sum(1) / z[:, 0]
        out = {"logp": lp, "lse": lse, "entropy": ent}
        if s["top"]:
            v, at = _top(x, s["top"])
            out["top"], out["top_tokens"] = v - lse[:, None], at
        return out
    if op == "logp_back":
        x = s["logits"].to(wide)
        lp = x - s["lse"][:, None]
        p = torch.exp(lp)
        tok = s["tokens"]
        used = (tok >= 0)
        gl = torch.where(used, s["dlogp"], 0.0)[:, None]
        dx = -gl * p
        if s["entropy"]:
            dx = dx - s["dent"][:, None] * p * (torch.where(p > 0, lp, 0.0) + s["ent"][:, None])
        dx.scatter_add_(1, tok.clamp_min(0)[:, None], gl)
        return dx.to(dt)
    if op == "gated":
        x = s["x"].float()
        g, u = x @ s["wg"].float().T, x @ s["wu"].float().T
        h = (_activate(s["act"], g)[0] * u).to(dt)
        return {"h": h, "g": g.to(dt), "u": u.to(dt)} if s["saved"] else {"h": h}
    if op == "gated_back":
        x, g, u, dh = (s[k].float() for k in ("x", "g", "u", "dh"))
        a, da = _activate(s["act"], g)
        dg, du = dh * u * da, dh * a
        dx = dg @ s["wg"].float() + du @ s["wu"].float()
        return {"dx": dx.to(dt), "dwg": (dg.T @ x).to(dt), "dwu": (du.T @ x).to(dt)}
    x = s["update"].to(torch.float32)
    tall = s["rows"] > s["cols"]
    x = x.transpose(1, 2) if tall else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    a, b, c = NS_COEFFICIENTS
    for _ in range(s["steps"]):
        y = x @ x.transpose(1, 2)
        x = a * x + (b * y + c * (y @ y)) @ x
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16)


def run(state):
    s = state
    if not own:
        return _plain(s)
    from fitre_b200 import api
    op, ctx = s["op"], s["ctx"]
    if op == "norm":
        api.layerNormForward(ctx, s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"], s["eps"])
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "norm_back":
        api.layerNormBackward(ctx, s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"], s["dgamma"],
                              s["dbeta"], s["ws"])
        return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if op == "logp":
        lp, lse, ent, top, at = s["out"]
        api.tokenLogProbs(ctx, s["logits"], s["tokens"], lp, lse, ent, top, at)
        out = {"logp": lp, "lse": lse, "entropy": ent}
        if s["top"]:
            out["top"], out["top_tokens"] = top, at
        return out
    if op == "logp_back":
        api.tokenLogProbsBackward(ctx, s["logits"], s["tokens"], s["lse"], s["ent"], s["dlogp"], s["dent"],
                                  s["dlogits"])
        return s["dlogits"]
    if op == "gated":
        api.gatedForward(ctx, s["x"], s["wg"], s["wu"], s["h"], s["g"], s["u"], s["act"], s["ws"])
        return {"h": s["h"], "g": s["g"], "u": s["u"]} if s["saved"] else {"h": s["h"]}
    if op == "gated_back":
        api.gatedBackward(ctx, s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], s["dx"], s["dwg"], s["dwu"],
                          s["act"], s["ws"])
        return {"dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"]}
    api.orthogonalizeUpdate(ctx, s["update"], s["out"], s["ws"], s["steps"])
    return s["out"]


def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op in ("norm", "norm_back"):
        n, c = case["rows"], case["cols"]
        if op == "norm":
            return {"bytes": 2 * n * c * e + 2 * c * e + 2 * n * max(4, e), "flops": 8 * n * c}
        return {"bytes": 3 * n * c * e + 3 * c * e + 2 * n * max(4, e), "flops": 14 * n * c}
    if op == "logp":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * e + n * (8 + 3 * max(4, e) + case["top"] * (8 + max(4, e))), "flops": 5 * n * v}
    if op == "logp_back":
        n, v = case["rows"], case["vocab"]
        return {"bytes": 2 * n * v * e + n * (8 + 4 * max(4, e)), "flops": 6 * n * v}
    if op in ("gated", "gated_back"):
        t, d, f = case["tokens"], case["width"], case["hidden"]
        if op == "gated":
            return {"bytes": e * (t * d + 2 * f * d + t * f * (3 if case["saved"] else 1)), "flops": 4 * t * d * f}
        return {"bytes": e * (2 * t * d + 4 * f * d + 3 * t * f), "flops": 8 * t * d * f}
    b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # the two symmetric products need one triangle each
    return {"bytes": b * m * n * (e + 2), "flops": case["steps"] * b * (3 * m * m * n + m * m * m)}


def exact(case, seed):
    """The outputs in 64 bits from the definitions; row blocks keep the memory down."""
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    op = case["op"]
    f64 = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()
           and op not in ("logp", "logp_back")}
    if op == "norm":
        var, mean = torch.var_mean(f64["x"], 1, unbiased=False, keepdim=True)
        std = torch.sqrt(var + s["eps"])
        return {"y": (f64["x"] - mean) / std * f64["gamma"] + f64["beta"], "mean": mean[:, 0], "rstd": 1 / std[:, 0]}
    if op == "norm_back":
        r = f64["rstd"][:, None]
        unit = (f64["x"] - f64["mean"][:, None]) * r
        dunit = f64["dy"] * f64["gamma"]
        c = case["cols"]
        along = torch.einsum("ij,ij->i", dunit, unit)[:, None]
        dx = (c * dunit - dunit.sum(1, keepdim=True) - unit * along) * r / c
        return {"dx": dx, "dgamma": torch.einsum("ij,ij->j", f64["dy"], unit), "dbeta": f64["dy"].sum(0)}
    if op == "logp":
        cols = {"logp": [], "lse": [], "entropy": [], "top": []}
        for part, tok in zip(s["logits"].split(256), s["tokens"].split(256)):
            x = part.double()
            lse = torch.logsumexp(x, 1)
            lp = torch.log_softmax(x, 1)
            cols["lse"].append(lse)
            picked = torch.gather(lp, 1, tok.clamp_min(0)[:, None])[:, 0]
            cols["logp"].append(picked.masked_fill(tok < 0, 0.0))
            cols["entropy"].append(torch.special.entr(lp.exp()).sum(1))
            if case["top"]:
                cols["top"].append(torch.topk(lp, case["top"], 1).values)
        out = {k: torch.cat(v) for k, v in cols.items() if v}
        if case["top"]:
            out["top_tokens"] = None
        return out
    if op == "logp_back":
        out = torch.empty(case["rows"], case["vocab"], device="cuda", dtype=torch.float64)
        for at in range(0, case["rows"], 256):
            part = slice(at, min(at + 256, case["rows"]))
            lp = s["logits"][part].double() - s["lse"][part].double()[:, None]
            p = lp.exp()
            tok = s["tokens"][part]
            gl = s["dlogp"][part].double().masked_fill(tok < 0, 0.0)[:, None]
            hot = torch.zeros_like(p).scatter_(1, tok.clamp_min(0)[:, None], 1.0)
            out[part] = gl * (hot - p)
            if case["entropy"]:
                out[part] += s["dent"][part].double()[:, None] * (
                    torch.special.entr(p) - p * s["ent"][part].double()[:, None])
        return out
    if op == "gated":
        g, u = torch.mm(f64["x"], f64["wg"].t()), torch.mm(f64["x"], f64["wu"].t())
        h = _act64(case["act"], g)[0] * u
        return {"h": h, "g": g, "u": u} if case["saved"] else {"h": h}
    if op == "gated_back":
        a, slope = _act64(case["act"], f64["g"])
        dg, du = f64["dh"] * f64["u"] * slope, f64["dh"] * a
        return {"dx": torch.mm(dg, f64["wg"]) + torch.mm(du, f64["wu"]), "dwg": torch.mm(dg.t(), f64["x"]),
                "dwu": torch.mm(du.t(), f64["x"])}
    x = f64["update"]
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + 1e-7)
    a, b, c = NS_COEFFICIENTS
    for _ in range(case["steps"]):
        # the same polynomial from whichever side is the smaller
        if case["rows"] <= case["cols"]:
            y = torch.bmm(x, x.mT)
            x = a * x + b * torch.bmm(y, x) + c * torch.bmm(y, torch.bmm(y, x))
        else:
            y = torch.bmm(x.mT, x)
            x = a * x + b * torch.bmm(x, y) + c * torch.bmm(torch.bmm(x, y), y)
    return x


def _act64(act, g):
    if act == RELU:
        return torch.relu(g), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    if act == SOFTPLUS:
        return torch.logaddexp(g, torch.zeros_like(g)), torch.sigmoid(g)
    s = torch.sigmoid(g)
    return g * s, s + g * s * torch.sigmoid(-g)
