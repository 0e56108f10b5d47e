"""Shared by the tests of the language-model operators: contexts, odd layouts, error bounds.

Bounds are of the form  half a step of the output type * |value|  +  k * u * (sum of the magnitudes
that went into the value),  u the unit roundoff of the arithmetic (2^-24, fp64 tensors 2^-53).
A sum whose longest chain of additions has n terms is off by at most n * u times the sum of the
magnitudes; the kernels' chains are <= 40 terms per thread plus <= 16 levels of joins unless a test says
otherwise, so k = 64 covers a sum and the few elementwise roundings around it."""
import torch

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CTX = {}


def ctx(stream=None):
    from fitre_b200 import api
    if stream is not None:
        return api.Context(torch.cuda.current_device(), stream.cuda_stream)
    if "c" not in _CTX:
        _CTX["c"] = api.Context(torch.cuda.current_device())
    return _CTX["c"]


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the spacing of the type's subnormal numbers (what a rounding near zero can lose), and what
    flushing the arithmetic's own subnormals can."""
    return {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -125)


def stat(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64) * scale).to(dtype)


def laid_out(t, how):
    """The same matrix with another layout: 'dense'; 'strided': rows a whole number of 16-byte units
    apart; 'odd': rows and base off the 16-byte grid.  The gaps hold a sentinel."""
    if how == "dense":
        return t.contiguous().clone()
    rows, cols = t.shape
    per = 16 // t.element_size()
    width = (cols + per - 1) // per * per + 2 * per if how == "strided" else cols + 2 * per + 1
    shift = per if how == "strided" else 1
    buf = torch.full((rows, width), 77.0, dtype=t.dtype, device=t.device)
    view = buf[:, shift:shift + cols]
    view.copy_(t)
    return view


def gaps_untouched(view):
    """The elements around a laid_out view still hold the sentinel."""
    base = view._base
    if base is None:
        return True
    shift = view.storage_offset()
    seen = base.clone()
    seen[:, shift:shift + view.shape[1]] = 77.0
    return bool((seen == 77.0).all())


def close(got, want, tol):
    """Every element of `got` within `tol` of `want` (fp64); NaN and infinities in the same places."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    other = ~fine & ~torch.isnan(want)
    assert torch.equal(got[other], want[other]), "infinities in other places"
    d = (got - want).abs()[fine]
    t = tol.expand_as(want)[fine] if torch.is_tensor(tol) else torch.full_like(d, tol)
    worst = (d / t.clamp_min(1e-300)).max().item() if d.numel() else 0.0
    assert bool((d <= t).all()), "error %.3g of the bound" % worst
    return worst
