"""What the tests of the operators at both ends of a training step share: comparisons against 64-bit forms, which are computed
on the GPU from elementary operations, and matrices whose rows lie apart.

E = 2^-24 is half a unit in the last place of 32 bits; results of 16 bits add half a unit in theirs: 2^-11 (float16, and 2^-25
near 0) or 2^-8 (bfloat16, and less than 1e-37 near 0)."""

import pytest
import torch

E = 2.0**-24
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HALF = {"float32": (E, 1e-37), "float16": (2.0**-11, 2.0**-25), "bfloat16": (2.0**-8, 1e-37)}


def package():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd

    return octex_amd


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def close(got, want, tol, what):
    """got (any type) within tol (elementwise) of want (64 bits); infinities and NaN in the same places."""
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = torch.as_tensor(tol, dtype=torch.float64, device=want.device).expand(want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = torch.isfinite(want)
    err, tol = (got - want).abs()[ok], tol[ok]
    assert (err <= tol).all(), f"{what}: off by {err.max():.3e}, {(err / tol.clamp_min(1e-300)).max():.2f} of its bound"


def rounded(tol, want, dtype):
    """A bound of 32-bit arithmetic, widened by the result's rounding to dtype."""
    rel, floor = HALF[dtype]
    return tol * (1 + rel) + rel * want.abs() + floor


def padded(t, pad, fill=7.0):
    """The same matrix as a slice of a wider one: rows `pad` elements further apart, at odd places."""
    if pad == 0:
        return t.clone()
    wide = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device="cuda")
    wide[:, 1 : 1 + t.shape[1]] = t
    return wide[:, 1 : 1 + t.shape[1]]


def softmax64(x, T=1.0):
    """lse, log p and p of rows of logits in 64 bits; a row of nothing has p = 0."""
    z = x.double() / T
    top = z.max(1, keepdim=True).values
    nothing = torch.isinf(top) & (top < 0)
    ref = torch.where(nothing, 0.0, top)
    s = torch.exp(z - ref).sum(1, keepdim=True)
    lse = torch.where(nothing, top, ref + torch.log(s))
    masked = z == float("-inf")
    logp = torch.where(masked, torch.where(torch.isnan(lse), lse, z), (z - ref) - torch.log(s))
    return lse[:, 0], logp, torch.where(masked, torch.where(torch.isnan(lse), lse, 0.0), logp.exp())


def sum_error(n):
    """Of a sum of n exponentials: a thread adds n / 256 of them at most, each addition adds E; exponents are rounded twice (their
    size times 2 E, which the terms' weights make small) and exponentials by 2 E."""
    return (n / 256 + 64) * E


def captured(work):
    """A graph of `work`, run once before on the stream it is captured on."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    return graph, out
