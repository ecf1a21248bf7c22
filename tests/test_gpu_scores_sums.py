"""Sums over long rows of scores: their error does not grow with the row.

With e = 2^-24: an exponential is off by 2 e and, its exponent being the rounded product of an exact difference with a rounded
factor, by 2 e of |z - max| (6 at most here); eight are added to each other (4.5 e) and up to 16 such sums again (8.5 e), then to
the thread's, which keeps what an addition loses (2 e); a row's sums are joined in 14 additions: under 45 e of the sum.
A logarithm adds 2 e of its size, and so do lse's and log
p's own additions.  The weighted sum has the same errors and 1 e of its product.  So
  lse, log p:  45 e + 4 e (|lse| + |z|)
  entropy:     45 e + 4 e |ln s| + 100 e of |sum p (z - max)|
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

E = 2.0**-24


@pytest.fixture(scope="module")
def O():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd

    return octex_amd


def rows_of(m, n, dtype, base):
    """Rows whose every 1000th score is `base`, so that all threads meet it, and all others the same of base - 6 to base - 0.5;
    how many there are of the former, and the difference."""
    below = torch.linspace(-6, -0.5, m, dtype=torch.float64).mul(64).round().div(64)
    x = (below + base).to(dtype).cuda()[:, None].repeat(1, n)
    x[:, ::1000] = base
    return x, -(-n // 1000), x[:, 1].cpu().double() - base


# rows that a workgroup reads by itself, and rows that 32 share: 16,384 scores a thread
@pytest.mark.parametrize("m,n", [(129, (1 << 22) + 5), (3, (1 << 27) + 1)])
@pytest.mark.parametrize("dtype,base", [(torch.bfloat16, 0.0), (torch.float32, 0.0), (torch.float32, 256.0)])
def test_sums_of_long_rows(O, m, n, dtype, base):
    x, many, below = rows_of(m, n, dtype, base)
    p1 = torch.exp(below)
    s = many + (n - many) * p1
    ln_s, t = torch.log(s), (n - many) * p1 * below / s
    lse, h = base + ln_s, ln_s - t
    ids = torch.tensor([[0, 1, n - 2]]).repeat(m, 1).cuda()
    logp = torch.stack([-ln_s, below - ln_s, below - ln_s], 1)
    bound = 45 * E + 4 * E * (base + ln_s.abs() + 6)

    def close(got, want, tol, what):
        err = (got.cpu().double() - want).abs()
        assert (err <= tol).all(), f"{what}: off by {err.max():.3e}, bound {torch.as_tensor(tol).min():.3e}"

    r = O.log_probs(x, ids, top=2)
    close(r.lse, lse, bound, "lse")
    close(r.log_probs, logp, bound[:, None], "log_probs")
    close(r.entropy, h, 45 * E + 4 * E * ln_s + 100 * E * t.abs(), "entropy")
    one = torch.zeros((m, 1)).cuda()
    loss, lse2 = O.distill(x, ids[:, :1], one)
    close(lse2, lse, bound, "distillation's lse")
    close(loss, ln_s, bound, "loss")
    # at base 256 the gradient makes the sums again; p within their error and 8 e |ln p| of its exponent's
    if base:
        w = torch.ones(m).cuda()
        p = torch.stack([torch.exp(-ln_s) - 1, torch.exp(below - ln_s), torch.exp(below - ln_s)], 1)
        grad = O.distill_backward(w, x, ids[:, :1], one, lse2)
        close(grad.gather(1, ids), p, (45 * E + 8 * E * logp.abs()) * torch.exp(logp) + 2 * E * p.abs(), "gradient")
    del x
    torch.cuda.empty_cache()
