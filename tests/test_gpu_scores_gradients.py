"""Gradients from a saved log-sum-exp l: p is that of the given l.

With e = 2^-24, beside the rounding of l itself, which is the caller's: the difference x - l T, its product with log2(e) / T and
that factor round three times, 3 e |ln p|; the power of two adds 2 e, what l T loses less than e, and the products of a gradient
3 e more: p (8 e + 4 e |ln p|).
"""

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


@pytest.mark.parametrize("n", [5, 1000, 40_000])
@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
@pytest.mark.parametrize("level", [-99.0, -33.0, 0.0, 13.0, 33.0, 60.0, 99.0])
def test_probabilities_of_a_saved_log_sum_exp(O, n, T, level):
    g = torch.Generator().manual_seed(n)
    m = 8
    lse = (level + 0.9 * torch.rand(m, generator=g)).float()
    z = lse.double()[:, None] - 12 * torch.rand((m, n), generator=g, dtype=torch.float64)
    x = (z * T).float()
    T32 = torch.tensor(T).double()  # the temperature that the call gets
    lnp = x.double() / T32 - lse.double()[:, None]
    p = lnp.exp()
    none = torch.full((m, 1), -1)
    bound = p * E * (8 + 4 * lnp.abs())

    def close(got, want, tol, what):
        err = (got.cpu().double() - want).abs()
        assert (err <= tol).all(), f"{what}: off by {err.max():.3e}, {(err / tol).max():.1f} of its bound"

    zero, w = torch.zeros((m, 1)).cuda(), torch.full((m,), 1.0)
    # entropy's gradient is -p (ln p + H) / T: the H that makes it p times a number of some size
    h = torch.full((m,), 20.0)
    got = O.log_probs_backward(None, w.cuda(), x.cuda(), none.cuda(), lse.cuda(), h.cuda(), temperature=T)
    close(-got * T, p * (lnp + 20), bound * 20 + p * E * 4 * (20 + lnp.abs()), "of the entropy")
    ids = torch.zeros((m, 1), dtype=torch.int64)
    got = O.log_probs_backward(w[:, None].cuda(), None, x.cuda(), ids.cuda(), lse.cuda(), h.cuda(), temperature=T)
    close(-got[:, 1:] * T, p[:, 1:], (bound + p * E)[:, 1:], "of log probabilities")
    got = O.distill_backward(w.cuda(), x.cuda(), ids.cuda(), zero, lse.cuda(), temperature=T)
    close(got[:, 1:] * T, p[:, 1:], (bound + p * E)[:, 1:], "of distillation")
