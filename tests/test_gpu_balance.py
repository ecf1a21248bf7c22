"""The balance of rows over experts against a plain 64-bit form.

Bounds, derived before the first run (S = sum_error of the row's logits, l its log-sum-exp):
- a probability has the relative error R = 2 S + E (8 |ln p| + 8 |l|), and l the error S + 4 E |l|;
- a mean probability adds the rows of a lane, at most m / 1024 + 1 of them, and a few joins: (m / 1024 + 64) E of it beside R's;
- the sum over f P rounds in 64 bits, so that the loss has its terms' errors and E of itself;
- a gradient multiplies p by a difference of f and a sum of f p, whose terms have R and 40 E more.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from operators64 import E, TYPES, captured, close, gen, package, padded, randn, rounded, softmax64, sum_error  # noqa: E402


@pytest.fixture(scope="module")
def O():
    return package()


class Rows:
    def __init__(self, m, e, k, dtype, padding=0.2, dropped=0.1, weight=0.7, z=0.3, seed=0):
        g = gen(seed + m * 3 + e * 5 + k)
        self.dtype, self.weight, self.z = dtype, weight, z
        self.x = (1.5 * randn(g, m, e) + randn(g, 1, e)).to(TYPES[dtype])
        self.experts = torch.randint(0, e, (m, k), generator=g, device="cuda")
        self.experts[torch.rand((m, k), generator=g, device="cuda") < dropped] = -1
        self.experts[torch.rand((m, k), generator=g, device="cuda") < dropped / 2] = e
        self.experts[torch.rand(m, generator=g, device="cuda") < padding] = -1
        self.grad_loss = torch.tensor(m * 3.0, device="cuda")

    @property
    def how(self):
        return dict(weight=self.weight, z_weight=self.z)

    def exact(self):
        m, e = self.x.shape
        w, zw = float(np.float32(self.weight)), float(np.float32(self.z))
        chosen = (self.experts >= 0) & (self.experts < e)
        use = chosen.any(1)
        rows = int(use.sum())
        counts = torch.bincount(self.experts[chosen].long(), minlength=e)
        f = counts.double() / max(1, int(counts.sum()))
        lse, logp, p = softmax64(self.x)
        p = torch.where(use[:, None], p, 0.0)
        some = use & ~(torch.isinf(lse) & (lse < 0))
        l = torch.where(some, lse, 0.0)
        S = sum_error(e)
        rel = 2 * S + E * (8 * torch.where(p > 0, logp.abs(), 0.0) + 8 * l.abs()[:, None])
        per = max(rows, 1)
        P = p.sum(0) / per
        dP = (p * rel).sum(0) / per + (m / 1024 + 64) * E * P
        loss = w * e * (f * P).sum() + zw * (l * l).sum() / per
        dl = S + 4 * E * l.abs()
        dloss = abs(w) * e * (f * dP).sum() + abs(zw) * ((2 * l.abs() * dl + 4 * E * l * l).sum() / per
                                                         + (m / 1024 + 64) * E * (l * l).sum() / per)
        dloss = dloss + 4 * E * (abs(w) * e * (f * P).sum() + abs(zw) * (l * l).sum() / per)
        inner = p @ f
        dinner = (p * rel) @ f + 40 * E * inner
        g = self.grad_loss.double() / per
        grad = g * p * (w * e * (f[None] - inner[:, None]) + 2 * zw * l[:, None])
        size = abs(w) * e * (f[None] + inner[:, None]) + 2 * abs(zw) * l.abs()[:, None]
        tol = g.abs() * p * (size * (rel + 12 * E) + abs(w) * e * dinner[:, None] + 2 * abs(zw) * dl[:, None])
        return dict(loss=(loss, dloss), counts=counts, rows=rows, probs=(P, dP), lse=(torch.where(use, lse, 0.0), dl)), grad, tol

    def check(self, O, x=None, experts=None):
        want, grad, tol = self.exact()
        args = (self.x if x is None else x, self.experts if experts is None else experts)
        r = O.balance_loss(*args, **self.how)
        back = O.balance_loss_backward(self.grad_loss, *args, r, **self.how)
        step, both = O.balance_step(self.grad_loss, *args, **self.how)
        for res, dx, which in ((r, back, "apart"), (step, both, "in one call")):
            assert res.counts.dtype == res.rows.dtype == torch.int64
            assert torch.equal(res.counts, want["counts"]) and int(res.rows) == want["rows"], which
            for name in ("loss", "probs", "lse"):
                close(getattr(res, name), *[t + 1e-37 * i for i, t in enumerate(want[name])], f"{name} {which}")
            assert dx.dtype == self.x.dtype
            close(dx, grad, rounded(tol, grad, self.dtype), f"gradient {which}")


EXPERTS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 60, 64, 65, 127, 128, 200, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2047, 2048]


@pytest.mark.parametrize("e", EXPERTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_and_gradients(O, e, dtype):
    for m, k in ((1, 1), (5, 2), (300, min(e, 8)), (5000, min(e, 3))):
        Rows(m, e, k, dtype).check(O)


@pytest.mark.parametrize("m,e,k", [(70_001, 256, 8), (40_000, 1000, 2), (20_001, 2048, 1), (600_000, 8, 2), (300_001, 60, 6)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_rows(O, m, e, k, dtype):
    """More rows than the workgroups of a launch take at a time."""
    Rows(m, e, k, dtype).check(O)


@pytest.mark.parametrize("m,e,k", [(10, 4, 0), (10, 4, 7), (3000, 8, 70), (2000, 3, 512), (40, 300, 512), (1000, 2000, 100)])
def test_choices_of_any_number(O, m, e, k):
    Rows(m, e, k, "float32", padding=0.5).check(O)


@pytest.mark.parametrize("weight,z", [(0.0, 0.0), (1.0, 0.0), (0.0, 1.0), (-0.5, -0.1)])
@pytest.mark.parametrize("m", [20, 6000])
def test_weights(O, m, weight, z):
    Rows(m, 40, 2, "float32", weight=weight, z=z).check(O)


@pytest.mark.parametrize("pad", [1, 5, 64])
@pytest.mark.parametrize("m,e", [(7, 3), (7, 60), (4000, 257), (900, 1300)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart(O, m, e, pad, dtype):
    r = Rows(m, e, 4, dtype)
    wide = torch.full((m, 4 + pad), 1, dtype=torch.int32, device="cuda")
    wide[:, :4] = r.experts
    r.check(O, padded(r.x, pad), wide[:, :4])


@pytest.mark.parametrize("m", [3, 5000])
def test_no_row_counts(O, m):
    r = Rows(m, 10, 2, "float32", padding=1.1)
    got, grad = O.balance_step(r.grad_loss, r.x * float("nan"), r.experts, **r.how)
    assert got.loss == 0 and (got.counts == 0).all() and got.rows == 0 and (got.probs == 0).all() and (got.lse == 0).all()
    assert (grad == 0).all()


def test_no_rows(O):
    x, experts = torch.zeros((0, 6), device="cuda"), torch.zeros((0, 2), dtype=torch.int64, device="cuda")
    got, grad = O.balance_step(None, x, experts, z_weight=1.0)
    assert got.loss == 0 and got.rows == 0 and torch.equal(got.counts, torch.zeros(6, dtype=torch.int64, device="cuda"))
    assert (got.probs == 0).all() and got.lse.shape == (0,) and grad.shape == (0, 6)
    assert O.balance_loss_backward(None, x, experts, got).shape == (0, 6)


@pytest.mark.parametrize("m", [9, 5000])
@pytest.mark.parametrize("e", [6, 100, 700])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_infinities_and_nan(O, m, e, dtype):
    r = Rows(m, e, 2, dtype, padding=0.0, dropped=0.0)
    r.x[0] = float("-inf")
    r.x[1, 1:] = float("-inf")
    r.x[2, torch.arange(e, device="cuda") % 3 > 0] = float("-inf")
    r.x[3] = torch.finfo(TYPES[dtype]).min
    r.z = 0.0  # the lowest value's square passes 32 bits
    r.check(O)
    r.z = 0.3
    r.x[3] = 0
    r.check(O)
    r.experts[4] = -1
    r.x[4] = float("nan")  # a row that does not count
    r.check(O)
    want, grad, tol = r.exact()
    r.x[5, e // 2], r.x[6, 0] = float("nan"), float("inf")
    for res, dx in (O.balance_step(r.grad_loss, r.x, r.experts, **r.how),):
        assert torch.isnan(res.loss) and torch.isnan(res.probs).all() and torch.isnan(res.lse[5:7]).all()
        assert torch.isnan(dx[5:7]).all()
        keep = torch.ones(m, dtype=torch.bool, device="cuda")
        keep[5:7] = False
        close(dx[keep], grad[keep], rounded(tol, grad, dtype)[keep], "gradient of the others")


def test_even_rows_have_loss_one(O):
    e = 16
    x = torch.zeros((160, e), device="cuda")
    r, grad = O.balance_step(None, x, torch.arange(160, device="cuda") % e)
    assert abs(r.loss.item() - 1) < 1e-6 and torch.equal(r.counts, torch.full((e,), 10, device="cuda"))
    assert grad.abs().max() < 1e-8


def test_counts_of_a_whole_job(O):
    """Two ranks' gradients from the sums of their counts and rows are those of all rows together."""
    a, b = Rows(500, 30, 2, "float32", seed=1), Rows(700, 30, 2, "float32", seed=2)
    x, experts = torch.cat([a.x, b.x]), torch.cat([a.experts, b.experts])
    whole, want = O.balance_step(a.grad_loss, x, experts, **a.how)
    ra, rb = O.balance_loss(a.x, a.experts, **a.how), O.balance_loss(b.x, b.experts, **a.how)
    both = ra._replace(counts=ra.counts + rb.counts, rows=ra.rows + rb.rows)
    assert torch.equal(both.counts, whole.counts) and torch.equal(both.rows, whole.rows)
    got = torch.cat([O.balance_loss_backward(a.grad_loss, r.x, r.experts, both, **a.how) for r in (a, b)])
    assert torch.equal(got, want)


def test_gradients_against_differences(O):
    """(f(x + h) - f(x - h)) / 2 h of the 64-bit loss, whose third derivative is at most about 10."""
    r = Rows(6, 5, 2, "float32", padding=0.3)
    r.grad_loss = torch.tensor(2.0, device="cuda")
    grad = O.balance_step(r.grad_loss, r.x, r.experts, **r.how)[1]
    x, h = r.x.double(), 1e-4
    for i in range(6):
        for j in range(5):
            f = []
            for sign in (1, -1):
                r.x = x.clone()
                r.x[i, j] += sign * h
                f.append(2 * r.exact()[0]["loss"][0].item())
            assert abs((f[0] - f[1]) / (2 * h) - grad[i, j].item()) < 1e-5


def test_operands_of_other_kinds(O):
    r = Rows(50, 20, 3, "float32")
    want, grad = O.balance_step(r.grad_loss, r.x, r.experts, **r.how)
    got, dx = O.balance_step(r.grad_loss.item(), r.x.cpu().numpy(), r.experts.int().cpu().numpy(), **r.how)
    assert isinstance(dx, np.ndarray) and np.array_equal(dx, grad.cpu().numpy()) and got.loss == want.loss.item()
    assert np.array_equal(got.counts, want.counts.cpu().numpy())
    back = O.balance_loss_backward(r.grad_loss.cpu().numpy(), r.x.cpu().numpy(), r.experts.cpu().numpy(), got, **r.how)
    assert np.array_equal(back, dx)
    one = O.balance_loss(r.x, r.experts[:, 0])
    assert torch.equal(one.counts, O.balance_loss(r.x, r.experts[:, :1]).counts)
    half = O.balance_step(r.grad_loss.double()[None], r.x, r.experts, **r.how)[1]
    assert torch.equal(half, grad)
    unit = O.balance_step(None, r.x, r.experts, **r.how)[1]
    assert torch.equal(unit, O.balance_step(torch.ones((), device="cuda"), r.x, r.experts, **r.how)[1])


@pytest.mark.parametrize("m,e", [(30, 20), (9000, 200)])
def test_results_repeat_on_any_stream_and_replay(O, m, e):
    r = Rows(m, e, 2, "bfloat16")
    work = lambda: [*O.balance_loss(r.x, r.experts, **r.how), *O.balance_step(r.grad_loss, r.x, r.experts, **r.how)[0],
                    O.balance_step(r.grad_loss, r.x, r.experts, **r.how)[1]]
    want = work()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph, out = captured(work)
    for seed in range(3):
        fresh = Rows(m, e, 2, "bfloat16", seed=seed + 1)
        r.x.copy_(fresh.x), r.experts.copy_(fresh.experts)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work()))


def test_rows_beyond_32_bit_offsets(O):
    r = Rows(5, 300, 2, "float16")
    flat = torch.zeros(4 * 1_200_000_000 + 300, dtype=torch.float16, device="cuda")
    x = flat.as_strided((5, 300), (1_200_000_000, 1))
    x.copy_(r.x)
    r.check(O, x)


def test_refusals(O):
    r = Rows(4, 20, 2, "float32")
    res = O.balance_loss(r.x, r.experts)
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    for args, how, error, text in [
        ((r.x, r.experts[:3]), {}, ValueError, "experts of 3 rows"), ((r.x, r.x), {}, TypeError, "int64 or int32"),
        ((z(4, 2049), r.experts), {}, RuntimeError, "2048"), ((z(4, 0), r.experts), {}, RuntimeError, "columns"),
        ((r.x, z(4, 513, dtype=torch.int64)), {}, RuntimeError, "512"),
        ((r.x, r.experts), dict(weight=float("nan")), RuntimeError, "finite"),
        ((r.x, r.experts), dict(z_weight=float("inf")), RuntimeError, "finite"),
    ]:
        with pytest.raises(error, match=text):
            O.balance_loss(*args, **how)
        with pytest.raises(error, match=text):
            O.balance_step(None, *args, **how)
    with pytest.raises(ValueError, match="grad_loss"):
        O.balance_step(z(2), r.x, r.experts)
    with pytest.raises(ValueError, match="counts"):
        O.balance_loss_backward(None, r.x, r.experts, res._replace(counts=res.counts[:3]))
    with pytest.raises(TypeError, match="counts must be int64"):
        O.balance_loss_backward(None, r.x, r.experts, res._replace(counts=res.counts.float()))


@pytest.mark.parametrize("m,e", [(9, 6), (40, 700), (5000, 6), (5000, 100), (900, 1300), (40_000, 60), (40_000, 500)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count_have_no_gradient(O, m, e, dtype):
    """Whatever the loss weighs: an overflowed loss scale leaves a batch's padding at 0."""
    r = Rows(m, e, 2, dtype, padding=0.4)
    r.experts[0], r.experts[1] = 0, -1
    use = ((r.experts >= 0) & (r.experts < e)).any(1)
    res = O.balance_loss(r.x, r.experts, **r.how)
    for size in (float("inf"), float("-inf"), float("nan")):
        g = torch.tensor(size, device="cuda")
        for grad in (O.balance_loss_backward(g, r.x, r.experts, res, **r.how), O.balance_step(g, r.x, r.experts, **r.how)[1]):
            assert (grad[~use] == 0).all() and not torch.isfinite(grad[0]).any()
