"""A policy's clipped loss and its gradient against plain 64-bit forms, at the sizes, masks and values where the kernels can go
wrong.

Bounds, derived before the first run (S = sum_error of the row's columns):
- ln p has the error D = S + E (4 |ln p| + 8 |lse|) that log probabilities have, the entropy 4 S (1 + H);
- a ratio's exponent adds E |ln p - old| to D, its exponential 4 E; a product of the loss rounds once, 2 E with its conversion;
- exp(d) - 1 - d moves by |exp(d) - 1| for each unit of d, and rounds its parts: 4 E |exp(d) - 1| + 2 E |d|;
- a gradient's p has the relative error 2 S + E (8 |ln p| + 8 |lse|), its slope c the errors above, and the products 8 E.
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
    """A policy's rows: some of padding, ratios on both sides of their bounds but not at them."""

    def __init__(self, m, n, dtype, T=1.0, clip=(0.2, 0.28), kl=0.1, entropy=0.05, padding=0.2, masked=0.0, seed=0):
        g = gen(seed + m * 7 + n)
        self.dtype, self.T, self.clip, self.kl, self.entropy = dtype, T, clip, kl, entropy
        self.x = (2.5 * randn(g, m, n)).to(TYPES[dtype])
        self.ids = torch.randint(0, n, (m,), generator=g, device="cuda")
        if masked:
            own = self.x.gather(1, self.ids[:, None])
            self.x.masked_fill_(torch.rand((m, n), generator=g, device="cuda") < masked, float("-inf"))
            self.x.scatter_(1, self.ids[:, None], own)
        out = torch.rand(m, generator=g, device="cuda") < padding
        self.ids[out] = torch.where(self.ids[out] % 2 == 0, -1, n)
        now = softmax64(self.x, T)[1].gather(1, self.ids.clamp(0, n - 1)[:, None])[:, 0]
        moved = 0.3 * randn(g, m).double()
        for border in (np.log(max(1 - clip[0], 1e-9)), np.log(1 + clip[1])):
            moved = torch.where((moved - border).abs() < 1e-2, border + 2e-2, moved)
        self.old = torch.where(torch.isfinite(now), now - moved, 0.0).float()
        self.ref = torch.where(torch.isfinite(now), now + 0.3 * randn(g, m), 0.0).float()
        self.adv, self.grad_loss = randn(g, m), randn(g, m)

    @property
    def args(self):
        return self.x, self.ids, self.old, self.adv

    @property
    def how(self):
        return dict(ref_log_probs=self.ref, clip=self.clip, kl=self.kl, entropy=self.entropy, temperature=self.T)

    def exact(self):
        """(values and bounds of loss, log_probs, entropy, lse; gradient and its bound)."""
        n = self.x.shape[1]
        use = (self.ids >= 0) & (self.ids < n)
        at = torch.where(use, self.ids, 0).long()[:, None]
        T, S = float(np.float32(self.T)), sum_error(n)
        lse, logp, p = softmax64(self.x, T)
        size = torch.where(torch.isfinite(lse), lse.abs(), 0.0)
        ln = torch.where(p > 0, logp, 0.0)
        h = -(p * ln).sum(1)
        now = logp.gather(1, at)[:, 0]
        old, adv, ref = self.old.double(), self.adv.double(), self.ref.double()
        r = (now - old).exp()
        low, high = 1 - self.clip[0], 1 + self.clip[1]
        bound = torch.where(adv < 0, low, high)
        clipped = torch.where(adv < 0, r < bound, r > bound)
        near = (now.abs() < 1e30) * now.nan_to_num(neginf=0.0).abs()
        D = S + E * (4 * near + 8 * size)
        dr = D + E * ((near + old.abs()) + 4)
        kept = torch.where(clipped, bound, r)
        loss = -adv * kept
        slope = torch.where(clipped, 0.0, -adv * r)
        dl = adv.abs() * kept * (dr + 3 * E)
        ds = torch.where(clipped, 0.0, adv.abs() * r * (dr + 3 * E))
        if self.kl:
            d = ref - now
            e = d.exp() - 1
            loss = loss + self.kl * (e - d)
            slope = slope - self.kl * e
            dl = dl + abs(self.kl) * (e.abs() * (D + E * d.abs()) + 6 * E * e.abs() + 4 * E * d.abs() + 2 * D * D)
            ds = ds + abs(self.kl) * ((e + 1) * (D + E * d.abs()) + 6 * E * e.abs())
        dh = 4 * S * (1 + h)
        if self.entropy:
            loss = loss - self.entropy * h
            dl = dl + abs(self.entropy) * (dh + 2 * E * h)
        dl = dl + 4 * E * loss.abs()
        w = self.entropy
        one = torch.zeros_like(p).scatter_(1, at, 1.0)
        inner = torch.where(p > 0, ln + h[:, None], 0.0)
        grad = slope[:, None] * (one - p) + w * p * inner
        rel = 2 * S + E * (8 * ln.abs() + 8 * size[:, None])
        terms = slope.abs()[:, None] * (one + p) + abs(w) * p * (ln.abs() + h[:, None])
        tol = rel * p * (slope.abs()[:, None] + abs(w) * (ln.abs() + h[:, None] + 1)) + ds[:, None] * (one + p) \
            + abs(w) * p * dh[:, None] + 12 * E * terms
        k = (self.grad_loss.double() / T)[:, None]
        grad, tol = torch.where(use[:, None], grad * k, 0.0), torch.where(use[:, None], tol * k.abs(), 0.0)
        values = [(loss, dl), (now, D), (h, dh), (lse, S + 4 * E * size)]
        return [(torch.where(use, v, 0.0), torch.where(use, t, 0.0)) for v, t in values], grad, tol

    def check(self, O, x=None):
        values, grad, tol = self.exact()
        x = self.x if x is None else x
        args = (x, *self.args[1:])
        r = O.policy_loss(*args, **self.how)
        back = O.policy_loss_backward(self.grad_loss, *args, r, **self.how)
        step, both = O.policy_step(self.grad_loss, *args, **self.how)
        for res, dx, which in ((r, back, "apart"), (step, both, "in one call")):
            for name, (want, t) in zip(res._fields, values):
                close(getattr(res, name), want, t + 1e-37, f"{name} {which}")
            assert dx.dtype == self.x.dtype
            close(dx, grad, rounded(tol, grad, self.dtype), f"gradient {which}")


# rows of few columns; in a wavefront, 256 or 1024 threads, held or in parts; more rows than workgroups
SIZES = [(3, 1), (5, 3), (4, 8), (7, 9), (3, 65), (2100, 5), (2100, 700), (2100, 3001), (2100, 7001), (5, 3001), (300, 20_011),
         (40, 30_001), (20, 60_003), (3, 65_537), (600, 100_003), (4, 131_079), (2, 200_003)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_values_and_gradients(O, m, n, dtype):
    Rows(m, n, dtype, T=[1.0, 0.7, 2.0][n % 3]).check(O)


@pytest.mark.parametrize("m,n", [(3, 7), (5, 1000), (4, 70_001), (600, 9001)])
@pytest.mark.parametrize("kl,entropy", [(0.0, 0.0), (0.3, 0.0), (0.0, 0.2), (-0.1, -0.1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_terms(O, m, n, kl, entropy, dtype):
    Rows(m, n, dtype, kl=kl, entropy=entropy, padding=0.5).check(O)


@pytest.mark.parametrize("clip", [(0.0, 0.0), (1.0, 0.5), (0.2, float("inf"))])
def test_bounds_of_ratios(O, clip):
    Rows(64, 300, "float32", clip=clip).check(O)


@pytest.mark.parametrize("pad", [1, 5, 64])
@pytest.mark.parametrize("m,n", [(3, 3), (3, 1000), (3, 40_000), (2100, 300), (3, 140_000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart(O, m, n, pad, dtype):
    r = Rows(m, n, dtype)
    r.check(O, padded(r.x, pad))


@pytest.mark.parametrize("m,n", [(8, 5), (8, 3000), (8, 100_003), (600, 9001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_columns(O, m, n, dtype):
    Rows(m, n, dtype, masked=0.7).check(O)


@pytest.mark.parametrize("n", [5, 1000, 70_001])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_infinities_and_nan(O, n, dtype):
    low = torch.finfo(TYPES[dtype]).min
    r = Rows(8, n, dtype, kl=0.0, entropy=0.1, padding=0.0)
    r.ids[:] = torch.arange(8, device="cuda") % n
    r.x[0] = float("-inf")
    r.x[1] = low
    r.x[2, 2] = float("-inf")  # the id of the row
    r.x[3] = float("-inf")
    r.x[3, 3] = 1.0  # nothing but the id
    r.x[4, 0] = float("nan")
    r.x[5, n - 1] = float("inf")
    r.x[6] = float("nan")
    r.ids[6] = -1  # padding, whatever its row holds
    r.x[7, 1:] = low
    finite = torch.tensor([0, 1, 2, 3, 6, 7], device="cuda")
    got, dx = O.policy_step(r.grad_loss, *r.args, **r.how)
    apart = O.policy_loss(*r.args, **r.how)
    for res, grad in ((got, dx), (apart, O.policy_loss_backward(r.grad_loss, *r.args, apart, **r.how))):
        for v in res:
            assert torch.isnan(v[4:6]).all() and v[6] == 0
        assert torch.isnan(grad[4:6]).all() and (grad[6] == 0).all()
        assert torch.isfinite(grad[finite]).all()
        assert res.log_probs[0] == float("-inf") and res.lse[0] == float("-inf") and res.entropy[0] == 0
        assert (grad[0] == 0).all()  # no probability anywhere
        assert res.log_probs[2] == float("-inf") and res.log_probs[3] == 0 and (grad[3] == 0).all()
        # ratio 0: the loss is that of the bound, or of nothing
        for row in (0, 2):
            want = -min(0.0, r.adv[row].item() * 0.8) if r.adv[row] >= 0 else -r.adv[row].item() * (1 - r.clip[0])
            assert abs(res.loss[row].item() + r.entropy * res.entropy[row].item() - want) < 1e-5
    r.x[4:6] = 0
    values, grad, tol = r.exact()
    for name, (want, t) in zip(got._fields[1:], values[1:]):
        close(getattr(got, name)[finite], want[finite], t[finite] + 1e-37, name)
    close(dx[finite], grad[finite], rounded(tol, grad, dtype)[finite], "gradient")


@pytest.mark.parametrize("n", [5, 3000, 140_000])
def test_kl_of_an_impossible_id(O, n):
    """Its loss is infinite, and its row's gradient says so."""
    r = Rows(3, n, "float32", kl=0.1, padding=0.0)
    r.ids[:] = 1
    r.x[1, 1] = float("-inf")
    res, grad = O.policy_step(r.grad_loss, *r.args, **r.how)
    assert res.loss[1] == float("inf") and not torch.isfinite(grad[1, 1]) and torch.isfinite(res.loss[[0, 2]]).all()
    assert torch.isfinite(grad[[0, 2]]).all()


def test_ratio_at_its_bound_counts_as_unclipped(O):
    """Two equal logits: ln p = -ln 2 to the last place, so that exp(ln p - old) can be made 1 exactly; both bounds 1."""
    x = torch.zeros((4, 2), device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    now = O.log_probs(x, ids).log_probs
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    old = now.clone()
    old[2] -= 0.1  # a ratio above its bound, which the loss of a positive advantage does not follow
    old[3] += 0.1
    r, grad = O.policy_step(torch.ones(4, device="cuda"), x, ids, old, adv, clip=0.0)
    assert torch.equal(r.loss, -adv)
    want = torch.tensor([[-0.5, 0.5], [0.5, -0.5], [0, 0], [0, 0]], device="cuda")
    assert torch.equal(grad, want)


def test_a_sampled_policy_is_unmoved(O):
    """With old the policy's own log probabilities the loss is -A and its gradient that of -A ln p."""
    r = Rows(33, 1000, "float32", kl=0.0, entropy=0.0, padding=0.0)
    old = O.policy_step(r.grad_loss, r.x, r.ids, r.adv, r.adv)[0].log_probs
    res, grad = O.policy_step(r.grad_loss, r.x, r.ids, old, r.adv)
    assert torch.equal(res.loss, -r.adv) and torch.equal(res.log_probs, old)
    own = O.log_probs(r.x, r.ids)
    want = O.log_probs_backward(-r.adv * r.grad_loss, None, r.x, r.ids, own.lse, own.entropy)
    close(grad, want, 4 * sum_error(1000) * want.abs() + 1e-9, "gradient")


@pytest.mark.parametrize("T", [1.0, 1.5])
def test_gradients_against_differences(O, T):
    """(f(x + h) - f(x - h)) / 2 h of the 64-bit loss: h^2 / 6 of a third derivative of at most about 10, and 1e-15 / h."""
    r = Rows(6, 7, "float32", T=T, padding=0.0)
    grad = O.policy_step(r.grad_loss, *r.args, **r.how)[1]
    h = 1e-4
    x = r.x.double()
    for i in range(6):
        for j in range(7):
            f = []
            for sign in (1, -1):
                r.x = x.clone()
                r.x[i, j] += sign * h
                f.append((r.exact()[0][0][0] * r.grad_loss.double()).sum())
            assert abs(((f[0] - f[1]) / (2 * h)).item() - grad[i, j].item()) < 1e-5 * (1 + abs(grad[i, j].item()))


def test_operands_of_other_kinds(O):
    r = Rows(9, 120, "float32")
    want, grad = O.policy_step(r.grad_loss, *r.args, **r.how)
    host = [v.cpu().numpy() for v in (r.grad_loss, *r.args)]
    how = dict(r.how, ref_log_probs=r.ref.cpu().numpy())
    got, dx = O.policy_step(*host, **how)
    assert isinstance(dx, np.ndarray) and np.array_equal(dx, grad.cpu().numpy())
    for a, b in zip(got, want):
        assert np.array_equal(a, b.cpu().numpy())
    got, dx = O.policy_step(r.grad_loss.double(), r.x, r.ids[:, None].int(), r.old.double(), r.adv.double(),
                            **dict(r.how, clip=list(r.clip)))
    assert torch.equal(dx, grad) and torch.equal(got.loss, want.loss)
    strided = torch.stack([r.ids, r.ids * 0 - 1], 1)[:, 0]
    assert torch.equal(O.policy_loss(r.x, strided, r.old, r.adv, **r.how).loss, want.loss)


def test_no_rows(O):
    empty = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    r, grad = O.policy_step(empty(0), empty(0, 30), empty(0, dtype=torch.int64), empty(0), empty(0))
    assert grad.shape == (0, 30) and all(v.shape == (0,) for v in r)


@pytest.mark.parametrize("m,n", [(2, 140_000), (600, 9001), (2100, 700)])
def test_results_repeat_on_any_stream(O, m, n):
    r = Rows(m, n, "bfloat16")
    want, grad = O.policy_step(r.grad_loss, *r.args, **r.how)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(O.policy_step(r.grad_loss, *r.args, **r.how))
    torch.cuda.synchronize()
    for res, dx in got:
        assert torch.equal(dx, grad) and all(torch.equal(a, b) for a, b in zip(res, want))


@pytest.mark.parametrize("m,n", [(2, 140_000), (40, 3000), (600, 9001)])
def test_captured_calls_replay(O, m, n):
    r = Rows(m, n, "float32")

    def work():
        res = O.policy_loss(*r.args, **r.how)
        return [*res, O.policy_loss_backward(r.grad_loss, *r.args, res, **r.how), *O.policy_step(r.grad_loss, *r.args, **r.how)[0],
                O.policy_step(r.grad_loss, *r.args, **r.how)[1]]

    graph, out = captured(work)
    for seed in range(3):
        fresh = Rows(m, n, "float32", seed=seed + 1)
        r.x.copy_(fresh.x), r.ids.copy_(fresh.ids), r.old.copy_(fresh.old), r.adv.copy_(fresh.adv), r.ref.copy_(fresh.ref)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, work()))


def test_rows_beyond_32_bit_offsets(O):
    m, n, stride = 5, 1000, 1_200_000_000
    r = Rows(m, n, "float16", padding=0.0)
    flat = torch.zeros((m - 1) * stride + n, dtype=torch.float16, device="cuda")
    x = flat.as_strided((m, n), (stride, 1))
    x.copy_(r.x)
    r.check(O, x)


def test_refusals(O):
    r = Rows(4, 20, "float32")
    step = lambda **k: O.policy_step(**{**dict(zip(("grad_loss", "logits", "ids", "old_log_probs", "advantages"),
                                                   (r.grad_loss, *r.args))), **k})
    for change, error, text in [
        (dict(ids=r.ids[:3]), ValueError, "ids has shape"), (dict(ids=torch.stack([r.ids, r.ids], 1)), ValueError, "ids has shape"),
        (dict(ids=r.adv), TypeError, "int64 or int32"), (dict(advantages=r.adv[:3]), ValueError, "advantages has shape"),
        (dict(old_log_probs=r.old[None]), ValueError, "old_log_probs must be a vector"),
        (dict(grad_loss=r.adv[:1]), ValueError, "grad_loss has shape"), (dict(kl=0.1), RuntimeError, "ref_log_probs"),
        (dict(kl=0.1, ref_log_probs=r.ref[:2]), ValueError, "ref_log_probs has shape"),
        (dict(kl=float("nan"), ref_log_probs=r.ref), RuntimeError, "finite"), (dict(entropy=float("inf")), RuntimeError, "finite"),
        (dict(clip=1.5), RuntimeError, "bounds"), (dict(clip=(-0.1, 0.2)), RuntimeError, "bounds"),
        (dict(clip=(0.2, -0.1)), RuntimeError, "bounds"), (dict(clip=float("nan")), RuntimeError, "bounds"),
        (dict(temperature=0.0), RuntimeError, "temperature"), (dict(logits=torch.zeros((4, 0), device="cuda")), RuntimeError, "columns"),
    ]:
        with pytest.raises(error, match=text):
            step(**change)


@pytest.mark.parametrize("m,n", [(800, 2), (800, 3000), (60, 140_000)])
def test_kl_of_near_policies_keeps_its_digits(O, m, n):
    """exp(d) - 1 - d where d is given exactly (the id's ln p is 0), from 1e-17 to 80 of both signs; kl 1, A 0: the loss itself.

    Bound: up to 1/2 by its series, d * d (E) times a sum (2 E, whose coefficients add E) rounds once more (E); from there on by
    expm1, whose unit in the last place (2 E |e|) weighs |e| / k <= 4.4 times, and a difference (E): 10 E."""
    size = torch.logspace(-17, np.log10(80.0), m // 2, dtype=torch.float64, device="cuda").float()
    ref = torch.cat([size, -size])
    x = torch.full((m, n), -1000.0, device="cuda")
    x[:, 0] = 0
    ids, none = torch.zeros(m, dtype=torch.int64, device="cuda"), torch.zeros(m, device="cuda")
    d = ref.double()
    series = sum(d**j / float(np.prod(np.arange(1.0, j + 3))) for j in range(12)) * d * d
    want = torch.where(d.abs() < 0.2, series, torch.expm1(d) - d)
    for r in (O.policy_loss(x, ids, none, none, ref_log_probs=ref, kl=1.0),
              O.policy_step(none, x, ids, none, none, ref_log_probs=ref, kl=1.0)[0]):
        assert (r.log_probs == 0).all() and (r.loss >= 0).all()
        close(r.loss, want, 10 * E * want, "KL term")
