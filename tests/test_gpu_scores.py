"""The operators on rows of scores (octex_amd/scores.py) against plain 64-bit forms, at the sizes, strides, masks and values
where their kernels can go wrong.

Tolerances, with e = 2^-24 (half a unit in the last place of 32 bits), derived before the first run:
- a product in 8 bits has an exact sum, its conversion, two products and the bias round once each: 4 e of |product| + |bias|;
- a sum of n exponentials takes a thread n / 256 additions at the least split, each adding e; its exponents are rounded
  twice (their size times 2 e, which the terms' weights make small) and its exponentials by 2 e: (n / 256 + 64) e of the sum,
  and the logarithm adds as much as a difference.  Log probabilities add 4 e of |z - max| and 2 e of |lse|;
- a gradient's probability has that relative error and 4 e |ln p| of its exponent's; shares add 8 e each;
- results of 16 bits add half a unit in their last place: 2^-11 (float16, and 2^-25 near 0) or 2^-8 / 2 (bfloat16).
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

E = 2.0**-24
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HALF = {"float32": (E, 0.0), "float16": (2.0**-11, 2.0**-25), "bfloat16": (2.0**-8, 0.0)}


@pytest.fixture(scope="module")
def O():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd

    return octex_amd


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, tol, what):
    """got (any type) within tol (elementwise) of want (64 bits); infinities and NaN in the same places."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = torch.isfinite(want)
    err = (got - want).abs()
    worst = ((err - tol) * ok.nan_to_num()).nan_to_num(nan=0.0, posinf=1e300) if want.numel() else err
    assert (err[ok] <= tol[ok]).all(), f"{what}: off by {err[ok].max():.3e}, over its bound by {worst.max():.3e}"


def padded(t, pad, fill=7.0):
    """The same matrix as a slice of a wider one on the GPU: rows `pad` elements further apart."""
    if pad == 0:
        return t.cuda()
    wide = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device="cuda")
    wide[:, : t.shape[1]] = t.cuda()
    return wide[:, : t.shape[1]]


# ------------------------------------------------------------------------------------------------------- 8-bit products


def codes_of(x):
    """The definition: 32-bit scale and quotients, whole numbers by ties to even."""
    x = x.float().numpy()
    scale = np.abs(x).max(1) * (np.float32(1) / np.float32(127))  # as torch's division by a number on the GPU
    safe = np.where(scale > 0, scale, np.float32(1)).astype(np.float32)
    c = np.clip(np.rint((x / safe[:, None]).astype(np.float32)), -127, 127)
    return torch.from_numpy(np.where(scale[:, None] > 0, c, 0).astype(np.int8)), torch.from_numpy(scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,pad", [(1, 1, 0), (3, 7, 0), (5, 16, 3), (2, 1000, 1), (4, 4096, 0), (300, 65, 0), (2, 20011, 5)])
def test_quantize_rows(O, dtype, m, k, pad):
    x = (torch.randn((m, k), generator=gen(k)) * 3).to(TYPES[dtype])
    if m > 1:
        x[1] = 0
    codes, scales = O.quantize_rows(padded(x, pad))
    want, ws = codes_of(x)
    assert torch.equal(codes.cpu(), want) and torch.equal(scales.cpu(), ws)


@pytest.mark.parametrize("k", [15, 31, 127, 128, 129, 255, 256, 257, 1023, 1025, 2047, 2048, 2049, 4095, 4097, 8193])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_of_every_width(O, dtype, k):
    """Rows that 16, 64 or 256 threads hold, and quotients at and beside the middle of two whole numbers."""
    g = gen(k)
    x = torch.randn((37, k), generator=g) * torch.logspace(-30, 3, 37)[:, None].clamp(min=1e-3 if dtype == "float16" else 0)
    x[::3] = torch.randint(-254, 255, x[::3].shape, generator=g) / 2  # halves: a scale of 1 where 127 is among them
    x[::3, 0] = 127
    x[5] = 0
    x = x.to(TYPES[dtype])
    codes, scales = O.quantize_rows(padded(x, 1))
    want, ws = codes_of(x)
    assert torch.equal(codes.cpu(), want) and torch.equal(scales.cpu(), ws)


def test_quantize_extremes(O):
    top = torch.finfo(torch.float32).max
    x = torch.zeros((7, 33))
    x[0, 5], x[0, 6] = top, -top / 2
    x[1, 32] = float("inf")
    x[2, 0] = float("nan")
    x[3, 3] = 1e-44  # its scale rounds to 0
    x[4] = 2.0**-126 * torch.arange(33)
    x[5, 1] = 190 * 2.0**-149  # a scale of one subnormal unit: the quotient passes 127
    x[6] = torch.arange(33) - 16.5
    codes, scales = O.quantize_rows(x.cuda())
    codes, scales = codes.cpu(), scales.cpu()
    assert torch.isnan(scales[1:3]).all() and (codes[1:3] == 0).all()
    keep = [0, 3, 4, 5, 6]
    want, ws = codes_of(x[keep])
    assert torch.equal(codes[keep], want) and torch.equal(scales[keep], ws)
    rows = torch.ones((4, 33), dtype=torch.int8).cuda()
    s = O.int8_scores(x.cuda(), rows, torch.ones(4).cuda())
    assert torch.isnan(s[1:3]).all() and torch.isfinite(s[3:]).all()


SHAPES = [(1, 1, 1), (1, 16, 5), (1, 1024, 300), (2, 100, 17), (3, 33, 64), (7, 128, 65), (15, 511, 1000), (16, 512, 130),
          (17, 64, 31), (33, 1001, 257), (64, 256, 64), (65, 129, 190), (100, 96, 1000), (130, 960, 513), (257, 384, 300),
          (300, 48, 700), (512, 2048, 512), (5, 4097, 700), (1, 20000, 40)]


def score_tolerance(prod, bias, dtype):
    rel, floor = HALF[dtype]
    return 4 * E * (prod.abs() + (bias.abs() if bias is not None else 0)) + rel * (prod + (bias if bias is not None else 0)).abs() \
        + floor


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_of_codes(O, m, k, n, dtype):
    g = gen(m * 7 + k + n)
    q = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    r = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8)
    qs, rs = torch.rand(m, generator=g) * 0.01, torch.rand(n, generator=g) * 0.01
    bias = torch.randn(n, generator=g) if n % 2 else None
    prod = (q.double() @ r.double().T) * qs.double()[:, None] * rs.double()
    want = prod + bias.double() if bias is not None else prod
    tol = score_tolerance(prod, bias.double() if bias is not None else None, dtype)
    for pad in (0, 1, 16):  # rows side by side, at odd addresses, 16 bytes further apart
        got = O.int8_scores(padded(q, pad, 99), padded(r, pad, 77), rs.cuda(), query_scales=qs.cuda(),
                            bias=None if bias is None else bias.cuda(), dtype=dtype)
        assert got.dtype == TYPES[dtype]
        close(got, want, tol, f"scores, rows {pad} bytes apart")


@pytest.mark.parametrize("m,k,n", [(1, 64, 50), (1, 1001, 3), (9, 960, 100), (70, 100, 200), (300, 512, 300), (1, 9000, 64),
                                   (2, 16384, 33)])
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_of_floats(O, m, k, n, dtype):
    g = gen(m + k * n)
    x = torch.randn((m, k), generator=g).to(TYPES[dtype])
    r = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    rs = torch.rand(n, generator=g)
    codes, scales = codes_of(x)
    prod = (codes.double() @ r.double().T) * scales.double()[:, None] * rs.double()
    rel, floor = HALF[dtype]
    got = O.int8_scores(padded(x, 3), r.cuda(), rs.cuda())
    assert got.dtype == TYPES[dtype]
    close(got, prod, (4 * E + rel) * prod.abs() + floor, "scores of floats")


@pytest.mark.parametrize("m,k,n,pad", [
    (600, 1040, 12345, 0), (2050, 4112, 4100, 0), (1000, 512, 30001, 16), (300, 100, 20001, 0), (70, 1001, 140_000, 0),
    (40, 999, 3000, 1), (2000, 64, 2000, 0), (130, 16, 70_001, 0), (9, 8192, 9000, 0),
])
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_of_every_tiling(O, m, k, n, pad, dtype):
    """Products large enough for every tiling, ragged at every edge, rows in place and laid out anew in several parts."""
    g = torch.Generator("cuda").manual_seed(m + n)
    q = torch.randint(-128, 128, (m, k + pad), generator=g, dtype=torch.int8, device="cuda")[:, :k]
    r = torch.randint(-128, 128, (n, k + pad), generator=g, dtype=torch.int8, device="cuda")[:, :k]
    qs, rs = torch.rand(m, generator=g, device="cuda") * 0.01, torch.rand(n, generator=g, device="cuda") * 0.01
    bias = torch.randn(n, generator=g, device="cuda")
    got = O.int8_scores(q, r, rs, query_scales=qs, bias=bias, dtype=dtype)
    rel, floor = HALF[dtype]
    for a in range(0, m, 256):
        prod = torch.mm(q[a : a + 256].double(), r.double().t()) * qs[a : a + 256].double()[:, None] * rs.double()
        want = prod + bias.double()
        err = (got[a : a + 256].double() - want).abs()
        tol = 4 * E * (prod.abs() + bias.double().abs()) + rel * want.abs() + floor
        assert (err <= tol).all(), f"queries {a}: off by {err.max():.3e}"


@pytest.mark.parametrize("m,k,n", [(17, 960, 20_001), (32, 128, 8257), (3, 4112, 9001), (16, 64, 70_003), (33, 80, 9000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_int8_scores_of_thin_batches(O, m, k, n, dtype):
    test_int8_scores_of_every_tiling(O, m, k, n, 0, dtype)


def test_int8_scores_at_the_ends_of_their_sums(O):
    k = 131071  # the widest rows: sums of -128 x -128 just stay under 2^31
    q = torch.full((2, k), -128, dtype=torch.int8)
    q[1] = 127
    r = torch.full((3, k), -128, dtype=torch.int8)
    got = O.int8_scores(q.cuda(), r.cuda(), torch.ones(3).cuda(), query_scales=torch.ones(2).cuda())
    want = q.double() @ r.double().T
    close(got, want, E * want.abs(), "the largest sums")


def test_scores_rank_as_distances(O):
    """With bias = -|row|^2 / 2 the scores' order is that of the 8-bit vectors' squared distances."""
    g = gen(5)
    X, Q = torch.randn((500, 96), generator=g), torch.randn((20, 96), generator=g)
    rc, rs = O.quantize_rows(X.cuda())
    qc, qs = O.quantize_rows(Q.cuda())
    x8, q8 = rc.cpu().double() * rs.cpu().double()[:, None], qc.cpu().double() * qs.cpu().double()[:, None]
    bias = (-0.5 * (x8 * x8).sum(1)).float()
    s = O.int8_scores(Q.cuda(), rc, rs, bias=bias.cuda()).cpu()
    d = torch.cdist(q8, x8, compute_mode="donot_use_mm_for_euclid_dist")
    assert (s.argmax(1) == d.argmin(1)).all()


# ------------------------------------------------------------------------------------------------------ log probabilities


def softmax64(x, T):
    """z, lse, log p and p of rows of logits in 64 bits; a row of nothing has p = 0."""
    z = x.double() / T
    top = z.max(1, keepdim=True).values
    ref = torch.where(torch.isinf(top) & (top < 0), 0.0, top)
    s = torch.exp(z - ref).sum(1, keepdim=True)
    lse = ref + torch.log(s)
    lse = torch.where(torch.isinf(top) & (top < 0), top, lse)
    # not z - lse, which loses ln s beside the lowest value of a type in 64 bits too
    logp = torch.where(z == float("-inf"), torch.where(torch.isnan(lse), lse, z), (z - ref) - torch.log(s))
    return z, lse[:, 0], logp, torch.where(z == float("-inf"), torch.where(torch.isnan(lse), lse, 0.0), logp.exp())


def entropy64(logp, p):
    return -torch.where(p > 0, p * logp, p).sum(1)


def top64(x, top):
    """(logit, lowest id) order by a stable sort; -1 where the logit is -inf or there is none."""
    at = torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    at = torch.where(x.gather(1, at) == float("-inf"), -1, at)
    return torch.nn.functional.pad(at, (0, top - at.shape[1]), value=-1)


def sum_error(n):
    return (n / 256 + 64) * E


def check_log_probs(r, x, ids, T, top):
    z, lse, logp, p = softmax64(x, T)
    n = x.shape[1]
    inside = (ids >= 0) & (ids < n)
    at = torch.where(inside, ids, 0).long()
    want = torch.where(inside, logp.gather(1, at), 0.0)
    spread = torch.where(torch.isfinite(lse), lse.abs(), 0.0)[:, None]
    far = torch.where(torch.isfinite(want), want.abs(), 0.0)
    close(r.log_probs.reshape(want.shape), want, sum_error(n) + E * (4 * far + 8 * spread), "log_probs")
    close(r.lse, lse, sum_error(n) + 4 * E * spread[:, 0], "lse")
    h = entropy64(logp, p)
    close(r.entropy, h, 4 * sum_error(n) * (1 + torch.where(torch.isfinite(h), h, 0.0)), "entropy")
    assert r.top_ids.shape == r.top_log_probs.shape == (x.shape[0], top) and r.top_ids.dtype == torch.int64
    if top:
        want = top64(x, top)
        bad = torch.isnan(lse)
        want[bad] = -1
        assert torch.equal(r.top_ids.cpu(), want), "top ids"
        lp = torch.where(want >= 0, logp.gather(1, want.clamp_min(0)), float("-inf"))
        lp[bad] = float("nan")
        far = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
        close(r.top_log_probs, lp, sum_error(n) + E * (4 * far + 8 * spread), "top_log_probs")


COLUMNS = [1, 2, 3, 7, 8, 9, 63, 64, 65, 500, 511, 512, 513, 1000, 2047, 2049, 8191, 8192, 8200, 32000, 50021, 131072, 200003]


@pytest.mark.parametrize("n", COLUMNS)
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs(O, n, dtype):
    g = gen(n)
    m, T = 3, [1.0, 0.7, 2.0][n % 3]
    x = (3 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    ids = torch.randint(0, n, (m, 4), generator=g)
    ids[0, 1], ids[1, 2], ids[2, 3] = -1, n, 0
    for top, pad in ((0, 0), (1, 1), (5, 3), (20, 0), (64, 8)):
        check_log_probs(O.log_probs(padded(x, pad), ids.cuda(), top=top, temperature=T), x, ids, T, top)


@pytest.mark.parametrize("m", [1, 2, 31, 300, 1200])
def test_log_probs_of_many_rows(O, m):
    g = gen(m)
    x = (2 * torch.randn((m, 3001), generator=g)).bfloat16()
    ids = torch.randint(0, 3001, (m, 1), generator=g)
    r = O.log_probs(x.cuda(), ids[:, 0].int().cuda(), top=7)
    assert r.log_probs.shape == (m,)
    check_log_probs(r, x, ids, 1.0, 7)


@pytest.mark.parametrize("m,n,t", [(129, 20_000, 1), (500, 1200, 2), (2500, 700, 130), (2500, 4096, 3), (2048, 5, 1),
                                   (1025, 4097, 300)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_log_probs_of_every_grouping(O, m, n, t, dtype):
    """A wavefront, 256 or 512 threads a row: values, alternatives and gradients."""
    g = gen(m + n)
    x = (2 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    x[m // 2] = float("-inf")
    ids = torch.randint(-1, n, (m, t), generator=g)
    r = O.log_probs(x.cuda(), ids.cuda(), top=20, temperature=1.3)
    check_log_probs(r, x, ids, 1.3, 20)
    gl, gh = torch.randn((m, t), generator=g), torch.randn(m, generator=g)
    want, tol = grad64(x, ids, 1.3, gl, gh)
    got = O.log_probs_backward(gl.cuda(), gh.cuda(), x.cuda(), ids.cuda(), r.lse, r.entropy, temperature=1.3)
    close(got, want, gradient_tolerance(want, tol, dtype), "gradient")


@pytest.mark.parametrize("n", [40, 1000, 9000, 70000])
@pytest.mark.parametrize("dtype", TYPES)
def test_top_of_equal_and_sorted_scores(O, n, dtype):
    """Ties go to the lowest id, wherever the equal scores lie; ascending rows raise the floor at every step."""
    g = gen(n)
    x = torch.zeros((7, n))
    x[1] = torch.randint(0, 3, (n,), generator=g)
    x[2] = torch.arange(n) % 7 - 3
    x[3, ::2] = -0.0  # equal to 0
    x[4] = torch.arange(n) / n * 50
    x[5] = -torch.arange(n) / n * 50
    x[6, n // 2] = 1
    x = x.to(TYPES[dtype])
    ids = torch.zeros((7, 1), dtype=torch.int64)
    for top in (1, 20, 64):
        check_log_probs(O.log_probs(x.cuda(), ids.cuda(), top=top), x, ids, 1.0, top)


@pytest.mark.parametrize("m,n", [(2100, 1000), (2100, 4001), (600, 9000), (300, 9000)])
def test_top_of_equal_and_sorted_scores_of_every_grouping(O, m, n):
    g = gen(m + n)
    x = torch.randint(0, 3, (m, n), generator=g).float()
    x[::4] = torch.arange(n) / n * 50
    x[1::4] = -torch.arange(n) / n * 50
    x[2::8] = 0
    ids = torch.zeros((m, 1), dtype=torch.int64)
    for top in (3, 64):
        check_log_probs(O.log_probs(x.cuda(), ids.cuda(), top=top), x, ids, 1.0, top)


@pytest.mark.parametrize("n", [5, 77, 1030, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_infinities_and_nan(O, n, dtype):
    g = gen(n)
    low = torch.finfo(TYPES[dtype]).min
    x = torch.randn((10, n), generator=g)
    x[0] = float("-inf")
    x[1] = low
    x[2, 1:] = float("-inf")
    x[3, :-1] = low
    x[4, torch.rand(n, generator=g) < 0.7] = float("-inf")
    x[5, torch.rand(n, generator=g) < 0.7] = low
    x[6, n // 3] = float("nan")
    x[7, n // 2] = float("inf")
    x[8, :-1] = float("-inf")
    x[9, 0] = -low  # the type's highest value
    x = x.to(TYPES[dtype])
    ids = torch.stack([torch.zeros(10, dtype=torch.int64), torch.full((10,), n - 1), torch.arange(10) % n], 1)
    with np.errstate(all="ignore"):
        z, lse, logp, p = softmax64(x, 1.0)
    lse[6] = lse[7] = float("nan")
    r = O.log_probs(x.cuda(), ids.cuda(), top=3)
    finite = torch.tensor([0, 1, 2, 3, 4, 5, 8, 9])
    check_log_probs(type(r)(*(v.cpu()[finite] for v in r)), x[finite], ids[finite], 1.0, 3)
    for v in (r.log_probs, r.entropy, r.lse, r.top_log_probs):
        assert torch.isnan(v[6:8]).all()
    assert (r.top_ids[6:8] == -1).all() and (r.top_ids[0] == -1).all()
    assert r.entropy[0] == 0 and r.lse[0] == float("-inf") and (r.log_probs[0] == float("-inf")).all()
    assert abs(r.entropy[1].item() - math.log(n)) < 1e-5  # a row of the lowest value is uniform


def grad64(x, ids, T, gl, gh):
    z, lse, logp, p = softmax64(x, T)
    inside = (ids >= 0) & (ids < x.shape[1])
    gl = torch.where(inside, gl.double(), 0.0)
    h = entropy64(logp, p)
    ln = torch.where(p > 0, logp, 0.0)
    share = torch.zeros_like(p)
    share.scatter_add_(1, torch.where(inside, ids, 0).long(), gl)
    size = torch.zeros_like(p).scatter_add_(1, torch.where(inside, ids, 0).long(), gl.abs())
    inner = torch.where(p > 0, ln + h[:, None], 0.0)
    grad = (share - p * (gl.sum(1, keepdim=True) + gh.double()[:, None] * inner)) / T
    # what the roundings act on: the probability's terms (its relative error grows with |ln p| and |lse|), then the shares
    lsz = torch.where(torch.isfinite(lse), lse.abs(), 0.0)[:, None]
    rel = sum_error(x.shape[1]) * 2 + E * (8 * ln.abs() + 8 * lsz)
    terms = p * (gl.abs().sum(1, keepdim=True) + gh.double().abs()[:, None] * (ln.abs() + h[:, None].abs() + 1))
    return grad, (rel * terms + 8 * E * (size + terms)) / T


def gradient_tolerance(grad, tol, dtype):
    rel, floor = HALF[dtype]
    return tol * (1 + rel) + rel * grad.abs() + floor + 1e-37


@pytest.mark.parametrize("n", [1, 3, 8, 65, 700, 4096, 4097, 33000, 131079])
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_backward(O, n, dtype):
    g = gen(n + 1)
    m, T = 4, [1.0, 0.7, 2.0][n % 3]
    x = (3 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    x[3] = float("-inf")
    ids = torch.randint(0, n, (m, 6), generator=g)
    ids[0, 1], ids[1, 2], ids[2, 5] = -1, n, ids[2, 0]  # padding twice, and an id given twice
    gl, gh = torch.randn((m, 6), generator=g), torch.randn(m, generator=g)
    for pad in (0, 3):
        xd = padded(x, pad)
        r = O.log_probs(xd, ids.cuda(), temperature=T)
        got = O.log_probs_backward(gl.cuda(), gh.cuda(), xd, ids.cuda(), r.lse, r.entropy, temperature=T)
        assert got.dtype == x.dtype
        want, tol = grad64(x, ids, T, gl, gh)
        close(got, want, gradient_tolerance(want, tol, dtype), "gradient")
        for a, b in ((gl, None), (None, gh)):
            got = O.log_probs_backward(None if a is None else a.cuda(), None if b is None else b.cuda(), xd, ids.cuda(), r.lse,
                                       r.entropy, temperature=T)
            want, tol = grad64(x, ids, T, gl if a is not None else 0 * gl, gh if b is not None else 0 * gh)
            close(got, want, gradient_tolerance(want, tol, dtype), "one of the two gradients")


def test_gradients_of_rows_far_from_zero(O):
    """Logits of one large offset, and rows of the lowest value: p does not come from a rounded log-sum-exp."""
    g = gen(2)
    x = torch.randn((3, 1000), generator=g)
    x[0] = (x[0] * 64).round() / 64 + 4096
    x[1] = torch.finfo(torch.float32).min
    x[2] -= 30000
    x[2] = (x[2] * 64).round() / 64
    ids = torch.tensor([[5], [7], [9]])
    gl, gh = torch.ones((3, 1)), torch.zeros(3)
    r = O.log_probs(x.cuda(), ids.cuda())
    got = O.log_probs_backward(gl.cuda(), None, x.cuda(), ids.cuda(), r.lse, r.entropy)
    _, _, logp, p = softmax64(x - x.max(1, keepdim=True).values, 1.0)
    want = -p
    want[torch.arange(3), ids[:, 0]] += 1
    close(got, want, sum_error(1000) * 2 * p + 16 * E, "gradient far from zero")
    t = torch.zeros((3, 1))
    loss, grad = O.distill_step(torch.ones(3).cuda(), x.cuda(), ids.cuda(), t.cuda())
    close(grad, -want, sum_error(1000) * 2 * p + 16 * E, "distillation far from zero")
    close(loss, -logp.gather(1, ids)[:, 0], sum_error(1000) + 64 * E, "loss far from zero")


@pytest.mark.parametrize("m,n", [(2, 5), (2, 1000), (2, 70_001), (2100, 300)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [0.5, 0.75])
def test_gradients_of_the_lowest_value_below_temperature_one(O, m, n, dtype, T):
    """A row masked by the type's lowest value is uniform, its log-sum-exp past fp32 or not; a row of -inf has p = 0."""
    x = torch.full((m, n), torch.finfo(TYPES[dtype]).min).to(TYPES[dtype])
    x[1::2] = float("-inf")
    ids = torch.full((m, 1), n - 1)
    one = torch.ones((m, 1))
    want = torch.full((m, n), -1 / n, dtype=torch.float64)
    want[1::2] = 0
    want[:, n - 1] += 1
    want /= T
    # p = 2^(0 - log2 n) by fp32 exponent and power; then a rounding of each term and of their sum
    tol = gradient_tolerance(want, (2 * sum_error(n) + 32 * E * (1 + math.log2(n))) / n / T + 8 * E * want.abs(), dtype)
    r = O.log_probs(x.cuda(), ids.cuda(), temperature=T)
    close(r.log_probs[::2], torch.full(((m + 1) // 2, 1), -math.log(n), dtype=torch.float64), sum_error(n) + 32 * E, "log_probs")
    got = O.log_probs_backward(one.cuda(), None, x.cuda(), ids.cuda(), r.lse, r.entropy, temperature=T)
    close(got, want, tol, "gradient")
    loss, lse = O.distill(x.cuda(), ids.cuda(), one.cuda(), temperature=T)
    got = O.distill_backward(one[:, 0].cuda(), x.cuda(), ids.cuda(), one.cuda(), lse, temperature=T)
    close(got, -want, tol, "distillation's gradient")
    step, got = O.distill_step(one[:, 0].cuda(), x.cuda(), ids.cuda(), one.cuda(), temperature=T)
    close(got, -want, tol, "distillation step's gradient")
    assert torch.equal(step, loss)


@pytest.mark.parametrize("T", [1.0, 1.5])
def test_gradients_against_differences(O, T):
    """Central differences of the kernels' own values: of step s they are off by s^2 / T^3 of the third derivative (under 1)
    and by the values' roundings over s, 64 e |value| / s."""
    g = gen(9)
    m, n, s = 1, 12, 2.0**-6
    x = torch.randn((m, n), generator=g)
    ids = torch.tensor([[3, 7, 3]])
    gl, gh = torch.tensor([[0.7, -0.4, 0.2]]), torch.tensor([0.9])
    teacher, tid = torch.tensor([[1.0, 0.3, -0.5]]), torch.tensor([[2, 11, 5]])
    each = x.repeat(2 * n, 1)
    for v in range(n):
        each[2 * v, v] += s
        each[2 * v + 1, v] -= s
    r = O.log_probs(each.cuda(), ids.repeat(2 * n, 1).cuda(), temperature=T)
    value = (r.log_probs.cpu().double() * gl).sum(1) + r.entropy.cpu().double() * gh
    slope = (value[0::2] - value[1::2]) / (2 * s)
    r = O.log_probs(x.cuda(), ids.cuda(), temperature=T)
    got = O.log_probs_backward(gl.cuda(), gh.cuda(), x.cuda(), ids.cuda(), r.lse, r.entropy, temperature=T)
    bound = 3 * s * s + 64 * E * 5 / s
    close(got[0], slope, bound, "differences of log probabilities and entropy")
    loss, _ = O.distill(each.cuda(), tid.repeat(2 * n, 1).cuda(), teacher.repeat(2 * n, 1).cuda(), temperature=T)
    slope = (loss.cpu().double()[0::2] - loss.cpu().double()[1::2]) / (2 * s)
    _, grad = O.distill_step(torch.ones(1).cuda(), x.cuda(), tid.cuda(), teacher.cuda(), temperature=T)
    close(grad[0], slope, bound, "differences of the distillation loss")


# ----------------------------------------------------------------------------------------------------------- distillation


def distill64(x, ids, teacher, T, g):
    z, lse, logp, p = softmax64(x, T)
    n = x.shape[1]
    inside = (ids >= 0) & (ids < n)
    t = torch.where(inside, teacher.double() / T, float("-inf"))
    some = t.max(1).values > float("-inf") if ids.shape[1] else torch.zeros(len(x), dtype=torch.bool)
    top = torch.where(some[:, None], t.max(1, keepdim=True).values, 0.0) if ids.shape[1] else 0.0
    w = torch.exp(t - top)
    total = torch.where(some, w.sum(1), 1.0)
    q, lq = w / total[:, None], t - top - torch.log(total)[:, None]
    at = torch.where(inside, ids, 0).long()
    lp = logp.gather(1, at)
    used = q > 0
    loss = torch.where(used, q * (torch.where(used, lq, 0.0) - torch.where(used, lp, 0.0)), 0.0).sum(1)
    g = torch.where(some, g.double(), 0.0)[:, None] / T
    grad = p.clone().scatter_add_(1, at, -q) * g
    lsz = torch.where(torch.isfinite(lse), lse.abs(), 0.0)[:, None]
    ln = torch.where(p > 0, logp, 0.0).abs()
    rel = sum_error(n) * 2 + E * (8 * ln + 8 * lsz)
    qe = E * (ids.shape[1] / 64 + 32 + 8 * torch.where(used, t.abs() + lq.abs(), 0.0))  # of q: its exponent and its sum
    spread = torch.zeros_like(p).scatter_add_(1, at, q * (qe + 8 * E))
    gtol = ((rel + 8 * E) * p + spread) * g.abs()
    fin = torch.where(used & torch.isfinite(lp), lp.abs() + lq.abs(), 0.0)
    ltol = sum_error(n) + (q * (E * (16 * fin + 8 * lsz) + qe * (1 + fin))).sum(1) + E * 8 * loss.abs().nan_to_num(posinf=0)
    return loss, torch.where(some[:, None], grad, 0.0), ltol, gtol


def check_distill(O, x, ids, teacher, T, g, dtype, pad=0):
    xd, idd, td, gd = padded(x, pad), ids.cuda(), teacher.cuda(), g.cuda()
    want_loss, want, ltol, gtol = distill64(x, ids, teacher, T, g)
    tol = gradient_tolerance(want, gtol, dtype)
    loss, grad = O.distill_step(gd, xd, idd, td, temperature=T)
    assert grad.dtype == x.dtype and loss.dtype == torch.float32
    close(loss, want_loss, ltol, "loss of a step")
    close(grad, want, tol, "gradient of a step")
    loss, lse = O.distill(xd, idd, td, temperature=T)
    close(loss, want_loss, ltol, "loss")
    close(O.distill_backward(gd, xd, idd, td, lse, temperature=T), want, tol, "gradient")


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 64, 513, 2048, 8193, 32000, 65536, 65537, 131072, 131080, 150001])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill(O, n, dtype):
    g = gen(n + 2)
    m, T = 3, [1.0, 0.5, 2.0][n % 3]
    x = (3 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    k = min(n, 10)
    ids = torch.stack([torch.randperm(n, generator=g)[:k] for _ in range(m)])
    teacher = 2 * torch.randn((m, k), generator=g)
    for pad in (0, 5):
        check_distill(O, x, ids, teacher, T, 0.5 + torch.rand(m, generator=g), dtype, pad)


@pytest.mark.parametrize("m,k", [(1, 1), (5, 63), (3, 64), (4, 65), (2, 256), (2, 512), (700, 10)])
def test_distill_lists(O, m, k):
    """Lists of every length, with padding, repeated ids and teachers that give nothing."""
    g = gen(k)
    n = 1500
    x = (2 * torch.randn((m, n), generator=g)).bfloat16()
    ids = torch.randint(0, n, (m, k), generator=g)
    teacher = (3 * torch.randn((m, k), generator=g)).half()
    ids[torch.rand((m, k), generator=g) < 0.2] = -1
    ids[0, k // 2 :] = n + 3
    ids[m - 1] = -1  # nothing listed
    if m > 2:
        teacher[1] = float("-inf")  # nothing given
        teacher[2, : k // 2] = float("-inf")
        ids[2, k - 1] = ids[2, 0] = 17
    check_distill(O, x, ids, teacher.float(), 1.0, torch.rand(m, generator=g), "bfloat16")
    loss, grad = O.distill_step(torch.ones(m).cuda(), x.cuda(), ids.int().cuda(), teacher.cuda())
    if m != 3:  # whose last row lists 17
        assert loss[m - 1] == 0 and (grad[m - 1] == 0).all()
    if m > 2:
        assert loss[1] == 0 and (grad[1] == 0).all()


@pytest.mark.parametrize("m,n,k,dtype", [
    (9000, 500, 5, "float32"), (2100, 3000, 20, "bfloat16"), (2100, 1000, 200, "bfloat16"), (1100, 9000, 10, "float16"),
    (200, 9000, 70, "float32"), (300, 40_001, 10, "bfloat16"), (520, 66_003, 70, "bfloat16"), (513, 33_000, 3, "float32"),
])
def test_distill_of_every_grouping(O, m, n, k, dtype):
    """A wavefront to 1,024 threads a row, and several rows one after another in a workgroup; some rows list nothing."""
    g = gen(m + n)
    x = (2 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    ids = torch.randint(-1, n, (m, k), generator=g)
    ids[:: 7] = -1
    teacher = 2 * torch.randn((m, k), generator=g)
    check_distill(O, x, ids, teacher, 1.0, (0.5 + torch.rand(m, generator=g)) * (1 if dtype == "float32" else 1024), dtype, 3)


@pytest.mark.parametrize("m,n,k", [(2100, 1000, 128), (2051, 523, 65), (2048, 4096, 100), (2100, 70, 64), (300, 2000, 512)])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_of_dense_lists(O, m, n, k, dtype):
    """Many listed ids in every piece of a row, most of them more than once."""
    g = gen(m + n + k)
    x = (2 * torch.randn((m, n), generator=g)).to(TYPES[dtype])
    ids = torch.randint(0, min(n, 2 * k), (m, k), generator=g) * torch.tensor(max(1, n // (2 * k)))
    ids[::5] = torch.randint(n - min(n, 40), n, ids[::5].shape, generator=g)
    ids[::9, ::3] = -1
    teacher = 2 * torch.randn((m, k), generator=g)
    check_distill(O, x, ids, teacher, 1.0, (0.5 + torch.rand(m, generator=g)) * (1 if dtype == "float32" else 1024), dtype, 3)


@pytest.mark.parametrize("m,n,k", [(3, 30, 4), (3, 5000, 512), (3, 140_000, 70), (2100, 700, 100)])
@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
def test_teachers_of_extreme_values(O, m, n, k, T):
    """A teacher's lowest and highest values are values: a list of the lowest is uniform, whatever the temperature."""
    g = gen(n + k)
    low = torch.finfo(torch.float32).min
    x = torch.randn((m, n), generator=g)
    ids = torch.randint(0, n, (m, k), generator=g)
    teacher = 2 * torch.randn((m, k), generator=g)
    teacher[0] = low
    teacher[1, 1:] = low
    teacher[2, : k // 2] = -low
    w = torch.ones(m)
    # the same q from logits of ordinary size, by which the tolerances go
    like = teacher.clamp_min(-1e6)
    like[0] = 0
    like[2] = torch.where(teacher[2] == -low, 0.0, -1e6)
    want_loss, want, ltol, gtol = distill64(x, ids, like, T, w)
    loss, grad = O.distill_step(w.cuda(), x.cuda(), ids.cuda(), teacher.cuda(), temperature=T)
    close(loss, want_loss, ltol, "loss of a step")
    close(grad, want, gradient_tolerance(want, gtol, "float32"), "gradient of a step")
    loss, lse = O.distill(x.cuda(), ids.cuda(), teacher.cuda(), temperature=T)
    close(loss, want_loss, ltol, "loss")
    got = O.distill_backward(w.cuda(), x.cuda(), ids.cuda(), teacher.cuda(), lse, temperature=T)
    close(got, want, gradient_tolerance(want, gtol, "float32"), "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [30, 5000, 140000])
def test_distill_masks_infinities_and_nan(O, dtype, n):
    g = gen(n + 5)
    low = torch.finfo(TYPES[dtype]).min
    x = torch.randn((7, n), generator=g)
    x[0, torch.rand(n, generator=g) < 0.5] = float("-inf")
    x[0, :3] = torch.tensor([0.5, 1.0, -1.0])
    x[1] = float("-inf")
    x[2] = low
    x[3, 3:] = low
    x[4, 1] = float("-inf")  # a listed id without probability: an infinite loss
    x[5, n // 2] = float("nan")
    x[6, 0] = float("nan")
    x = x.to(TYPES[dtype])
    ids = torch.tensor([[0, 1, 2]] * 7)
    ids[6] = -1
    teacher = torch.tensor([[1.0, 0.0, -1.0]] * 7)
    w = torch.ones(7)
    loss, grad = O.distill_step(w.cuda(), x.cuda(), ids.cuda(), teacher.cuda())
    keep = torch.tensor([0, 1, 2, 3, 4])
    want_loss, want, ltol, gtol = distill64(x[keep], ids[keep], teacher[keep], 1.0, w[keep])
    # a log-sum-exp of the lowest value has no digits left for ln n: such rows are held to log p instead
    close(grad[keep.cuda()][[0, 3, 4]], want[[0, 3, 4]], gradient_tolerance(want, gtol, dtype)[[0, 3, 4]], "gradient")
    close(loss[keep.cuda()][[0, 1, 3, 4]], want_loss[[0, 1, 3, 4]], ltol[[0, 1, 3, 4]], "loss")
    q = torch.softmax(teacher[0].double(), 0)
    assert abs(loss[2].item() - (math.log(n) + (q * q.log()).sum().item())) < 1e-4
    flat = torch.full((n,), 1 / n, dtype=torch.float64)
    flat[:3] -= q
    close(grad[2], flat, HALF[dtype][0] * flat.abs() + HALF[dtype][1] + 1e-6 * flat.abs(), "uniform row")
    assert loss[1] == float("inf") and loss[4] == float("inf")
    near = torch.zeros(n, dtype=torch.float64)
    near[:3] = -q
    close(grad[1], near, (HALF[dtype][0] + 64 * E) * near.abs(), "row of nothing")
    assert torch.isnan(loss[5]) and torch.isnan(grad[5]).all()
    assert loss[6] == 0 and (grad[6] == 0).all()  # nothing to learn, whatever the row holds


# --------------------------------------------------------------------------------------- callers: memory, streams, graphs


def test_operands_of_other_kinds(O):
    """numpy and CPU tensors are copied and answered in kind; other types and orders are converted."""
    g = gen(1)
    x, ids = torch.randn((4, 300), generator=g), torch.randint(0, 300, (4, 2), generator=g)
    r = O.log_probs(x.cuda(), ids.cuda(), top=3)
    for a, b in ((x.numpy(), ids.numpy()), (x, ids), (x.double(), ids.int()), (x.t().contiguous().t(), ids)):
        s = O.log_probs(a, b, top=3)
        assert isinstance(s.lse, type(a)) and np.array_equal(np.asarray(s.top_ids), r.top_ids.cpu().numpy())
        assert np.array_equal(np.asarray(s.log_probs), r.log_probs.cpu().numpy())
    s = O.log_probs(x.cuda().t().contiguous().t(), ids.cuda(), top=3)
    assert torch.equal(s.log_probs, r.log_probs)
    w = torch.rand(4, generator=g)
    t = torch.randn((4, 2), generator=g)
    loss, grad = O.distill_step(w.numpy(), x.numpy(), ids.numpy(), t.numpy())
    l2, g2 = O.distill_step(w.cuda(), x.cuda(), ids.cuda(), t.cuda())
    assert np.array_equal(loss, l2.cpu().numpy()) and np.array_equal(grad, g2.cpu().numpy())
    l3, g3 = O.distill_step(torch.ones(1).cuda().expand(4), x[:1].cuda().expand(4, 300), ids.cuda(), t.cuda())
    l4, g4 = O.distill_step(torch.ones(4).cuda(), x[:1].repeat(4, 1).cuda(), ids.cuda(), t.cuda())
    assert torch.equal(l3, l4) and torch.equal(g3, g4)  # broadcast inputs
    codes, scales = O.quantize_rows(x.numpy())
    assert isinstance(codes, np.ndarray) and codes.dtype == np.int8 and scales.dtype == np.float32
    y = O.int8_scores(x.numpy(), codes, scales)
    assert np.array_equal(y, O.int8_scores(x.cuda(), torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()).cpu().numpy())


class Exported:
    """An array of another framework, in the memory of a torch tensor."""

    def __init__(self, t):
        self.t = t

    def __dlpack__(self, **kw):
        return self.t.__dlpack__()

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()


def test_views_and_other_frameworks_on_either_side(O):
    """numpy's backward, read-only and broadcast views; arrays of other frameworks are answered where they lie."""
    g = gen(4)
    x, ids = torch.randn((4, 300), generator=g), torch.randint(0, 300, (4, 2), generator=g)
    want = O.log_probs(x.flip(0).flip(1).cuda(), ids.flip(1).cuda(), top=3)
    got = O.log_probs(x.numpy()[::-1, ::-1], ids.numpy()[:, ::-1], top=3)
    assert all(np.array_equal(a, b.cpu().numpy()) for a, b in zip(got, want))
    row = np.broadcast_to(x.numpy()[0], (4, 300))
    assert np.array_equal(O.log_probs(row, ids.numpy()).lse, O.log_probs(x[:1].repeat(4, 1).cuda(), ids.cuda()).lse.cpu().numpy())
    want = O.log_probs(x.cuda(), ids.cuda(), top=3)
    for side in ("cpu", "cuda"):
        xs = x.to(side)
        torch.cuda.synchronize()
        got = O.log_probs(Exported(xs), ids, top=3)
        torch.cuda.synchronize()
        assert all(a.device.type == side and torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


def test_scalars_of_any_kind(O):
    x, ids = torch.randn((3, 50)).cuda(), torch.zeros((3, 1), dtype=torch.int64).cuda()
    want = O.log_probs(x, ids, top=2, temperature=2.0)
    for two in (2, np.float32(2), np.int64(2), torch.tensor(2.0)):
        r = O.log_probs(x, ids, top=np.int32(2), temperature=two)
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_no_rows(O):
    x, ids = torch.zeros((0, 50)).cuda(), torch.zeros((0, 3), dtype=torch.int64).cuda()
    r = O.log_probs(x, ids, top=4)
    assert r.log_probs.shape == (0, 3) and r.top_ids.shape == (0, 4)
    loss, grad = O.distill_step(torch.zeros(0).cuda(), x, ids, torch.zeros((0, 3)).cuda())
    assert loss.shape == (0,) and grad.shape == (0, 50)
    codes, scales = O.quantize_rows(x)
    assert codes.shape == (0, 50) and scales.shape == (0,)
    some = torch.zeros((2, 50)).cuda()
    assert O.int8_scores(some, codes, scales).shape == (2, 0)
    assert O.int8_scores(x, *O.quantize_rows(some)).shape == (0, 2)
    r = O.log_probs(some, torch.zeros((2, 0), dtype=torch.int64).cuda(), top=1)  # no ids: entropy and alternatives alone
    assert r.log_probs.shape == (2, 0) and r.top_ids[:, 0].tolist() == [0, 0]


def every_operator(O, x, ids, w, teacher, rows, scales):
    r = O.log_probs(x, ids, top=5)
    out = list(r) + [O.log_probs_backward(w[:, None].expand(ids.shape), w, x, ids, r.lse, r.entropy)]
    loss, lse = O.distill(x, ids, teacher)
    out += [loss, O.distill_backward(w, x, ids, teacher, lse), *O.distill_step(w, x, ids, teacher)]
    return out + [O.int8_scores(x, rows, scales)]


@pytest.mark.parametrize("m,n", [(2, 40000), (40, 3000)])
def test_results_repeat_on_any_stream(O, m, n):
    g = gen(m)
    args = [(2 * torch.randn((m, n), generator=g)).bfloat16().cuda(), torch.randint(0, n, (m, 6), generator=g).cuda(),
            torch.rand(m, generator=g).cuda(), torch.randn((m, 6), generator=g).cuda(),
            *O.quantize_rows(torch.randn((70, n), generator=g).cuda())]
    torch.cuda.synchronize()
    want = every_operator(O, *args)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        filler = torch.randn((2000, 2000), device="cuda")
        for _ in range(5):
            filler = filler @ filler / 100  # the operands change behind this work, on this stream
        x2 = args[0] * 1
        got = every_operator(O, x2, *args[1:])
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("m,n", [(1, 40000), (40, 3000)])
def test_captured_calls_replay(O, m, n):
    g = gen(m + 1)
    x = (2 * torch.randn((m, n), generator=g)).bfloat16().cuda()
    ids, w = torch.randint(0, n, (m, 6), generator=g).cuda(), torch.rand(m, generator=g).cuda()
    teacher = torch.randn((m, 6), generator=g).cuda()
    rows, scales = O.quantize_rows(torch.randn((70, n), generator=g).cuda())
    every_operator(O, x, ids, w, teacher, rows, scales)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = every_operator(O, x, ids, w, teacher, rows, scales)
    for seed in range(4):
        x.copy_((2 * torch.randn((m, n), generator=gen(seed))).bfloat16())
        ids.copy_(torch.randint(0, n, (m, 6), generator=gen(seed + 50)))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        want = every_operator(O, x, ids, w, teacher, rows, scales)
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets(O):
    """Matrices of more than 2^32 elements: the last rows are as right as the first."""
    m, n = 40, 120_000_000  # 4.8e9 float16 logits
    x = torch.zeros((m, n), dtype=torch.float16, device="cuda")
    ids = torch.full((m, 1), n - 1, device="cuda")
    x[:, -1] = 3.0
    x[-1, n // 2] = 5.0
    r = O.log_probs(x, ids, top=2)
    lse = math.log(n - 1 + math.exp(3))
    assert abs(r.lse[m - 2].item() - lse) < (n / 256 + 64) * E * 4
    assert r.top_ids[0].tolist() == [n - 1, 0] and r.top_ids[m - 1].tolist() == [n // 2, n - 1]
    loss, grad = O.distill_step(torch.full((m,), 4096.0, device="cuda"), x, ids, torch.zeros((m, 1), device="cuda"))
    assert abs(loss[0].item() - (lse - 3)) < 1e-3
    assert grad[0, n - 1].item() < -4000 and grad[m - 1, n - 1].item() < -4000 and grad[m - 2, 0].item() >= 0
    del x, grad
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m,k", [(1, 2048), (20, 2048), (300, 2048), (2000, 2048), (20, 2047)])
def test_scores_beyond_32_bit_offsets(O, m, k):
    """Rows of more than 2^32 bytes, and (of 2000 queries) more than 2^32 scores."""
    n = 2_200_000
    rows = torch.zeros((n, k), dtype=torch.int8, device="cuda")
    rows[-1], rows[n // 2] = 1, 2
    rs = torch.ones(n, device="cuda")
    q = torch.ones((m, k), dtype=torch.int8, device="cuda")
    q[-1] = 3
    s = O.int8_scores(q, rows, rs, query_scales=torch.full((m,), 2.0**-8, device="cuda"), dtype="float16")
    want = torch.zeros(n, dtype=torch.float16, device="cuda")
    want[-1], want[n // 2] = k / 256, 2 * k / 256
    assert torch.equal(s[-1], 3 * want)
    for i in (0, m // 2) if m > 1 else ():
        assert torch.equal(s[i], want)
    del rows, s
    torch.cuda.empty_cache()


def test_quantized_rows_and_gradients_beyond_32_bit_offsets(O):
    x = torch.zeros((2_200_000, 2048), dtype=torch.float16, device="cuda")
    x[-1, 5], x[-1, 6], x[1_100_000] = 127, -3, 2
    codes, scales = O.quantize_rows(x)
    assert codes[-1, 5] == 127 and codes[-1, 6] == -3 and (codes[1_100_000] == 127).all() and scales[-1] == 1
    assert scales[-2] == 0 and (codes[-2] == 0).all()
    del x, codes
    m, n = 36_000, 120_000  # a workgroup holds a row
    x = torch.zeros((m, n), dtype=torch.float16, device="cuda")
    ids = torch.full((m, 1), n - 1, device="cuda")
    loss, grad = O.distill_step(torch.full((m,), 4096.0, device="cuda"), x, ids, torch.zeros((m, 1), device="cuda"))
    want = torch.full((n,), 4096 / n, device="cuda")
    want[-1] -= 4096
    for i in (0, m // 2, m - 1):
        assert abs(loss[i].item() - math.log(n)) < 1e-3
        assert torch.allclose(grad[i].float(), want, rtol=2e-3)
    del x, grad
    torch.cuda.empty_cache()


def test_the_example_learns(O):
    """examples/distill_queries.py: search, scores, distillation and log probabilities together."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "distill_queries.py")
    spec = importlib.util.spec_from_file_location("distill_queries", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, before, after = example.main(steps=30, n=5000, quiet=True)
    assert last < 0.7 * first and after > before


# --------------------------------------------------------------------------------------------------------------- refusals


def test_refusals(O):
    x, ids = torch.randn((3, 50)).cuda(), torch.zeros((3, 2), dtype=torch.int64).cuda()
    t, w = torch.zeros((3, 2)).cuda(), torch.ones(3).cuda()
    r = O.log_probs(x, ids)
    codes, scales = O.quantize_rows(x)
    bad = [
        (ValueError, lambda: O.log_probs(x, ids, top=65)),
        (ValueError, lambda: O.log_probs(x, ids, top=-1)),
        (RuntimeError, lambda: O.log_probs(x, ids, temperature=0.0)),
        (RuntimeError, lambda: O.log_probs(x, ids, temperature=-1.0)),
        (RuntimeError, lambda: O.log_probs(x, ids, temperature=float("nan"))),
        (RuntimeError, lambda: O.log_probs(x, ids, temperature=float("inf"))),
        (ValueError, lambda: O.log_probs(x, ids[:2])),
        (TypeError, lambda: O.log_probs(x, t)),
        (ValueError, lambda: O.log_probs(x[None], ids)),
        (RuntimeError, lambda: O.log_probs(x, ids.repeat(1, 300))),
        (RuntimeError, lambda: O.log_probs(x[:, :0], ids)),
        (ValueError, lambda: O.log_probs_backward(w, None, x, ids, r.lse, r.entropy)),
        (ValueError, lambda: O.log_probs_backward(t, w[:2], x, ids, r.lse, r.entropy)),
        (ValueError, lambda: O.log_probs_backward(t, w, x, ids, r.lse[:1], r.entropy)),
        (ValueError, lambda: O.distill(x, ids, t[:, :1])),
        (ValueError, lambda: O.distill_step(w[:2], x, ids, t)),
        (ValueError, lambda: O.distill_backward(w, x, ids, t, w[:1])),
        (ValueError, lambda: O.int8_scores(x, codes[:, :49], scales)),
        (ValueError, lambda: O.int8_scores(x, codes, scales[:2])),
        (ValueError, lambda: O.int8_scores(x, codes, scales, bias=scales[:2])),
        (TypeError, lambda: O.int8_scores(x, x, scales)),
        (TypeError, lambda: O.int8_scores(x, codes, scales, query_scales=w)),
        (ValueError, lambda: O.int8_scores(codes, codes, scales, query_scales=w[:2])),
        (ValueError, lambda: O.int8_scores(x, codes, scales, dtype="int8")),
        (RuntimeError, lambda: O.quantize_rows(torch.zeros((1, 131072)).cuda())),
        (RuntimeError, lambda: O.quantize_rows(x[:, :0])),
    ]
    for kind, call in bad:
        with pytest.raises(kind, match="octex"):
            call()
    assert torch.isfinite(O.log_probs(x, ids).lse).all()  # a refusal leaves nothing behind
