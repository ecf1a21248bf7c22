"""Rows of a table by ids, and the table's gradient, against plain 64-bit forms.

Bounds, derived before the first run: a row's value rounds its scale once (int8 rows their product of scales once more) and the
product once, 3 E of it; a sum of c gradients rounds at most c times, by E of the sum of sizes so far each, then its product with
the scale and, added to what the table held, their sum: (c + 3) E of the sum of sizes and E of the result.

Which tokens are sorted: none of up to 1024, and of up to 4096 only those of wide rows (m^2 ceil(d / 512) beyond 2^25), so that tests
of fewer tokens look them through.  The sort by one workgroup (2, 4 or 8 tokens a thread; one to four digits) and by many is
reached by test_gradient_on_both_sides_of_the_sort and what follows it."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from operators64 import E, TYPES, captured, close, gen, package, padded, randn, rounded  # noqa: E402

WIDTHS = [1, 3, 7, 8, 9, 12, 31, 63, 64, 65, 96, 100, 128, 129, 200, 256, 257, 500, 512, 513, 960, 1001, 4096, 4100]


@pytest.fixture(scope="module")
def O():
    return package()


def table_of(g, n, d, kind):
    """A table and its row_scales."""
    if kind == "int8":
        return torch.randint(-128, 128, (n, d), generator=g, device="cuda", dtype=torch.int8), torch.rand(n, generator=g, device="cuda")
    return randn(g, n, d).to(TYPES[kind]), None


def rows64(table, scales, ids, scale):
    n = table.shape[0]
    inside = (ids >= 0) & (ids < n)
    at = torch.where(inside, ids, 0).long()
    rows = table.double()[at] * float(np.float32(scale))
    if scales is not None:
        rows = rows * scales.double()[at][..., None]
    return torch.where(inside[..., None], rows, 0.0)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("kind", ["int8", *TYPES])
def test_embed(O, d, kind):
    g = gen(d)
    table, scales = table_of(g, 77, d, kind)
    for m, out, pad in ((1, None, 0), (5, "bfloat16", 3), (130, "float32", 0), (1000, "float16", 1)):
        ids = torch.randint(-3, 80, (m,), generator=g, device="cuda")
        ids[0] = 76
        scale = 0.37
        got = O.embed(padded(table, pad) if kind != "int8" or pad == 0 else torch.cat([table, table], 1)[:, :d], ids,
                      row_scales=scales, scale=scale, dtype=out)
        dtype = out or ("float32" if kind == "int8" else kind)
        assert got.dtype == TYPES[dtype]
        want = rows64(table, scales, ids, scale)
        close(got, want, rounded(3 * E * want.abs(), want, dtype), "rows")


@pytest.mark.parametrize("kind", TYPES)
def test_rows_as_they_are(O, kind):
    """Scale 1 and the table's own type: indexing, bit for bit, of any value."""
    g = gen(1)
    table = randn(g, 50, 40).to(TYPES[kind])
    table[3, :6] = torch.tensor([float("inf"), float("-inf"), float("nan"), 0.0, -0.0, torch.finfo(TYPES[kind]).min])
    table[3, 6:9] = torch.tensor([torch.finfo(TYPES[kind]).max, torch.finfo(TYPES[kind]).tiny, torch.finfo(TYPES[kind]).tiny / 4])
    ids = torch.arange(50, device="cuda").flip(0)
    got = O.embed(table, ids)
    keep = ~torch.isnan(table[ids])
    size = {2: torch.int16, 4: torch.int32}[table.element_size()]
    assert torch.equal(torch.isnan(got), ~keep)
    assert torch.equal(got.view(size)[keep], table[ids].view(size)[keep])


def test_ids_of_any_shape(O):
    g = gen(2)
    table = randn(g, 30, 20)
    ids = torch.randint(0, 30, (4, 5, 3), generator=g, device="cuda")
    want = table[ids]
    assert torch.equal(O.embed(table, ids), want) and torch.equal(O.embed(table, ids.int()), want)
    assert torch.equal(O.embed(table, ids.transpose(0, 2)), want.transpose(0, 2))
    assert torch.equal(O.embed(table, ids[:, 0, ::2]), want[:, 0, ::2]) and torch.equal(O.embed(table, ids[0, 0, 0]), want[0, 0, 0])
    assert torch.equal(O.embed(table, ids[0, 0, 0].expand(7)), want[0, 0, 0].expand(7, 20))
    assert O.embed(table, ids[:0]).shape == (0, 5, 3, 20) and O.embed(table[:, :0], ids).shape == (4, 5, 3, 0)
    assert torch.equal(O.embed(table[:0], ids), torch.zeros_like(want))
    assert torch.equal(O.embed(table, [3, -1, 29]), torch.stack([table[3], table[0] * 0, table[29]]))
    grad = randn(g, 4, 5, 3, 20)
    want = O.embed_backward(grad.reshape(60, 20), ids.reshape(-1), 30)
    assert torch.equal(O.embed_backward(grad, ids, 30), want)
    assert torch.equal(O.embed_backward(grad[0, 0, 0], ids[0, 0, 0], 30)[ids[0, 0, 0]], grad[0, 0, 0])


def test_numpy(O):
    g = np.random.default_rng(0)
    table, ids = g.standard_normal((40, 24), dtype=np.float32), g.integers(-1, 40, (6, 3))
    got = O.embed(table, ids, scale=2.0)
    want = 2 * table[ids] * (ids >= 0)[..., None]
    assert isinstance(got, np.ndarray) and np.array_equal(got, want)
    grad = O.embed_backward(got, ids, 40)
    assert isinstance(grad, np.ndarray) and grad.shape == (40, 24)
    with pytest.raises(TypeError, match="bfloat16"):
        O.embed(table, ids, dtype="bfloat16")


def gradient64(grad, ids, n, scale, old=None):
    """The gradient and its bound but for the rounding of the result."""
    inside = (ids >= 0) & (ids < n)
    at = torch.where(inside, ids, n).long()
    d = grad.shape[1]
    s = float(np.float32(scale))
    total = torch.zeros((n + 1, d), dtype=torch.float64, device="cuda").index_put_((at,), grad.double() * s, accumulate=True)[:n]
    size = torch.zeros((n + 1, d), dtype=torch.float64, device="cuda").index_put_((at,), grad.double().abs() * abs(s),
                                                                                 accumulate=True)[:n]
    count = torch.bincount(at, minlength=n + 1)[:n, None]
    tol = (count + 3) * E * size
    if old is not None:
        total = total + torch.where(count > 0, old.double(), old.double())
        tol = tol + torch.where(count > 0, E * total.abs(), 0.0)
    return total, tol, count[:, 0] > 0


def check_gradient(O, grad, ids, n, scale=0.37, dtype=None, given=None):
    name = dtype or str(grad.dtype).replace("torch.", "")
    want, tol, used = gradient64(grad, ids, n, scale)
    got = O.embed_backward(grad if given is None else given, ids, n, scale=scale, dtype=dtype)
    assert got.dtype == TYPES[name]
    close(got, want, rounded(tol, want, name), "gradient")
    assert (got[~used] == 0).all()
    g = gen(9)
    old = randn(g, n, grad.shape[1]).to(TYPES[name])
    sums = padded(old, 3)
    want, tol, used = gradient64(grad, ids, n, scale, old)
    assert O.embed_backward(grad if given is None else given, ids, scale=scale, add_to=sums) is sums
    close(sums, want, rounded(tol, want, name), "added gradient")
    size = {2: torch.int16, 4: torch.int32}[old.element_size()]
    assert torch.equal(sums[~used].contiguous().view(size), old[~used].view(size)), "rows without an id"
    if sums.stride(0) > sums.shape[1] and n > 1:  # beside the matrix
        wide = sums.as_strided((n - 1, 3), (sums.stride(0), 1), sums.storage_offset() + sums.shape[1])
        assert (wide == 7).all()


def ids_of(g, m, n, kind):
    if kind == "one":
        return torch.full((m,), n // 2, device="cuda")
    if kind == "few":  # long runs that begin and end anywhere
        return torch.randint(0, 5, (m,), generator=g, device="cuda") * (n // 5)
    if kind == "common":  # the i-th commonest falls as 1 / i
        return (torch.exp(torch.rand(m, generator=g, device="cuda").double() * np.log(n + 1)) - 1).long().clamp(0, n - 1)
    if kind == "padding":
        return torch.where(torch.rand(m, generator=g, device="cuda") < 0.5, -1, n + 5)
    ids = torch.randint(0, n, (m,), generator=g, device="cuda")
    ids[torch.rand(m, generator=g, device="cuda") < 0.1] = -1
    return ids


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient(O, d, dtype):
    g = gen(d)
    for m, n, kind in ((1, 1, "one"), (3, 40, "any"), (50, 7, "any"), (700, 301, "common"), (1500, 90, "few")):
        grad = randn(g, m, d).to(TYPES[dtype])
        check_gradient(O, grad, ids_of(g, m, n, kind), n)


# of one and of several tiles, their borders, and of chunks of every width
@pytest.mark.parametrize("m", [2, 15, 16, 17, 31, 32, 33, 48, 49, 4095, 4096, 4097, 8192, 12_289, 50_000, 150_001])
@pytest.mark.parametrize("kind", ["one", "few", "common", "any", "padding"])
def test_gradient_of_runs(O, m, kind):
    g = gen(m)
    for n, d in ((40, 24), (1000, 520) if m < 60_000 else (1000, 64)):
        check_gradient(O, randn(g, m, d), ids_of(g, m, n, kind), n)


@pytest.mark.parametrize("m,n,d", [(30_000, 20_000, 1024), (20_000, 3000, 2056), (9000, 100, 8192)])
@pytest.mark.parametrize("kind", ["few", "common"])
def test_gradient_of_wide_chunks(O, m, n, d, kind):
    g = gen(m)
    check_gradient(O, randn(g, m, d).bfloat16(), ids_of(g, m, n, kind), n)


@pytest.mark.parametrize("m,widths", [(1024, (8, 100, 600)), (1025, (5, 24, 600)), (2048, (3, 64, 1001)), (2049, (7, 130, 520)),
                                      (2896, (9, 513)), (4095, (1, 65, 512)), (4096, (8, 256, 511))])
@pytest.mark.parametrize("kind", ["one", "few", "common", "any", "padding"])
def test_gradient_of_unsorted_tokens(O, m, widths, kind):
    """Up to 4096 tokens, which are looked through; runs that a workgroup adds up."""
    for d in widths:
        g = gen(m + d)
        check_gradient(O, randn(g, m, d), ids_of(g, m, 700, kind), 700)


@pytest.mark.parametrize("d", [5, 130, 520])
@pytest.mark.parametrize("share", [0.5, 1.0])
def test_gradient_of_a_batch_that_is_padded_with_a_row(O, d, share):
    """A run of thousands of chunks; whole numbers, whose sums are exact in any order."""
    m, n = 66_000, 800
    g = gen(d)
    ids = torch.randint(0, n, (m,), generator=g, device="cuda")
    ids[torch.rand(m, generator=g, device="cuda") < share] = 300
    grad = torch.randint(-2, 3, (m, d), generator=g, device="cuda").bfloat16()
    want = torch.zeros((n, d), dtype=torch.float64, device="cuda").index_add_(0, ids, grad.double())
    assert torch.equal(O.embed_backward(grad, ids, n, dtype="float32").double(), want)


@pytest.mark.parametrize("m", [524_288, 524_289, 3_000_017])
@pytest.mark.parametrize("kind", ["few", "common", "any"])
def test_gradient_of_many_tokens(O, m, kind):
    """More tiles than a workgroup adds up; whole numbers, whose sums are exact in any order."""
    g = gen(m)
    n, d = 70_000, 4
    ids = ids_of(g, m, n, kind)
    grad = torch.randint(-2, 3, (m, d), generator=g, device="cuda").half()
    at = torch.where((ids >= 0) & (ids < n), ids, n)
    want = torch.zeros((n + 1, d), dtype=torch.float64, device="cuda").index_add_(0, at, grad.double())[:n]
    assert torch.equal(O.embed_backward(grad, ids, n, dtype="float32").double(), want)


@pytest.mark.parametrize("n", [1, 2, 511, 512, 513, 300_000, 5_000_000, 140_000_000])
@pytest.mark.parametrize("m", [100, 9000])
def test_gradient_of_tables_of_any_length(O, n, m):
    """Ids of one to four digits; their ends."""
    g = gen(n)
    ids = torch.randint(0, n, (m,), generator=g, device="cuda")
    ids[0], ids[1], ids[2], ids[3] = 0, n - 1, n, -(2**40)
    grad = randn(g, m, 1).half()
    got = O.embed_backward(grad, ids, n)
    want = torch.zeros((n, 1), dtype=torch.float64, device="cuda")
    keep = (ids >= 0) & (ids < n)
    want.index_put_((ids[keep],), grad[keep].double(), accumulate=True)
    close(got, want, rounded(m * E * 4 * max(1.0, m / n), want, "float16"), "gradient")


@pytest.mark.parametrize("m", [700, 1500, 30_000])
@pytest.mark.parametrize("kind", ["one", "few", "common", "any", "padding"])
@pytest.mark.parametrize("n,d,apart", [(45_000, 1001, 0), (9000, 7, 1), (5000, 64, 5), (301, 513, 1), (40, 300_000, 0), (150_000, 512, 0)])
def test_every_row_without_an_id_is_cleared(O, m, kind, n, d, apart):
    """Tables larger than what is filled beside the sort, and rows that lie apart; whatever the memory held."""
    from octex_amd import scores

    if m * d > 40_000_000:
        m = 40_000_000 // d
    g = gen(m)
    ids = ids_of(g, m, n, kind)
    grad = torch.randint(-4, 5, (m, d), generator=g, device="cuda").bfloat16()
    wide = torch.full((n, d + apart), float("nan"), device="cuda")
    out, column = wide[:, :d], ids[:, None]
    c = scores._Call(grad, "grad", scores.FLOATS)
    c.run_sized("octexEmbedBackward", c.matrix(grad), c.matrix(column), 1.0, 0, c.matrix(out))
    at = torch.where((ids >= 0) & (ids < n), ids, n)
    want = torch.zeros((n + 1, d), device="cuda").index_add_(0, at, grad.float())[:n]  # whole numbers: exact in any order
    assert torch.equal(out, want)
    assert wide[:, d:].isnan().all()


@pytest.mark.parametrize("given", TYPES)
@pytest.mark.parametrize("result", TYPES)
def test_gradient_types(O, given, result):
    g = gen(3)
    for d in (5, 72, 600):
        grad = randn(g, 300, d).to(TYPES[given])
        check_gradient(O, grad, ids_of(g, 300, 60, "common"), 60, dtype=result)


@pytest.mark.parametrize("d", [3, 24, 513])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_rows_apart_and_ids_of_other_kinds(O, d, dtype):
    g = gen(4)
    grad = randn(g, 900, d).to(TYPES[dtype])
    ids = ids_of(g, 900, 200, "any")
    check_gradient(O, grad, ids, 200, given=padded(grad, 5))
    check_gradient(O, grad, torch.stack([ids, ids * 0], 1)[:, 0], 200)
    check_gradient(O, grad, ids.int(), 200)


def test_gradient_of_nothing(O):
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    none = z(0, dtype=torch.int64)
    assert torch.equal(O.embed_backward(z(0, 30), none, 7), z(7, 30))
    assert O.embed_backward(z(5, 30), z(5, dtype=torch.int64), 0).shape == (0, 30)
    assert O.embed_backward(z(5, 0), z(5, dtype=torch.int64), 4).shape == (4, 0)
    ones = z(7, 30) + 1
    assert O.embed_backward(z(0, 30), none, add_to=ones) is ones and (ones == 1).all()


def test_gradient_of_infinities(O):
    """A NaN or infinity reaches its own row alone."""
    g = gen(6)
    grad = randn(g, 500, 40)
    ids = torch.arange(500, device="cuda") % 100
    grad[3, 2], grad[4, 5], grad[104, 5], grad[5, 1] = float("nan"), float("inf"), float("-inf"), float("inf")
    got = O.embed_backward(grad, ids, 100)
    assert torch.isnan(got[3, 2]) and torch.isnan(got[4, 5]) and got[5, 1] == float("inf")
    assert (~torch.isfinite(got)).sum() == 3


@pytest.mark.parametrize("m,n,d", [(3000, 50, 40), (30_000, 900, 264)])
def test_results_repeat(O, m, n, d):
    """The order of a row's sum is that of the ids alone, on any stream."""
    g = gen(m)
    grad, ids = randn(g, m, d), ids_of(g, m, n, "common")
    want = O.embed_backward(grad, ids, n)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(4)]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(O.embed_backward(grad, ids, n))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got)


@pytest.mark.parametrize("m,n,d", [(40, 30, 24), (9000, 900, 264)])
def test_captured_calls_replay(O, m, n, d):
    g = gen(m)
    grad, ids, table = randn(g, m, d), ids_of(g, m, n, "common"), randn(g, n, d).bfloat16()
    sums = torch.zeros((n, d), device="cuda")
    work = lambda: [O.embed(table, ids, scale=3.0), O.embed_backward(grad, ids, n), O.embed_backward(grad, ids, add_to=sums)]
    graph, out = captured(work)
    for _ in range(3):
        grad.copy_(randn(g, m, d)), ids.copy_(ids_of(g, m, n, "any"))
        sums.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = sums.clone()
        sums.zero_()
        want = work()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(again, sums)


def test_rows_beyond_32_bit_offsets(O):
    g = gen(7)
    n, d = 1_200_000, 4096
    table = torch.zeros((n, d), dtype=torch.float16, device="cuda")
    ids = torch.tensor([0, n - 1, n - 2, n // 2, 1_048_576, 524_288], device="cuda")
    rows = randn(g, 6, d).half()
    table[ids] = rows
    assert torch.equal(O.embed(table, ids), rows)
    assert O.embed_backward(rows, ids, add_to=table.zero_()) is table
    assert torch.equal(table[ids], rows) and torch.count_nonzero(table.sum(1)) <= 6
    out = O.embed_backward(rows, ids, n)
    assert torch.equal(out[ids], rows) and torch.equal(out, table)
    del table, out
    many = torch.zeros((n, d), dtype=torch.float16, device="cuda")  # gradients
    many[ids] = rows
    at = torch.full((n,), -1, device="cuda")
    at[ids] = torch.arange(6, device="cuda")
    assert torch.equal(O.embed_backward(many, at, 6), rows)
    del many
    assert torch.equal(O.embed(rows, at)[ids], rows)


def test_gradient_and_lookup_are_adjoint(O):
    """sum(embed(T) G) = sum(T embed_backward(G)), both sides in 64 bits from results of 32."""
    g = gen(8)
    table, ids, grad = randn(g, 300, 50), ids_of(g, 2000, 300, "any"), randn(g, 2000, 50)
    left = (O.embed(table, ids, scale=1.7).double() * grad.double()).sum()
    right = (table.double() * O.embed_backward(grad, ids, 300, scale=1.7).double()).sum()
    assert abs(left - right) < 1e-3


def test_versions_of_what_is_added_to(O):
    sums = torch.zeros((5, 8), device="cuda")
    before = sums._version
    O.embed_backward(torch.ones((2, 8), device="cuda"), torch.tensor([1, 1], device="cuda"), add_to=sums)
    assert sums._version > before and sums[1, 0] == 2


def test_refusals(O):
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    ids, t8 = z(4, dtype=torch.int64), z(9, 16, dtype=torch.int8)
    for call, error, text in [
        (lambda: O.embed(t8, ids), TypeError, "row_scales"), (lambda: O.embed(z(9, 16), ids, row_scales=z(9)), TypeError, "int8"),
        (lambda: O.embed(t8, ids, row_scales=z(8)), ValueError, "row_scales has shape"),
        (lambda: O.embed(z(9, 16), z(4)), TypeError, "int64 or int32"),
        (lambda: O.embed(z(9, 16), ids, dtype="int8"), ValueError, "float32"),
        (lambda: O.embed(z(2, 3, 4), ids), ValueError, "matrix"),
        (lambda: O.embed(z(1, (1 << 24) + 1, dtype=torch.float16), ids), RuntimeError, "at most"),
        (lambda: O.embed_backward(z(4, 16), ids), TypeError, "number of rows"),
        (lambda: O.embed_backward(z(4, 16), ids, -1), ValueError, "-1 rows"),
        (lambda: O.embed_backward(z(3, 16), ids, 9), ValueError, "ids"),
        (lambda: O.embed_backward(z(4, 16), ids[None], 9), ValueError, "ids"),
        (lambda: O.embed_backward(z(4, 16), ids, 9, add_to=z(8, 16)), ValueError, "add_to"),
        (lambda: O.embed_backward(z(4, 16), ids, add_to=z(9, 15)), ValueError, "add_to"),
        (lambda: O.embed_backward(z(4, 16), ids, add_to=z(9, 16).cpu()), ValueError, "add_to"),
        (lambda: O.embed_backward(z(4, 16), ids, add_to=z(9, 16).double()), ValueError, "add_to"),
        (lambda: O.embed_backward(z(4, 16), ids, add_to=z(16, 9).t()), ValueError, "side by side"),
        (lambda: O.embed_backward(z(4, 16), ids, add_to=z(1, 16).expand(9, 16)), ValueError, "apart"),
        (lambda: O.embed_backward(z(4, 16), ids, dtype="float32", add_to=z(9, 16)), ValueError, "type"),
        (lambda: O.embed_backward(z(4, 16).cpu(), ids.cpu(), add_to=z(9, 16)), ValueError, "add_to"),
    ]:
        with pytest.raises(error, match=text):
            call()


def test_gradients_as_lists(O):
    got = O.embed_backward([[1.0, 2.0], [3.0, 4.0]], [1, 1], 3)
    assert isinstance(got, np.ndarray) and np.array_equal(got, [[0, 0], [4, 6], [0, 0]])
    got = O.embed_backward([[[1.0, 2.0]], [[3.0, 4.0]]], [[0], [2]], 3)
    assert np.array_equal(got, [[1, 2], [0, 0], [3, 4]])
    with pytest.raises(ValueError, match="ids"):
        O.embed_backward([[1.0, 2.0], [3.0, 4.0]], [1], 3)


@pytest.mark.parametrize("shape", [(2, 3), (0, 3), (2, 1, 4)])
def test_gradients_of_no_width(O, shape):
    ids = torch.zeros(shape, dtype=torch.int64, device="cuda")
    grad = torch.zeros((*shape, 0), device="cuda")
    assert O.embed_backward(grad, ids, 4).shape == (4, 0)
    sums = torch.zeros((4, 0), device="cuda")
    assert O.embed_backward(grad, ids, add_to=sums) is sums


def check_whole_numbers(O, m, n, d, kind):
    """Gradients of whole numbers, whose sums in 32 bits are exact in any order; the ends of the table have tokens, and places
    outside it."""
    g = gen(m + n + d)
    ids = ids_of(g, m, n, kind)
    if m >= 8:
        ids[1], ids[m // 2], ids[m - 2], ids[m - 1] = 0, n - 1, n, -(2**40)
    grad = torch.randint(-2, 3, (m, d), generator=g, device="cuda").half()
    inside = (ids >= 0) & (ids < n)
    want = torch.zeros((n, d), device="cuda").index_add_(0, ids[inside], grad[inside].float())
    assert torch.equal(O.embed_backward(grad, ids, n, dtype="float32"), want)
    sums = torch.ones((n, d), device="cuda")
    O.embed_backward(grad, ids, add_to=sums)
    assert torch.equal(sums, want + 1)


# Up to 1024 tokens are looked through, up to 4096 while m^2 ceil(d / 512) is at most 2^25, others are sorted: both sides.  A
# single workgroup sorts 2 tokens a thread up to 2048, 4 up to 4096, 8 up to 8192
@pytest.mark.parametrize("m,d", [(1024, 16_000), (1025, 15_872), (1025, 15_873), (2000, 4104), (2048, 4096), (2048, 4097),
                                 (2049, 3585), (2896, 2048), (2896, 2049), (3000, 2056), (4096, 1024), (4096, 1025), (4097, 8)])
@pytest.mark.parametrize("kind", ["one", "few", "common", "any", "padding"])
def test_gradient_on_both_sides_of_the_sort(O, m, d, kind):
    check_whole_numbers(O, m, 700, d, kind)


@pytest.mark.parametrize("m,d", [(300, 1600), (1024, 4100), (2896, 2000), (4096, 1024)])
@pytest.mark.parametrize("share", [0.3, 1.0])
def test_long_runs_of_wide_rows(O, m, d, share):
    """A slice's sums are those of its columns alone, bit for bit, whoever adds them up."""
    g = gen(m + d)
    ids = torch.randint(0, 500, (m,), generator=g, device="cuda")
    ids[torch.rand(m, generator=g, device="cuda") < share] = 77
    grad = randn(g, m, d)
    got = O.embed_backward(grad, ids, 500)
    for at in range(0, d - 511, 512):
        assert torch.equal(got[:, at : at + 512], O.embed_backward(grad[:, at : at + 512], ids, 500))
    check_gradient(O, grad, ids, 500)


# of one to four digits, by 2, 4 and 8 tokens a thread
@pytest.mark.parametrize("m,d", [(2048, 4104), (4096, 1032), (5000, 8), (8192, 1)])
@pytest.mark.parametrize("n", [1, 2, 511, 512, 513, 262_143, 262_144, 300_000])
@pytest.mark.parametrize("kind", ["common", "any"])
def test_digits_that_a_workgroup_sorts_alone(O, m, d, n, kind):
    check_whole_numbers(O, m, n, d, kind)


@pytest.mark.parametrize("m", [100, 4097, 8192, 9000, 66_000, 524_289])
@pytest.mark.parametrize("n", [1, 2, 3, 134_217_727, 134_217_728, 140_000_000])
def test_shortest_and_longest_tables(O, m, n):
    check_whole_numbers(O, m, n, 1, "any")


# of more tiles than a workgroup adds up, and of fewer
@pytest.mark.parametrize("m", [66_000, 524_288, 524_289, 600_001])
@pytest.mark.parametrize("kind", ["one", "common", "any", "padding"])
def test_three_digits_of_many_tiles(O, m, kind):
    check_whole_numbers(O, m, 300_000, 4, kind)
