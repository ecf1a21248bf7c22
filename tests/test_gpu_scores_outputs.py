"""The C entries of the operators on rows of scores write their outputs and nothing else: outputs whose rows lie apart, at odd
places, between bytes that must stay as they are, have the values of dense ones."""

import ctypes as ct

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
GUARD = 0x5A


@pytest.fixture(scope="module")
def O():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd

    return octex_amd


@pytest.fixture(scope="module")
def S():
    from octex_amd import scores

    return scores


class Guarded:
    """A matrix or vector in the midst of guard bytes, `pad` elements between its rows, `odd` elements off a 256-byte place."""

    made = []

    def __init__(self, shape, dtype=torch.float32, pad=0, odd=1):
        size = torch.empty((), dtype=dtype).element_size()
        self.rows, self.cols = shape if len(shape) == 2 else (1, shape[0])
        self.stride = self.cols + pad
        elements = 256 // size + odd + self.rows * self.stride + 256
        self.bytes = torch.full((elements * size,), GUARD, dtype=torch.uint8, device="cuda")
        self.t = self.bytes.view(dtype).as_strided(shape, (self.stride, 1) if len(shape) == 2 else (1,), 256 // size + odd)
        Guarded.made.append(self)

    def matrix(self, S):
        return S._Matrix(self.t.data_ptr(), S._TYPES[str(self.t.dtype).replace("torch.", "")], self.rows, self.cols, self.stride)

    @property
    def at(self):
        return self.t.data_ptr()


def check(pairs):
    """The outputs' values are those of the dense ones, bit for bit; every other byte is as it was."""
    torch.cuda.synchronize()
    for what, got, want in pairs:
        assert got.t.dtype == want.dtype and torch.equal(got.t.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)), what
    for g in Guarded.made:
        if g.t.numel():
            g.t.view(torch.uint8 if g.t.dtype in (torch.int8, torch.uint8) else g.t.dtype).copy_(
                torch.full((g.t.element_size(),), GUARD, dtype=torch.uint8).view(g.t.dtype).cuda().expand(g.t.shape))
        assert (g.bytes == GUARD).all(), f"bytes beside an output of {tuple(g.t.shape)} were written"
    Guarded.made.clear()


def call(S, name, *args):
    from octex_amd import _lib

    if S._entry(name)(*args, torch.cuda.current_stream().cuda_stream) != _lib.CUVS_SUCCESS:
        raise RuntimeError(_lib.lib().cuvsGetLastErrorText().decode())


def sized(S, name, *args):
    """A call with exactly the workspace that it asks for, guarded."""
    size = ct.c_int64(-1)
    call(S, name, *args, None, 0, ct.addressof(size))
    w = Guarded((size.value,), torch.int8, odd=0) if size.value else None
    assert w is None or w.at % 256 == 0
    call(S, name, *args, w.at if w else None, size.value, None)


def whole(S, t):
    return S._Matrix(t.data_ptr(), S._TYPES[str(t.dtype).replace("torch.", "")], t.shape[0], t.shape[1], t.stride(0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 7, 100, 1000, 4099, 20_011])
def test_codes(O, S, k, dtype):
    x = torch.randn((21, k), generator=torch.Generator().manual_seed(k)).to(TYPES[dtype]).cuda()
    want = O.quantize_rows(x)
    for pad, odd in ((0, 1), (1, 0), (13, 3)):
        codes, scales = Guarded((21, k), torch.int8, pad, odd), Guarded((21,))
        call(S, "octexQuantizeRows", whole(S, x), codes.matrix(S), scales.at)
        check([("codes", codes, want[0]), ("scales", scales, want[1])])


@pytest.mark.parametrize("m,k,n", [(1, 1024, 301), (5, 4097, 700), (9, 960, 103), (20, 64, 300), (24, 1000, 8203), (65, 129, 190),
                                   (300, 512, 299), (40, 999, 3001), (600, 1040, 12_345), (1000, 512, 30_001),
                                   (2050, 4112, 4101), (300, 100, 20_001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores(O, S, m, k, n, dtype):
    g = torch.Generator().manual_seed(m + k + n)
    x = torch.randn((m, k), generator=g).cuda()
    rows, scales = O.quantize_rows(torch.randn((n, k), generator=g).cuda())
    for q, qs in (O.quantize_rows(x), (x, None)):
        want = O.int8_scores(q, rows, scales, query_scales=qs, dtype=dtype)
        for pad, odd in ((0, 1), (1, 0), (37, 5), (64 - n % 64, 0)):
            out = Guarded((m, n), TYPES[dtype], pad, odd)
            sized(S, "octexInt8Scores", whole(S, q), None if qs is None else qs.data_ptr(), whole(S, rows), scales.data_ptr(),
                  None, out.matrix(S))
            check([("scores", out, want)])


# rows of a few columns, in parts, and of every number of threads
ROWS = [(3, 1), (3, 5), (2, 131_079), (200, 9001), (600, 9000), (2100, 1001), (2100, 4001), (130, 70_001)]


@pytest.mark.parametrize("m,n", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs(O, S, m, n, dtype):
    g = torch.Generator().manual_seed(m + n)
    x = (2 * torch.randn((m, n), generator=g)).to(TYPES[dtype]).cuda()
    ids = torch.randint(-1, n, (m, 3), generator=g).cuda()
    gl, gh = torch.randn((m, 3), generator=g).cuda(), torch.randn(m, generator=g).cuda()
    for top in (0, 1, 20, 64):
        want = O.log_probs(x, ids, top=top)
        logp, entropy, lse = Guarded((m, 3)), Guarded((m,)), Guarded((m,))
        top_logp, top_ids = Guarded((m, top)), Guarded((m, top), torch.int64)
        sized(S, "octexLogProbs", whole(S, x), whole(S, ids), 1.0, top, logp.at, entropy.at, lse.at, top_logp.at, top_ids.at)
        check(list(zip(("log_probs", "entropy", "lse", "top_log_probs", "top_ids"), (logp, entropy, lse, top_logp, top_ids), want)))
    r = want
    want = O.log_probs_backward(gl, gh, x, ids, r.lse, r.entropy)
    for pad, odd in ((0, 1), (1, 0), (37, 3)):
        grad = Guarded((m, n), TYPES[dtype], pad, odd)
        call(S, "octexLogProbsBackward", whole(S, x), whole(S, ids), 1.0, gl.data_ptr(), gh.data_ptr(), r.lse.data_ptr(),
             r.entropy.data_ptr(), grad.matrix(S))
        check([("gradient", grad, want)])


@pytest.mark.parametrize("m,n", ROWS + [(9000, 500), (520, 66_003), (300, 40_001), (2, 150_001), (4100, 17_001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill(O, S, m, n, dtype):
    k = 70 if dtype == "float16" else 1
    g = torch.Generator().manual_seed(m + n + k)
    x = (2 * torch.randn((m, n), generator=g)).to(TYPES[dtype]).cuda()
    ids = torch.randint(-1, n, (m, k), generator=g).cuda()
    teacher, w = torch.randn((m, k), generator=g).cuda(), torch.rand(m, generator=g).cuda()
    args = whole(S, x), whole(S, ids), whole(S, teacher), 1.5
    want = O.distill(x, ids, teacher, temperature=1.5)
    back = O.distill_backward(w, x, ids, teacher, want[1], temperature=1.5)
    step = O.distill_step(w, x, ids, teacher, temperature=1.5)
    loss, lse = Guarded((m,)), Guarded((m,))
    sized(S, "octexDistill", *args, loss.at, lse.at)
    check([("loss", loss, want[0]), ("lse", lse, want[1])])
    for pad, odd in ((0, 1), (1, 0), (37, 3)):
        grad = Guarded((m, n), TYPES[dtype], pad, odd)
        call(S, "octexDistillBackward", *args, w.data_ptr(), want[1].data_ptr(), grad.matrix(S))
        check([("gradient", grad, back)])
        loss, lse, grad = Guarded((m,)), Guarded((m,)), Guarded((m, n), TYPES[dtype], pad, odd)
        sized(S, "octexDistillStep", *args, w.data_ptr(), loss.at, lse.at, grad.matrix(S))
        check([("loss of a step", loss, step[0]), ("gradient of a step", grad, step[1])])
