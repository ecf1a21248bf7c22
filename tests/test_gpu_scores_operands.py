"""The operators on rows of scores on operands of several frameworks, each ordered on a stream of its own.  This module plays
one of these frameworks: it has a current stream (`cuda`), arrays that export DLPack, and from_dlpack."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def O():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import octex_amd

    cuda.stream = torch.cuda.Stream()
    return octex_amd


class cuda:
    stream = None  # the framework's current one

    class _Handle:
        def __init__(self, ptr):
            self.ptr = ptr

    @staticmethod
    def get_current_stream():
        return cuda._Handle(cuda.stream.cuda_stream)


class Array:
    """An array of this framework; its export orders its reader's stream after its own, as DLPack asks of it."""

    def __init__(self, t):
        self.t = t

    def __dlpack__(self, *, stream=None, **kw):
        if stream is not None and stream != cuda.stream.cuda_stream:
            reader = torch.cuda.ExternalStream(stream) if stream > 2 else torch.cuda.default_stream()
            reader.wait_stream(cuda.stream)
        return self.t.__dlpack__()

    def __dlpack_device__(self):
        return self.t.__dlpack_device__()


def from_dlpack(t):
    return Array(t)


class Nameless(Array):
    """The same of a framework that names no stream."""


Nameless.__module__ = "nowhere"


class Interface:
    """An array that has __cuda_array_interface__ alone, with the stream that it is ordered on."""

    def __init__(self, t):
        self.t = t
        code = cuda.stream.cuda_stream
        self.__cuda_array_interface__ = dict(shape=tuple(t.shape), typestr={torch.float32: "<f4", torch.int64: "<i8"}[t.dtype],
                                             data=(t.data_ptr(), False), version=3, stream=code)


Interface.__module__ = "nowhere"


def delay():
    """Some 10 ms of work on the current stream."""
    a = torch.ones((4096, 4096), device="cuda")
    for _ in range(8):
        a = a @ a / 4096


KINDS = {"torch": lambda t: t, "array": Array, "nameless": Nameless, "interface": Interface}


@pytest.mark.parametrize("logits,ids", [("array", "torch"), ("torch", "array"), ("torch", "interface"), ("interface", "torch"),
                                        ("nameless", "torch"), ("nameless", "array"), ("array", "interface"),
                                        ("interface", "array")])
def test_operands_of_several_frameworks_are_ordered(O, logits, ids):
    """Each operand changes behind work that is still on its own stream when the call is made, and again after the call, on the
    same stream: the results are those of its values at the call.  Nothing is synchronized in between.  (What a framework that
    names no stream does after the call is its own to order.)"""
    g = torch.Generator().manual_seed(3)
    m, n, k = 300, 5000, 4
    right = [torch.randn((m, n), generator=g).cuda(), torch.randint(0, n, (m, k), generator=g).cuda()]
    weight, teacher = torch.rand(m, generator=g).cuda(), torch.randn((m, k), generator=g).cuda()
    torch.cuda.synchronize()
    want = list(O.log_probs(*right, top=3)) + list(O.distill_step(weight, right[0], right[1], teacher))
    ours, theirs = torch.cuda.Stream(), torch.cuda.Stream()
    cuda.stream = theirs
    held = [torch.zeros_like(t) for t in right]
    streams = [ours if kind == "torch" else theirs for kind in (logits, ids)]
    for s in (ours, theirs):  # the allocator's first calls are made
        with torch.cuda.stream(s):
            delay()
    torch.cuda.synchronize()
    for s, t, r in zip(streams, held, right):
        with torch.cuda.stream(s):
            delay()
            t.copy_(r)
    with torch.cuda.stream(ours):
        x, i = (KINDS[kind](t) for kind, t in zip((logits, ids), held))
        r = O.log_probs(x, i, top=3)
        loss, grad = O.distill_step(weight, x, i, teacher)
    for kind, s, t in zip((logits, ids), streams, held):
        if kind != "nameless":
            with torch.cuda.stream(s):
                t.zero_()
    got = list(r) + [loss, grad]
    # what comes back is ordered on the first operand's stream, or on torch's
    with torch.cuda.stream(theirs if isinstance(got[0], Array) else ours):
        got = [(v.t if isinstance(v, Array) else v).clone() for v in got]
    torch.cuda.synchronize()
    assert isinstance(r.lse, Array) == (logits == "array")
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_codes_without_their_scales_are_refused(O):
    """int8 queries are codes: taken for values, they would be quantized once more, as if their scales were 1."""
    codes, scales = O.quantize_rows(torch.randn((3, 50), generator=torch.Generator().manual_seed(1)).cuda())
    for queries in (codes, codes.cpu(), codes.cpu().numpy(), codes[0], Nameless(codes)):
        with pytest.raises(TypeError, match="octex: int8 queries need their query_scales"):
            O.int8_scores(queries, codes, scales)
    s = O.int8_scores(codes.int().float(), codes, scales)  # whole numbers in a float type are values
    assert s.dtype == torch.float32 and s.shape == (3, 3)


def test_vectors_and_lists_of_ids(O):
    """One id a row, and its teacher's logit, as a tensor, numpy's, a list, or an array that has only DLPack."""
    g = torch.Generator().manual_seed(2)
    x, ids, teacher = torch.randn((4, 30), generator=g).cuda(), torch.tensor([3, 29, -1, 0]), torch.randn(4, generator=g)
    want = O.log_probs(x, ids.cuda()[:, None])
    loss, lse = O.distill(x, ids.cuda()[:, None], teacher.cuda()[:, None])
    torch.cuda.synchronize()
    for kind in (lambda t: t.cuda(), lambda t: t, lambda t: t.numpy(), lambda t: t.tolist(), lambda t: Nameless(t.cuda()),
                 lambda t: Nameless(t)):
        r = O.log_probs(x, kind(ids))
        assert r.log_probs.shape == (4,) and torch.equal(r.log_probs, want.log_probs[:, 0])
        one = kind(torch.ones(4))
        grad = O.log_probs_backward(one, None, x, kind(ids), r.lse, r.entropy)
        assert torch.equal(grad, O.log_probs_backward(torch.ones((4, 1)).cuda(), None, x, ids.cuda()[:, None], r.lse, r.entropy))
        assert torch.equal(O.distill(x, kind(ids), kind(teacher))[0], loss)
        assert torch.equal(O.distill_step(one, x, kind(ids), kind(teacher))[0], loss)
    r = O.log_probs(x.tolist(), ids[:, None].tolist())
    assert torch.equal(torch.as_tensor(r.log_probs), want.log_probs.cpu())


def test_types_of_scores_by_any_name(O):
    x = torch.randn((3, 50), generator=torch.Generator().manual_seed(6)).cuda()
    codes, scales = O.quantize_rows(x)
    for name in ("float32", "float16", "bfloat16"):
        names = [name, getattr(torch, name), f"torch.{name}"]
        if name != "bfloat16":
            names += [np.dtype(name), np.dtype(name).type]
        for dtype in names:
            assert O.int8_scores(x, codes, scales, dtype=dtype).dtype == getattr(torch, name)
    for dtype in (np.dtype("int8"), np.int32, torch.float64, "double"):
        with pytest.raises(ValueError, match="octex: scores are of type"):
            O.int8_scores(x, codes, scales, dtype=dtype)


def test_views_with_a_lazy_sign(O):
    """The imaginary part of a conjugate is a view of the values before their sign is turned."""
    z = torch.randn((4, 60), dtype=torch.complex64, generator=torch.Generator().manual_seed(8)).cuda()
    ids = torch.zeros((4, 1), dtype=torch.int64).cuda()
    w = torch._neg_view(torch.ones(4).cuda())
    x = z.conj().imag
    assert x.is_neg() and w.is_neg()
    for a, b in zip(O.log_probs(x, ids, top=2), O.log_probs(-z.imag, ids, top=2)):
        assert torch.equal(a, b)
    loss, grad = O.distill_step(w, x, ids, x[:, :1])
    want = O.distill_step(-torch.ones(4).cuda(), -z.imag, ids, -z.imag[:, :1])
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
