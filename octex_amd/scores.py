"""Operators on rows of scores: what a model that makes the queries, or reads the neighbors, computes next to a search.

    codes, scales = octex.quantize_rows(vectors)                     # once: 8 bits a value, a scale a row
    logits = octex.int8_scores(queries, codes, scales)               # every query against every row
    r = octex.log_probs(logits, ids, top=10)                         # log p of given ids, entropy, alternatives
    distances, neighbors = index.search(queries, k=10)               # a teacher: its nearest rows ...
    loss, grad = octex.distill_step(weights, logits, neighbors, -distances, temperature=2.0)   # ... and the lesson
    r, grad = octex.policy_step(weights, logits, ids, old, advantages)   # or one from rewards: a policy's clipped loss
    r, grad = octex.balance_step(None, router, experts, weight=0.01)     # rows spread evenly over experts or shards

Every operator is a hand-written kernel and takes matrices whose rows may lie apart (a slice of a padded vocabulary's
columns, say).  Operands in GPU memory are read in place: the work is ordered on the first one's stream (torch's current
stream, or the one its framework names) and not waited for; operands of other streams precede it, and what those streams do
next comes after it.  Host operands are copied to the GPU and results come back as the first operand is.  Types that an
operator does not take are converted, as for a search.  Results carry no autograd graph: the gradients have calls of their own.
"""

import collections
import contextlib
import ctypes as ct
import functools
import sys

import numpy as np

from . import _arrays, _lib

FLOATS = ("float32", "float16", "bfloat16")
INTS = ("int64", "int32")
_TYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "int8": 3, "int32": 4, "int64": 5}

LogProbs = collections.namedtuple("LogProbs", "log_probs entropy lse top_log_probs top_ids")
PolicyLoss = collections.namedtuple("PolicyLoss", "loss log_probs entropy lse")
BalanceLoss = collections.namedtuple("BalanceLoss", "loss counts rows probs lse")


class _Matrix(ct.Structure):
    """struct octexMatrix (octex_amd.h)."""

    _fields_ = [("data", ct.c_void_p), ("type", ct.c_int32), ("rows", ct.c_int64), ("cols", ct.c_int64),
                ("stride", ct.c_int64)]


_P, _I32, _I64, _F = ct.c_void_p, ct.c_int32, ct.c_int64, ct.c_float
_M = ct.POINTER(_Matrix)
_SIZED = [_P, _I64, _P]  # workspace, bytes, size
_POLICY = [_M, _M, _F, _P, _P, _P, _F, _F, _F, _F]  # logits, ids, temperature, a row's terms, bounds and weights
_ENTRIES = {
    "octexQuantizeRows": [_M, _M, _P],
    "octexInt8Scores": [_M, _P, _M, _P, _P, _M] + _SIZED,
    "octexLogProbs": [_M, _M, _F, _I32, _P, _P, _P, _P, _P] + _SIZED,
    "octexLogProbsBackward": [_M, _M, _F, _P, _P, _P, _P, _M],
    "octexDistill": [_M, _M, _M, _F, _P, _P] + _SIZED,
    "octexDistillBackward": [_M, _M, _M, _F, _P, _P, _M],
    "octexDistillStep": [_M, _M, _M, _F, _P, _P, _P, _M] + _SIZED,
    "octexPolicyLoss": _POLICY + [_P, _P, _P, _P] + _SIZED,
    "octexPolicyLossBackward": _POLICY + [_P, _P, _P, _P, _M],
    "octexPolicyLossStep": _POLICY + [_P, _P, _P, _P, _P, _M] + _SIZED,
    "octexBalanceLoss": [_M, _M, _F, _F, _P, _P, _P, _P, _P, _P, _M] + _SIZED,
    "octexBalanceLossBackward": [_M, _M, _F, _F, _P, _P, _P, _M],
    "octexEmbed": [_M, _P, _M, _F, _M],
    "octexEmbedBackward": [_M, _M, _F, _I32, _M] + _SIZED,
}


@functools.lru_cache(None)
def _entry(name):
    f = getattr(_lib.lib(), name)
    f.argtypes = _ENTRIES[name] + [_P]  # the stream
    return f


@functools.lru_cache(None)
def _torch():
    """torch, the names of its element types, and the raw handle of a GPU's current stream."""
    import torch

    names = {getattr(torch, n): n for n in _TYPES}
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the public call makes an object of 2 us
    return torch, names, raw if raw is not None else lambda index: torch.cuda.current_stream(index).cuda_stream


_HERE = contextlib.nullcontext()
_WORKSPACES = {}  # bytes, by entry and sizes


class _Call:
    """One call's operands and results, all on one GPU, and the stream that they are ordered on: torch's current one, or
    (`side`) another that the first operand's framework names.  `others` are the streams of the remaining operands."""

    __slots__ = ("torch", "names", "origin", "device", "stream", "side", "others", "on_host", "foreign", "first", "lead",
                 "scratch")

    def __init__(self, first, name, types, flat=False):
        self.torch, self.names, raw_stream = _torch()
        self.origin, self.side, self.others = first, None, ()
        self.foreign = not isinstance(first, self.torch.Tensor) and _arrays.is_foreign_device(first)
        t = first if isinstance(first, self.torch.Tensor) else self.view(first)
        self.on_host = not t.is_cuda
        self.device = self.torch.device("cuda", self.torch.cuda.current_device()) if self.on_host else t.device
        self.stream = raw_stream(self.device.index)
        if self.foreign and t.is_cuda:  # of a framework that names no stream: its export has ordered it on torch's
            named = _arrays.named_stream(first)
            if named is not None and named != self.stream:
                self.stream, self.side = named, self.external(named)
        if flat:
            self.lead = t.shape[:-1]
            if t.ndim > 2:  # all but the last dimension are one
                with self.context():
                    t = t.flatten(0, -2)
        self.first = self.take(t, name, types)

    def view(self, a):
        """Any array as a torch tensor in the memory where it lies."""
        if _arrays.is_foreign_device(a):
            return self.torch.from_dlpack(a) if hasattr(a, "__dlpack__") else self.torch.as_tensor(a, device="cuda")
        x = np.asarray(a)  # torch takes no views of read-only arrays, nor backward ones
        return self.torch.from_numpy(x if x.flags.writeable and min(x.strides, default=0) >= 0 else x.copy())

    def external(self, handle):
        cuda = self.torch.cuda
        return cuda.ExternalStream(handle, device=self.device) if handle else cuda.default_stream(self.device)

    def own_stream(self):
        return self.side if self.side is not None else self.torch.cuda.current_stream(self.device)

    def join(self, stream):
        """Orders the call after all that `stream` holds; run orders what the stream does next after the call."""
        if stream not in self.others:
            self.own_stream().wait_stream(stream)
            self.others += (stream,)

    def array(self, a):
        """An operand behind the first as a torch tensor in the memory where it lies, ordered with the call."""
        if isinstance(a, self.torch.Tensor):
            if self.side is not None and a.is_cuda:
                self.join(self.torch.cuda.current_stream(self.device))
            return a
        if not _arrays.is_foreign_device(a):
            return self.view(a)
        with self.context():  # DLPack orders its producer on the stream that is current
            t = self.view(a)
        if t.is_cuda:  # __cuda_array_interface__ leaves that to its reader
            named = _arrays.named_stream(a)
            if named is not None and named != self.stream:
                self.join(self.external(named))
        return t

    def take(self, t, name, types, ndim=2, shape=None):
        """The operand (as array gives it) on the call's GPU: of one of `types` (else converted to the first), the elements
        of a row side by side.  A vector is one row unless ndim is 1."""
        torch = self.torch
        if t.device != self.device:
            if t.is_cuda:
                raise ValueError(f"octex: {name} lies on {t.device}, the other operands on {self.device}")
            if t.device.type != "cpu":
                raise TypeError(f"octex: {name} must lie in host or GPU memory, not on {t.device}")
            with self.context():
                t = t.to(self.device)
        if self.names.get(t.dtype) not in types:
            if types in (("int8",), ("int64",)) or (types is INTS and t.is_floating_point()):
                raise TypeError(f"octex: {name} must be {' or '.join(types)}, not {str(t.dtype).replace('torch.', '')}")
            with self.context():
                t = t.to(getattr(torch, types[0]))
        if t.ndim != ndim:
            if ndim == 2 and t.ndim == 1:
                t = t[None, :]
            else:
                raise ValueError(f"octex: {name} must be a {'matrix' if ndim == 2 else 'vector'}, "
                                 f"not of {t.ndim} dimensions")
        s = t.shape
        if shape is not None and s != shape:
            raise ValueError(f"octex: {name} has shape {tuple(s)}, expected {tuple(shape)}")
        if t.is_neg():  # a view whose sign torch has yet to turn in memory, as of a conjugate's imaginary part
            with self.context():
                t = t.resolve_neg()
        if not t.is_contiguous() and (s[-1] > 1 and t.stride(-1) != 1 or (ndim == 2 and s[0] > 1 and t.stride(0) < s[1])):
            with self.context():
                t = t.contiguous()
        return t

    def dense(self, a, name, shape):
        """A float32 operand without gaps between its rows."""
        t = self.take(self.array(a), name, ("float32",), len(shape), shape)
        if t.is_contiguous():
            return t
        with self.context():
            return t.contiguous()

    def context(self):
        """For torch's own work (conversions, allocations) on the call's stream."""
        return _HERE if self.side is None else self.torch.cuda.stream(self.side)

    def matrix(self, t):
        rows, cols = t.shape
        return _Matrix(t.data_ptr(), _TYPES[self.names[t.dtype]], rows, cols, max(t.stride(0), cols))

    def new(self, *shapes, dtype=None):
        """New results: float32, or of a torch type."""
        empty, device, dtype = self.torch.empty, self.device, dtype or self.torch.float32
        if self.side is not None:
            with self.context():
                out = [empty(s, dtype=dtype, device=device) for s in shapes]
        else:
            out = [empty(s, dtype=dtype, device=device) for s in shapes]
        return out if len(out) > 1 else out[0]

    def like(self, t):
        """A new dense result of t's shape and type (quicker than by its shape)."""
        if self.side is not None or not t.is_contiguous():
            return self.new(t.shape, dtype=t.dtype)
        return self.torch.empty_like(t)

    def run(self, entry, *args):
        if _entry(entry)(*args, self.stream) != _lib.CUVS_SUCCESS:
            raise _lib.OctexError(_lib.lib().cuvsGetLastErrorText().decode())
        for stream in self.others:
            stream.wait_stream(self.own_stream())

    def run_sized(self, entry, *args, sizes=None):
        """run with the workspace that the arguments need; its tensor is kept with the call.  Where `sizes` (the entry and all
        that its workspace depends on: sizes and types) is given, the answer is asked for once."""
        need = _WORKSPACES.get(sizes)
        if need is None:
            size = _I64(0)
            self.run(entry, *args, None, 0, ct.addressof(size))
            need = size.value
            if sizes is not None:
                if len(_WORKSPACES) >= 4096:
                    _WORKSPACES.clear()
                _WORKSPACES[sizes] = need
        if need == 0:
            return self.run(entry, *args, None, 0, None)
        self.scratch = self.new((need,), dtype=self.torch.int8)
        return self.run(entry, *args, self.scratch.data_ptr(), need, None)

    def give(self, t):
        """A result in the framework, and the memory, of the first operand."""
        if not self.on_host and not self.foreign:
            return t
        if self.on_host:
            t = t.cpu()
        if self.foreign:
            conv = getattr(sys.modules.get(_arrays._module_of(self.origin)), "from_dlpack", None)
            if conv is not None:
                with self.context():
                    return conv(t)
            if self.side is not None:  # a torch tensor after all, which is read on torch's stream
                current = self.torch.cuda.current_stream(self.device)
                current.wait_stream(self.side)
                t.record_stream(current)
            return t
        return t if isinstance(self.origin, self.torch.Tensor) else t.numpy()


def quantize_rows(x):
    """(codes, scales) of the rows of x [m, k] in 8 bits: scale = max |x| / 127, as the float32 product with 1 / 127, code = the
    whole number nearest to x / scale (ties to even): x is about codes * scales[:, None].  torch's x.abs().amax(1) / 127 is that
    product on the GPU; on the CPU, as numpy's, it is a quotient, which differs by one unit in some rows.

    A row of zeros has scale 0; a row with a NaN or an infinity has scale NaN, which makes all its scores NaN.
    """
    c = _Call(x, "x", FLOATS)
    x = c.first
    codes, scales = c.new(x.shape, dtype=c.torch.int8), c.new((x.shape[0],))
    c.run("octexQuantizeRows", c.matrix(x), c.matrix(codes), scales.data_ptr())
    return c.give(codes), c.give(scales)


def _float_type(c, dtype, what, of):
    """The torch type that `dtype` (a name, numpy's or torch's type) asks for."""
    if not isinstance(dtype, str):
        dtype = np.dtype(dtype).name if isinstance(dtype, (type, np.dtype)) else str(dtype)
    dtype = dtype.replace("torch.", "")
    if dtype not in FLOATS:
        raise ValueError(f"octex: {what} are of type {', '.join(FLOATS)}, not {dtype}")
    if dtype == "bfloat16" and c.on_host and not isinstance(c.origin, c.torch.Tensor):
        raise TypeError(f"octex: numpy has no bfloat16 for the {what} of its {of}")
    return getattr(c.torch, dtype)


def int8_scores(queries, rows, row_scales, *, query_scales=None, bias=None, dtype=None):
    """The scores [m, n] of every query against every row, a product in 8-bit integers:
    scores[i, j] = query_scales[i] * row_scales[j] * sum(queries[i] * rows[j]) + bias[j].

    `rows` [n, k] and `row_scales` [n] are quantize_rows' of an index's vectors, a pool of candidates or a vocabulary's
    embeddings.  `queries` [m, k] are codes with their `query_scales` [m], or floats, which the call quantizes the same way.
    The integer sums are exact.  With bias = -|row|^2 / 2 a query's scores rank the rows as squared distances do.  `dtype`
    ("float32", "float16" or "bfloat16") is that of the scores: the queries' own if they are floats, else float32.
    """
    coded = query_scales is not None
    c = _Call(queries, "queries", ("int8",) if coded else FLOATS + ("int8",))
    q = c.first
    if not coded and c.names[q.dtype] == "int8":
        raise TypeError("octex: int8 queries need their query_scales")
    rows = c.take(c.array(rows), "rows", ("int8",))
    (m, k), n = q.shape, rows.shape[0]
    if rows.shape[1] != k:
        raise ValueError(f"octex: queries have {k} values, rows {rows.shape[1]}")
    row_scales = c.dense(row_scales, "row_scales", (n,))
    if coded:
        query_scales = c.dense(query_scales, "query_scales", (m,))
    if bias is not None:
        bias = c.dense(bias, "bias", (n,))
    if dtype is None:
        dtype = "float32" if coded else c.names[q.dtype]
    out = c.new((m, n), dtype=_float_type(c, dtype, "scores", "queries"))
    c.run_sized("octexInt8Scores", c.matrix(q), query_scales.data_ptr() if coded else None, c.matrix(rows),
                row_scales.data_ptr(), None if bias is None else bias.data_ptr(), c.matrix(out))
    return c.give(out)


def _columns(c, a):
    """An operand as array gives it, a vector (one entry a row) as a matrix of one column; and its own shape."""
    t = c.array(a)
    return (t[:, None] if t.ndim == 1 else t), tuple(t.shape)


def _ids(c, ids, m):
    """The ids of m rows as a matrix, and the shape their values come back in."""
    ids, shape = _columns(c, ids)
    t = c.take(ids, "ids", INTS)
    if t.shape[0] != m:
        raise ValueError(f"octex: ids of {t.shape[0]} rows, logits of {m}")
    return t, shape


def log_probs(logits, ids, *, top=0, temperature=1.0):
    """Log probabilities under p = softmax(logits / temperature) of each row's given ids [m] or [m, t].

    Returns LogProbs(log_probs, entropy, lse, top_log_probs, top_ids): the ids' log probabilities in their shape, each row's
    entropy and log-sum-exp [m], and its `top` (at most 64) likeliest entries [m, top] by (logit, lowest id).  Everything is
    float32, top_ids int64.

    An id outside [0, n) is padding: its log probability is 0.  Logits of -inf (a masked vocabulary) have probability 0 and
    are no alternatives: top_ids is padded with -1, as a search's neighbors are, and top_log_probs with -inf.  A row of
    nothing but -inf has lse and log probabilities -inf and entropy 0; a row with a NaN or +inf is NaN.
    """
    c = _Call(logits, "logits", FLOATS)
    x = c.first
    m, top = x.shape[0], int(top)
    if not 0 <= top <= 64:
        raise ValueError(f"octex: 0 to 64 top entries, not {top}")
    t, shape = _ids(c, ids, m)
    logp, entropy, top_logp = c.new(shape, (m,), (m, top))
    lse = c.like(entropy)
    top_ids = c.new((m, top), dtype=c.torch.int64)
    c.run_sized("octexLogProbs", c.matrix(x), c.matrix(t), float(temperature), top, logp.data_ptr(), entropy.data_ptr(),
                lse.data_ptr(), top_logp.data_ptr(), top_ids.data_ptr())
    return LogProbs(c.give(logp), c.give(entropy), c.give(lse), c.give(top_logp), c.give(top_ids))


def log_probs_backward(grad_log_probs, grad_entropy, logits, ids, lse, entropy, *, temperature=1.0):
    """The gradient by the logits of sum(grad_log_probs * log_probs) + sum(grad_entropy * entropy), in the logits' type.

    lse and entropy are log_probs' of the same logits and temperature; either gradient may be None.  An id given more than
    once in a row gets the sum of its gradients.
    """
    c = _Call(logits, "logits", FLOATS)
    x = c.first
    m = x.shape[0]
    t, shape = _ids(c, ids, m)
    gl = None if grad_log_probs is None else c.dense(grad_log_probs, "grad_log_probs", shape)
    gh = None if grad_entropy is None else c.dense(grad_entropy, "grad_entropy", (m,))
    lse, entropy = c.dense(lse, "lse", (m,)), c.dense(entropy, "entropy", (m,))
    grad = c.like(x)
    c.run("octexLogProbsBackward", c.matrix(x), c.matrix(t), float(temperature), None if gl is None else gl.data_ptr(),
          None if gh is None else gh.data_ptr(), lse.data_ptr(), entropy.data_ptr(), c.matrix(grad))
    return c.give(grad)


def _teacher(logits, ids, teacher):
    c = _Call(logits, "logits", FLOATS)
    t, _ = _ids(c, ids, c.first.shape[0])
    return c, c.first, t, c.take(_columns(c, teacher)[0], "teacher", FLOATS, shape=t.shape)


def distill(logits, ids, teacher, *, temperature=1.0):
    """(loss, lse) of a student's logits [m, n] against a teacher's top logits [m, k] of the columns ids [m, k]:
    loss = sum q (ln q - ln p), q = softmax(teacher / temperature) over the listed ids, p = softmax(logits / temperature)
    over all columns.

    The teacher may be a search (its neighbors and -distances) or a larger model's top logits.  Ids outside [0, n), as a
    search's -1, are padding; a row that lists nothing has loss 0.  A listed logit of -inf that the teacher gives a
    probability makes its loss inf.  lse is the logits' log-sum-exp [m], for distill_backward.
    """
    c, x, t, teacher = _teacher(logits, ids, teacher)
    m = x.shape[0]
    loss = c.new((m,))
    lse = c.like(loss)
    c.run_sized("octexDistill", c.matrix(x), c.matrix(t), c.matrix(teacher), float(temperature), loss.data_ptr(),
                lse.data_ptr())
    return c.give(loss), c.give(lse)


def distill_backward(grad_loss, logits, ids, teacher, lse, *, temperature=1.0):
    """The gradient by the logits of sum(grad_loss * loss), in the logits' type: grad_loss (p - q) / temperature.

    lse is distill's of the same logits and temperature.  A row that lists nothing has gradient 0.
    """
    c, x, t, teacher = _teacher(logits, ids, teacher)
    m = x.shape[0]
    g, lse = c.dense(grad_loss, "grad_loss", (m,)), c.dense(lse, "lse", (m,))
    grad = c.like(x)
    c.run("octexDistillBackward", c.matrix(x), c.matrix(t), c.matrix(teacher), float(temperature), g.data_ptr(),
          lse.data_ptr(), c.matrix(grad))
    return c.give(grad)


def distill_step(grad_loss, logits, ids, teacher, *, temperature=1.0):
    """(loss, grad): distill and distill_backward in one call, which reads the logits less often."""
    c, x, t, teacher = _teacher(logits, ids, teacher)
    m = x.shape[0]
    g = c.dense(grad_loss, "grad_loss", (m,))
    loss, grad = c.like(g), c.like(x)
    lse = c.like(loss)
    c.run_sized("octexDistillStep", c.matrix(x), c.matrix(t), c.matrix(teacher), float(temperature), g.data_ptr(),
                loss.data_ptr(), lse.data_ptr(), c.matrix(grad))
    return c.give(loss), c.give(grad)


def _policy(logits, ids, old_log_probs, advantages, ref_log_probs, clip, kl, entropy, temperature):
    """A call on a policy's rows: its operands, and the arguments that all of its entries begin with."""
    c = _Call(logits, "logits", FLOATS)
    x = c.first
    m = x.shape[0]
    t = c.array(ids)
    if t.ndim == 1:  # a column of m rows
        t = c.take(t, "ids", INTS, 1, (m,))
        column = _Matrix(t.data_ptr(), _TYPES[c.names[t.dtype]], m, 1, 1)
    else:
        t = c.take(t, "ids", INTS, shape=(m, 1))
        column = c.matrix(t)
    terms = [c.dense(old_log_probs, "old_log_probs", (m,)), c.dense(advantages, "advantages", (m,))]
    if kl != 0 and ref_log_probs is not None:
        terms.append(c.dense(ref_log_probs, "ref_log_probs", (m,)))
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    args = (c.matrix(x), column, float(temperature), terms[0].data_ptr(), terms[1].data_ptr(),
            terms[2].data_ptr() if len(terms) > 2 else None, 1.0 - low, 1.0 + high, float(kl), float(entropy))
    return c, x, (t, terms), args


def policy_loss(logits, ids, old_log_probs, advantages, *, ref_log_probs=None, clip=0.2, kl=0.0, entropy=0.0, temperature=1.0):
    """A policy's clipped loss on rows of logits [m, n]: of the id that each row sampled, ids [m], its log probability then,
    old_log_probs [m], and its advantage A [m]; with p = softmax(logits / temperature), r = p of the id / exp(old) and
    d = ref_log_probs - ln p of the id,

        loss = -min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(d) - 1 - d) - entropy H(p).

    `clip` is (low, high), or one number for both.  The KL term holds the policy to a reference model, whose log probabilities
    [m] it needs; at kl = 0 they are not read.  Returns PolicyLoss(loss, log_probs, entropy, lse), float32 [m] each.

    A row whose id lies outside [0, n), a prompt's token say, is padding: it is not read and has 0 everywhere.  An id whose
    logit is -inf has r = 0; with a KL term its loss is inf and its row's gradient not finite.  A row with a NaN or +inf is NaN.
    """
    c, x, keep, args = _policy(logits, ids, old_log_probs, advantages, ref_log_probs, clip, kl, entropy, temperature)
    r = PolicyLoss(*c.new(*[(x.shape[0],)] * 4))
    c.run_sized("octexPolicyLoss", *args, *[v.data_ptr() for v in r], sizes=("octexPolicyLoss", x.shape))
    return PolicyLoss(*map(c.give, r))


def policy_loss_backward(grad_loss, logits, ids, old_log_probs, advantages, result, *, ref_log_probs=None, clip=0.2, kl=0.0,
                         entropy=0.0, temperature=1.0):
    """The gradient by the logits of sum(grad_loss * loss), in the logits' type; `result` is policy_loss's of the same operands.

    A ratio beyond its bound, on the side where the loss is clipped, has no gradient; one at the bound has.
    """
    c, x, keep, args = _policy(logits, ids, old_log_probs, advantages, ref_log_probs, clip, kl, entropy, temperature)
    shape = (x.shape[0],)
    g = c.dense(grad_loss, "grad_loss", shape)
    saved = [c.dense(getattr(result, name), name, shape) for name in ("log_probs", "entropy", "lse")]
    grad = c.like(x)
    c.run("octexPolicyLossBackward", *args, g.data_ptr(), *[v.data_ptr() for v in saved], c.matrix(grad))
    return c.give(grad)


def policy_step(grad_loss, logits, ids, old_log_probs, advantages, *, ref_log_probs=None, clip=0.2, kl=0.0, entropy=0.0,
                temperature=1.0):
    """(PolicyLoss, grad): policy_loss and policy_loss_backward in one call, which reads rows of up to 256 KB (131,072 16-bit logits;
    half of that of fewer than 512 rows) once, and longer ones as often as the two calls do."""
    c, x, keep, args = _policy(logits, ids, old_log_probs, advantages, ref_log_probs, clip, kl, entropy, temperature)
    g = c.dense(grad_loss, "grad_loss", (x.shape[0],))
    r, grad = PolicyLoss(*[c.like(g) for _ in range(4)]), c.like(x)
    c.run_sized("octexPolicyLossStep", *args, g.data_ptr(), *[v.data_ptr() for v in r], c.matrix(grad),
                sizes=("octexPolicyLossStep", x.shape, x.dtype))
    return PolicyLoss(*map(c.give, r)), c.give(grad)


def _balance(logits, experts):
    c = _Call(logits, "logits", FLOATS)
    t = c.take(_columns(c, experts)[0], "experts", INTS)
    if t.shape[0] != c.first.shape[0]:
        raise ValueError(f"octex: experts of {t.shape[0]} rows, logits of {c.first.shape[0]}")
    return c, c.first, t


def _one(c, a, name, types):
    """One number, as an array of no dimension or one."""
    t = c.array(a)
    if t.ndim != 1:
        t = t.reshape(-1)
    return c.take(t, name, types, 1, (1,))


def _balance_results(c, x):
    m, e = x.shape
    counts, rows = c.new((e,), (), dtype=c.torch.int64)
    loss, probs, lse = c.new((), (e,), (m,))
    return BalanceLoss(loss, counts, rows, probs, lse)


def balance_loss(logits, experts, *, weight=1.0, z_weight=0.0):
    """How evenly rows are spread over experts (parts of a model, or shards of an index), from their logits [m, e] (e at most
    2048) and the experts that they chose, [m] or [m, k], log_probs' top_ids say:

        loss = weight e sum(f P) + z_weight mean(lse^2),

    f the experts' shares of all choices, P their mean probabilities under softmax(logits).  Returns BalanceLoss(loss, counts,
    rows, probs, lse): the loss and the number of rows that count as arrays of no dimension, the experts' choices [e] (int64),
    P [e], and the rows' log-sum-exp [m].

    Ids outside [0, e) are no choice (one that found its expert full); a row without a choice (a batch's padding) does not
    count: its lse is 0.  Logits of -inf have probability 0; a row of nothing else adds nothing to P or the loss.  A NaN or
    +inf makes the loss NaN.
    """
    c, x, t = _balance(logits, experts)
    r = _balance_results(c, x)
    c.run_sized("octexBalanceLoss", c.matrix(x), c.matrix(t), float(weight), float(z_weight), *[v.data_ptr() for v in r], None,
                None, sizes=("octexBalanceLoss", x.shape, t.shape, x.dtype))
    return BalanceLoss(*map(c.give, r))


def balance_loss_backward(grad_loss, logits, experts, result, *, weight=1.0, z_weight=0.0):
    """The gradient by the logits of grad_loss * loss, in the logits' type; the choices are constants.

    grad_loss is one number, as an array (None: 1).  `result` is balance_loss's of the same operands; one whose counts and rows
    were added up over the ranks of a job gives the gradient of the job's balance.
    """
    c, x, t = _balance(logits, experts)
    g = None if grad_loss is None else _one(c, grad_loss, "grad_loss", ("float32",))
    counts = c.take(c.array(result.counts), "counts", ("int64",), 1, (x.shape[1],))
    rows = _one(c, result.rows, "rows", ("int64",))
    grad = c.like(x)
    c.run("octexBalanceLossBackward", c.matrix(x), c.matrix(t), float(weight), float(z_weight), counts.data_ptr(),
          rows.data_ptr(), None if g is None else g.data_ptr(), c.matrix(grad))
    return c.give(grad)


def balance_step(grad_loss, logits, experts, *, weight=1.0, z_weight=0.0):
    """(BalanceLoss, grad): balance_loss and balance_loss_backward in one call, which reads the logits once."""
    c, x, t = _balance(logits, experts)
    g = None if grad_loss is None else _one(c, grad_loss, "grad_loss", ("float32",))
    r, grad = _balance_results(c, x), c.like(x)
    c.run_sized("octexBalanceLoss", c.matrix(x), c.matrix(t), float(weight), float(z_weight), *[v.data_ptr() for v in r],
                None if g is None else g.data_ptr(), c.matrix(grad), sizes=("octexBalanceLoss", x.shape, t.shape, x.dtype))
    return BalanceLoss(*map(c.give, r)), c.give(grad)
