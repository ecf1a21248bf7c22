"""Rows of a table by ids, and the table's gradient: what goes into a model beside a search, the rows of a vocabulary's tokens or
of a search's neighbors.

    x = octex.embed(table, tokens, scale=dim**0.5)                      # a row a token
    rows = octex.embed(codes, neighbors, row_scales=scales)             # of quantize_rows' codes; a search's -1 gives 0
    grad = octex.embed_backward(grad_x, tokens, len(table), scale=dim**0.5)

Operands, streams, results and errors are as octex_amd/scores.py has them.
"""

from . import scores
from .scores import FLOATS, INTS


def _flat_ids(c, ids):
    """Ids of any shape as a vector, that as a matrix of one column, and their shape."""
    t = c.array(ids)
    shape = t.shape
    if t.ndim != 1:
        with c.context():
            t = t.reshape(-1)
    t = c.take(t, "ids", INTS, 1)
    return t, _rows(c, t, t.shape[0], 1), shape


def _rows(c, t, rows, cols):
    """A dense tensor as a matrix of `rows` rows."""
    return scores._Matrix(t.data_ptr(), scores._TYPES[c.names[t.dtype]], rows, cols, cols)


def embed(table, ids, *, row_scales=None, scale=1.0, dtype=None):
    """scale * table[ids], [..., d] of ids of any shape: rows of a table [n, d] of floats, or of int8 with their row_scales [n]
    (quantize_rows').

    Ids outside [0, n), as a search's -1, give rows of 0.  `dtype` ("float32", "float16" or "bfloat16") is that of the result:
    the table's own if it holds floats, else float32.  The products are float32, rounded once more to the result.
    """
    coded = row_scales is not None
    c = scores._Call(table, "table", ("int8",) if coded else FLOATS + ("int8",))
    x = c.first
    if not coded and c.names[x.dtype] == "int8":
        raise TypeError("octex: an int8 table needs its row_scales")
    n, d = x.shape
    t, flat, shape = _flat_ids(c, ids)
    if coded:
        row_scales = c.dense(row_scales, "row_scales", (n,))
    if dtype is None:
        dtype = "float32" if coded else c.names[x.dtype]
    out = c.new((*shape, d), dtype=scores._float_type(c, dtype, "rows", "table"))
    c.run("octexEmbed", c.matrix(x), row_scales.data_ptr() if coded else None, flat, float(scale),
          _rows(c, out, t.shape[0], d))
    return c.give(out)


def embed_backward(grad, ids, rows=None, *, scale=1.0, dtype=None, add_to=None):
    """The gradient [rows, d] of a table of `rows` rows, given that of embed's result, grad [..., d], and its ids [...]: row v is
    scale times the sum of grad over the places where ids is v.

    Sums are float32, in an order that the ids and sizes alone determine, and rounded once to `dtype` (grad's own type).  Ids
    outside [0, rows) are left out.  With `add_to`, a torch matrix [rows, d] of floats on grad's GPU that shares no memory with
    grad, the gradient is added to it in place, and it is returned; rows without an id are not touched.
    """
    c = scores._Call(grad, "grad", FLOATS, flat=True)
    g = c.first
    t, flat, shape = _flat_ids(c, ids)
    m, d = g.shape
    if c.lead != shape:
        raise ValueError(f"octex: grad has shape {(*c.lead, d)}, ids {tuple(shape)}")
    if add_to is None:
        if rows is None:
            raise TypeError("octex: the table's number of rows, or add_to, must be given")
        rows = int(rows)
        if rows < 0:
            raise ValueError(f"octex: a table of {rows} rows")
        out = c.new((rows, d), dtype=scores._float_type(c, c.names[g.dtype] if dtype is None else dtype, "gradients", "grad"))
        c.run_sized("octexEmbedBackward", c.matrix(g), flat, float(scale), 0, _rows(c, out, rows, d),
                    sizes=("octexEmbedBackward", m, rows, d, 0))
        return c.give(out)
    out = add_to
    if not isinstance(out, c.torch.Tensor) or out.device != c.device or c.on_host:
        raise ValueError("octex: add_to must be a torch matrix on grad's GPU")
    if dtype is not None:
        raise ValueError("octex: the gradient has add_to's type")
    if c.names.get(out.dtype) not in FLOATS or out.ndim != 2 or out.shape[1] != d or rows not in (None, out.shape[0]):
        raise ValueError(f"octex: add_to is {tuple(out.shape)} of {out.dtype}, expected a matrix [{'rows' if rows is None else rows}"
                         f", {d}] of {', '.join(FLOATS)}")
    if out.is_neg() or (d > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < d):
        raise ValueError("octex: add_to's rows must lie apart, their values side by side")
    c.array(out)  # ordered with the call
    c.run_sized("octexEmbedBackward", c.matrix(g), flat, float(scale), 1, c.matrix(out),
                sizes=("octexEmbedBackward", m, out.shape[0], d, 1))
    c.torch.autograd.graph.increment_version(out)
    return out
