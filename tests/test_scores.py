"""The C entries of the operators on rows of scores without a GPU: arguments are refused by their shapes, types and memory
before anything is launched, and the workspace's size is answered."""

import ctypes as ct

import numpy as np
import pytest

from octex_amd import _lib
from octex_amd import scores as S

FLOAT32, FLOAT16, INT8, INT32, INT64 = 0, 1, 3, 4, 5


def matrix(a, kind, rows=None, cols=None, stride=None):
    return S._Matrix(a.ctypes.data, kind, a.shape[0] if rows is None else rows, a.shape[1] if cols is None else cols,
                     a.shape[1] if stride is None else stride)


def refused(name, *args):
    assert getattr(_lib.lib(), name)(*args) == _lib.CUVS_ERROR
    return _lib.lib().cuvsGetLastErrorText().decode()


@pytest.fixture()
def host():
    x = np.zeros((3, 40), np.float32)
    return dict(x=x, ids=np.zeros((3, 2), np.int64), t=np.zeros((3, 2), np.float32), v=np.zeros(3, np.float32),
                codes=np.zeros((3, 40), np.int8))


def entry(name):
    S._entry(name)
    return name


def log_probs(h, x=None, ids=None, T=1.0, top=0, size=None):
    x = matrix(h["x"], FLOAT32) if x is None else x
    ids = matrix(h["ids"], INT64) if ids is None else ids
    v = h["v"].ctypes.data
    return (entry("octexLogProbs"), x, ids, T, top, v, v, v, v, v, None, 0, size, None)


def test_host_memory_is_refused(host):
    assert "must lie in GPU memory" in refused(*log_probs(host))


@pytest.mark.parametrize("change,text", [
    (dict(T=0.0), "temperature"), (dict(T=float("nan")), "temperature"), (dict(T=float("inf")), "temperature"),
    (dict(top=65), "top"), (dict(top=-1), "top"),
    (dict(x=dict(kind=INT8)), "float32, float16 or bfloat16"), (dict(x=dict(kind=9)), "float32, float16 or bfloat16"),
    (dict(x=dict(cols=0)), "columns"), (dict(x=dict(cols=(1 << 30) + 1, stride=1 << 31)), "columns"),
    (dict(x=dict(rows=-1)), "negative"), (dict(x=dict(stride=39)), "overlap"),
    (dict(ids=dict(rows=2)), "ids is"), (dict(ids=dict(kind=FLOAT32)), "int32 or int64"),
    (dict(ids=dict(cols=513, stride=513)), "512"),
])
def test_log_probs_refusals(host, change, text):
    args = {k: v for k, v in change.items() if k in ("T", "top")}
    for name, kind in (("x", FLOAT32), ("ids", INT64)):
        if name in change:
            args[name] = matrix(host[name], **dict(dict(kind=kind), **change[name]))
    assert text in refused(*log_probs(host, **args))


def test_null_matrices_are_refused(host):
    for at in (1, 2):
        args = list(log_probs(host))
        args[at] = None
        assert "NULL" in refused(*args)


def test_sizes_are_answered(host):
    size = ct.c_int64(-1)
    at = ct.addressof(size)
    f = S._entry("octexLogProbs")
    assert f(*log_probs(host, size=at)[1:]) == _lib.CUVS_SUCCESS and size.value >= 0
    f = S._entry("octexInt8Scores")
    many = np.zeros((300, 40), np.float32)
    x, codes, out = matrix(many, FLOAT32), matrix(host["codes"], INT8), matrix(np.zeros((300, 3), np.float32), FLOAT32)
    v = host["v"].ctypes.data
    assert f(x, None, codes, v, None, out, None, 0, at, None) == _lib.CUVS_SUCCESS
    need = size.value
    assert need >= 300 * 40 + 300 * 4  # the quantized queries and their scales
    own = matrix(np.zeros((300, 40), np.int8), INT8)
    assert f(own, v, codes, v, None, out, None, 0, at, None) == _lib.CUVS_SUCCESS and size.value >= 0
    assert "workspace" in refused("octexInt8Scores", x, None, codes, v, None, out, v, need - 1, None, None)


def test_int8_scores_refusals(host):
    entry("octexInt8Scores")
    x, codes, out = matrix(host["x"], FLOAT32), matrix(host["codes"], INT8), matrix(np.zeros((3, 3), np.float32), FLOAT32)
    v = host["v"].ctypes.data

    def call(q=x, qs=None, r=codes, o=out):
        return refused("octexInt8Scores", q, qs, r, v, None, o, v, 1 << 30, None, None)

    assert "int8, float32" in call(q=matrix(host["x"], INT32))
    assert "query_scales" in call(qs=v)
    assert "rows is" in call(r=matrix(host["codes"], INT8, cols=39))
    assert "rows must be int8" in call(r=x)
    assert "out is" in call(o=matrix(np.zeros((3, 4), np.float32), FLOAT32))
    assert "out must be" in call(o=matrix(np.zeros((3, 3), np.int8), INT8))
    wide = dict(rows=1, cols=131072, stride=131072)
    assert "131071" in call(q=matrix(host["x"], FLOAT32, **wide), r=matrix(host["codes"], INT8, **wide))
    assert "must lie in GPU memory" in call()


def test_gradient_refusals(host):
    x, ids, t = matrix(host["x"], FLOAT32), matrix(host["ids"], INT64), matrix(host["t"], FLOAT32)
    v = host["v"].ctypes.data
    entry("octexLogProbsBackward"), entry("octexDistillBackward"), entry("octexDistillStep"), entry("octexDistill")
    half, short = matrix(host["x"], FLOAT16), matrix(host["x"], FLOAT32, cols=39)
    for grad, text in ((half, "type of the logits"), (short, "grad is"), (None, "grad is NULL")):
        assert text in refused("octexLogProbsBackward", x, ids, 1.0, v, v, v, v, grad, None)
        assert text in refused("octexDistillBackward", x, ids, t, 1.0, v, v, grad, None)
        assert text in refused("octexDistillStep", x, ids, t, 1.0, v, v, v, grad, None, 0, None, None)
    assert "teacher is" in refused("octexDistill", x, ids, matrix(host["t"], FLOAT32, cols=1), 1.0, v, v, None, 0, None, None)
    assert "teacher must" in refused("octexDistill", x, ids, matrix(host["ids"], INT64), 1.0, v, v, None, 0, None, None)
    assert "GPU memory" in refused("octexDistillStep", x, ids, t, 1.0, v, v, v, x, None, 0, None, None)


def test_no_rows_are_no_work():
    none = S._Matrix(None, FLOAT32, 0, 40, 40)
    ids = S._Matrix(None, INT64, 0, 2, 2)
    f = S._entry("octexDistillStep")
    assert f(none, ids, S._Matrix(None, FLOAT32, 0, 2, 2), 1.0, None, None, None, none, None, 0, None, None) == _lib.CUVS_SUCCESS
