"""The C entries of the operators at both ends of a training step without a GPU: arguments are refused by their shapes, types,
values and memory before anything is launched, and the workspace's size is answered."""

import ctypes as ct
import os
import subprocess

import numpy as np
import pytest
from conftest import ROOT

from octex_amd import _lib
from octex_amd import scores as S

FLOAT32, FLOAT16, INT8, INT32, INT64 = 0, 1, 3, 4, 5
HOST = np.zeros(4096, np.float32).ctypes.data


def matrix(rows, cols, kind=FLOAT32, stride=None, data=HOST):
    return S._Matrix(data, kind, rows, cols, cols if stride is None else stride)


def refused(name, *args):
    assert S._entry(name)(*args, None) == _lib.CUVS_ERROR
    return _lib.lib().cuvsGetLastErrorText().decode()


def accepted(name, *args):
    assert S._entry(name)(*args, None) == _lib.CUVS_SUCCESS, _lib.lib().cuvsGetLastErrorText().decode()


def policy(x=None, ids=None, T=1.0, ref=None, low=0.8, high=1.2, kl=0.0, entropy=0.0):
    return (matrix(3, 40) if x is None else x, matrix(3, 1, INT64) if ids is None else ids, T, HOST, HOST, ref, low, high, kl,
            entropy)


@pytest.mark.parametrize("change,text", [
    (dict(x=matrix(3, 40, INT8)), "float32, float16 or bfloat16"), (dict(x=matrix(3, 0)), "columns"),
    (dict(x=matrix(3, 40, stride=39)), "overlap"), (dict(x=matrix(-1, 40)), "negative"),
    (dict(ids=matrix(3, 2, INT64)), "ids is"), (dict(ids=matrix(2, 1, INT64)), "ids is"), (dict(ids=matrix(3, 1)), "int32 or int64"),
    (dict(T=0.0), "temperature"), (dict(T=float("nan")), "temperature"), (dict(low=-0.1), "bounds"), (dict(low=1.1), "bounds"),
    (dict(high=0.9), "bounds"), (dict(high=float("nan")), "bounds"), (dict(kl=0.1), "ref_log_probs"),
    (dict(kl=float("inf"), ref=HOST), "finite"), (dict(entropy=float("nan")), "finite"), (dict(), "must lie in GPU memory"),
])
def test_policy_refusals(change, text):
    args, out, grad = policy(**change), [HOST] * 4, matrix(3, 40)
    if "x" in change:
        grad = change["x"]
    assert text in refused("octexPolicyLoss", *args, *out, None, 0, None)
    assert text in refused("octexPolicyLossBackward", *args, HOST, HOST, HOST, HOST, grad)
    assert text in refused("octexPolicyLossStep", *args, HOST, *out, grad, None, 0, None)


def test_policy_gradients_and_null_operands():
    for grad, text in ((matrix(3, 40, FLOAT16), "type of the logits"), (matrix(3, 39), "grad is"), (None, "grad is NULL")):
        assert text in refused("octexPolicyLossBackward", *policy(), HOST, HOST, HOST, HOST, grad)
        assert text in refused("octexPolicyLossStep", *policy(), HOST, *[HOST] * 4, grad, None, 0, None)
    assert "logits is NULL" in refused("octexPolicyLoss", None, *policy()[1:], *[HOST] * 4, None, 0, None)
    assert "ids is NULL" in refused("octexPolicyLoss", policy()[0], None, *policy()[2:], *[HOST] * 4, None, 0, None)


def test_policy_sizes():
    size = ct.c_int64(-1)
    at = ct.addressof(size)
    accepted("octexPolicyLoss", *policy(), *[None] * 4, None, 0, at)
    assert size.value == 0
    wide = policy(x=matrix(3, 200_000))
    accepted("octexPolicyLoss", *wide, *[None] * 4, None, 0, at)
    need = size.value
    assert need > 0 and "workspace has" in refused("octexPolicyLoss", *wide, *[HOST] * 4, HOST, need - 1, None)
    none = (matrix(0, 40, data=None), matrix(0, 1, INT64, data=None), 1.0, None, None, None, 0.8, 1.2, 0.0, 0.0)
    accepted("octexPolicyLossStep", *none, None, *[None] * 4, matrix(0, 40, data=None), None, 0, None)


@pytest.mark.parametrize("x,experts,weights,text", [
    (matrix(3, 8), matrix(3, 2, INT64), (1.0, 0.0), "must lie in GPU memory"), (matrix(3, 8), matrix(2, 2, INT64), (1.0, 0.0), "experts is"),
    (matrix(3, 8), matrix(3, 2), (1.0, 0.0), "experts must be"), (matrix(3, 2049), matrix(3, 2, INT64), (1.0, 0.0), "2048"),
    (matrix(3, 0), matrix(3, 2, INT64), (1.0, 0.0), "columns"), (matrix(3, 8), matrix(3, 513, INT32), (1.0, 0.0), "512"),
    (matrix(3, 8, INT64), matrix(3, 2, INT64), (1.0, 0.0), "float32, float16"), (None, matrix(3, 2, INT64), (1.0, 0.0), "logits is NULL"),
    (matrix(3, 8), None, (1.0, 0.0), "experts is NULL"), (matrix(3, 8), matrix(3, 2, INT64), (float("nan"), 0.0), "finite"),
    (matrix(3, 8), matrix(3, 2, INT64), (1.0, float("inf")), "finite"),
    (matrix(1 << 30, 8), matrix(1 << 30, 2, INT64), (1.0, 0.0), "choices"),
])
def test_balance_refusals(x, experts, weights, text):
    assert text in refused("octexBalanceLoss", x, experts, *weights, *[HOST] * 5, None, None, None, 0, None)
    assert text in refused("octexBalanceLoss", x, experts, *weights, *[HOST] * 5, HOST, x, None, 0, None)
    assert text in refused("octexBalanceLossBackward", x, experts, *weights, HOST, HOST, None, x)


def test_balance_gradients_and_sizes():
    x, experts = matrix(3, 8), matrix(3, 2, INT64)
    for grad, text in ((matrix(3, 8, FLOAT16), "type of the logits"), (matrix(3, 9), "grad is")):
        assert text in refused("octexBalanceLoss", x, experts, 1.0, 0.0, *[HOST] * 5, None, grad, None, 0, None)
        assert text in refused("octexBalanceLossBackward", x, experts, 1.0, 0.0, HOST, HOST, None, grad)
    assert "grad is NULL" in refused("octexBalanceLossBackward", x, experts, 1.0, 0.0, HOST, HOST, None, None)
    size = ct.c_int64(-1)
    at = ct.addressof(size)
    many, chosen = matrix(100_000, 64), matrix(100_000, 2, INT64)
    accepted("octexBalanceLoss", many, chosen, 1.0, 0.0, *[None] * 5, None, None, None, 0, at)
    need = size.value
    assert need > 0
    assert "workspace has" in refused("octexBalanceLoss", many, chosen, 1.0, 0.0, *[HOST] * 5, None, None, HOST, need - 1, None)
    none = matrix(0, 8, data=None), matrix(0, 2, INT64, data=None)
    accepted("octexBalanceLossBackward", *none, 1.0, 0.0, None, None, None, none[0])


@pytest.mark.parametrize("table,scales,ids,out,text", [
    (matrix(9, 16), None, matrix(4, 1, INT64), matrix(4, 16), "must lie in GPU memory"),
    (matrix(9, 16, INT64), None, matrix(4, 1, INT64), matrix(4, 16), "the table must be"),
    (matrix(9, 16), HOST, matrix(4, 1, INT64), matrix(4, 16), "only int8"),
    (matrix(9, 16), None, matrix(4, 2, INT64), matrix(4, 16), "ids is"), (matrix(9, 16), None, matrix(4, 1), matrix(4, 16), "int32 or int64"),
    (matrix(9, 16), None, matrix(4, 1, INT64), matrix(3, 16), "out is"), (matrix(9, 16), None, matrix(4, 1, INT64), matrix(4, 15), "out is"),
    (matrix(9, 16), None, matrix(4, 1, INT64), matrix(4, 16, INT8), "out must be"), (None, None, matrix(4, 1, INT64), matrix(4, 16), "table is NULL"),
    (matrix(1 << 31, 16), None, matrix(4, 1, INT64), matrix(4, 16), "2^31"),
    (matrix(9, 16), None, matrix(1 << 31, 1, INT64), matrix(1 << 31, 16), "2^31"),
    (matrix(9, (1 << 24) + 1), None, matrix(4, 1, INT64), matrix(4, (1 << 24) + 1), "at most 16777216"),
])
def test_embed_refusals(table, scales, ids, out, text):
    assert text in refused("octexEmbed", table, scales, ids, 1.0, out)


@pytest.mark.parametrize("grad,ids,out,text", [
    (matrix(4, 16), matrix(4, 1, INT64), matrix(9, 16), "must lie in GPU memory"), (matrix(4, 16, INT8), matrix(4, 1, INT64), matrix(9, 16), "grad must be"),
    (matrix(4, 16), matrix(3, 1, INT64), matrix(9, 16), "ids is"), (matrix(4, 16), matrix(4, 1), matrix(9, 16), "int32 or int64"),
    (matrix(4, 16), matrix(4, 1, INT64), matrix(9, 15), "out is"), (matrix(4, 16), matrix(4, 1, INT64), matrix(9, 16, INT32), "out must be"),
    (matrix(4, 16), matrix(4, 1, INT64), matrix(1 << 31, 16), "2^31"), (matrix(4, 16), matrix(4, 1, INT64), None, "out is NULL"),
])
def test_embed_backward_refusals(grad, ids, out, text):
    for add in (0, 1):
        assert text in refused("octexEmbedBackward", grad, ids, 1.0, add, out, HOST, 1 << 40, None)


def test_embed_sizes_and_no_work():
    size = ct.c_int64(-1)
    at = ct.addressof(size)
    args = matrix(5000, 16), matrix(5000, 1, INT64), 1.0, 0, matrix(9, 16)
    accepted("octexEmbedBackward", *args, None, 0, at)
    need = size.value
    assert need >= 2 * 5000 * 8 and "workspace has" in refused("octexEmbedBackward", *args, HOST, need - 1, None)
    none = matrix(0, 16, data=None), matrix(0, 1, INT64, data=None)
    accepted("octexEmbed", matrix(9, 16), None, none[1], 1.0, none[0])
    accepted("octexEmbedBackward", *none, 1.0, 1, matrix(9, 16), None, 0, None)
    accepted("octexEmbedBackward", *none, 1.0, 0, none[0], None, 0, None)


def test_a_workspace_is_asked_for_once_for_its_sizes(monkeypatch):
    import torch

    asked, ran = [], []

    def entry(name):
        def call(rows, workspace, size, at, stream):
            if at is None:
                ran.append((rows, size, workspace is not None))
            else:
                asked.append(rows)
                ct.c_int64.from_address(at).value = 100 * rows
            return _lib.CUVS_SUCCESS

        return call

    monkeypatch.setattr(S, "_entry", entry)
    monkeypatch.setattr(S, "_WORKSPACES", {})
    c = S._Call.__new__(S._Call)
    c.torch, c.device, c.stream, c.side, c.others = torch, torch.device("cpu"), None, None, ()
    for rows in (3, 3, 0, 4, 3, 0):
        c.run_sized("any", rows, sizes=("any", rows))
    assert asked == [3, 0, 4]
    assert ran == [(3, 300, True), (3, 300, True), (0, 0, False), (4, 400, True), (3, 300, True), (0, 0, False)]
    c.run_sized("any", 5), c.run_sized("any", 5)
    assert asked == [3, 0, 4, 5, 5]
    S._WORKSPACES.update((("full", i), 0) for i in range(4096))  # as many as are kept
    c.run_sized("any", 6, sizes=("any", 6))
    assert S._WORKSPACES == {("any", 6): 600}


def test_balance_of_more_choices_than_64_bits_count():
    """A product of rows and choices that passes 64 bits is refused like any that passes 31."""
    size = ct.c_int64(-1)
    for rows, k in ((1 << 62, 4), (1 << 55, 512), (1 << 31, 1), (1 << 32, 0)):
        x, experts = matrix(rows, 8), matrix(rows, k, INT64)
        assert "choices" in refused("octexBalanceLoss", x, experts, 1.0, 0.0, *[HOST] * 5, None, None, None, 0, ct.addressof(size))
        assert "choices" in refused("octexBalanceLossBackward", x, experts, 1.0, 0.0, HOST, HOST, None, x)
    assert size.value == -1


def test_tables_of_any_size_are_cleared_in_one_launch(tmp_path):
    """A table as large as the GPU's memory, of rows of just over 16 KB, has more of them than a launch has workgroups."""
    exe = str(tmp_path / "table_clears")
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(rocm, "include"),
                    os.path.join(ROOT, "tests", "c", "table_clears.cpp"), "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout
