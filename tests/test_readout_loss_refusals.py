"""Refusals of the read-out's cross-entropy and of the tensor-list operators: every call here is turned down before any
kernel is launched (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

from gncde import _lib, autograd, engine

LIB = _lib.load()
E_ARG, E_SHAPE, E_UNSUPPORTED, E_WORKSPACE = 1, 2, 3, 4
P = 0x10000  # an aligned address that is never read


def _xent(grad=False, rows=4, hidden=8, classes=5, dtype=_lib.DTYPE_FP32, x=P, W=P, b=None, kind=_lib.TARGET_INDEX64,
          target=P, mask=None, loss=P, stats=P, ws=P, ws_bytes=1 << 40):
    if grad:
        return LIB.gncde_linear_cross_entropy_grad(rows, hidden, classes, dtype, x, W, b, kind, target, mask, stats, loss,
                                                   None, None, None, ws, ws_bytes, None)
    return LIB.gncde_linear_cross_entropy(rows, hidden, classes, dtype, x, W, b, kind, target, mask, loss, stats, ws,
                                          ws_bytes, None)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("change,code", [
    (dict(rows=-1), E_SHAPE),
    (dict(hidden=0), E_SHAPE),
    (dict(classes=0), E_SHAPE),
    (dict(kind=3), E_ARG),
    (dict(kind=-1), E_ARG),
    (dict(dtype=_lib.DTYPE_FP16), E_UNSUPPORTED),
    (dict(dtype=7), E_UNSUPPORTED),
    (dict(rows=1 << 25), E_UNSUPPORTED),
    (dict(hidden=1 << 17), E_UNSUPPORTED),
    (dict(classes=1 << 27), E_UNSUPPORTED),
    (dict(x=None), E_ARG),
    (dict(W=None), E_ARG),
    (dict(target=None), E_ARG),
    (dict(x=P + 2), E_ARG),
    (dict(W=P + 1), E_ARG),
    (dict(b=P + 2), E_ARG),
    (dict(target=P + 4), E_ARG),
    (dict(ws=None), E_WORKSPACE),
    (dict(ws=P + 16), E_WORKSPACE),
    (dict(ws_bytes=64), E_WORKSPACE),
    (dict(loss=None), E_ARG),
    (dict(stats=None), E_ARG),
])
def test_entry_point_refuses(grad, change, code):
    assert _xent(grad=grad, **change) == code


def test_no_rows_is_nothing_to_do():
    assert _xent(rows=0, x=None, target=None, ws=None, ws_bytes=0) == 0


def test_workspace_is_sized_for_what_is_accepted():
    f = LIB.gncde_linear_cross_entropy_workspace_bytes
    for dtype in (_lib.DTYPE_FP32, _lib.DTYPE_BF16):
        for grad in (0, 1):
            assert f(1, 1, 1, dtype, grad) > 0
            # a piece of the classes at a time: the workspace of a long batch does not grow with the vocabulary (the
            # size of a piece goes by how its products fill the GPU, the loss keeps a pair for 128 classes of a row)
            a, b = f(8192, 4096, 1 << 17, dtype, grad), f(8192, 4096, 1 << 20, dtype, grad)
            assert a < 4 << 30 and b < 1.5 * a + (8192 << 20) / 8 * (not grad)
    assert f(1, 1, 1, _lib.DTYPE_FP16, 0) == 0
    assert f(-1, 1, 1, 0, 0) == 0 and f(1, 0, 1, 0, 0) == 0 and f(1, 1, 0, 0, 0) == 0


def _case(rows=3, hidden=4, classes=5, dtype=torch.float32):
    return dict(x=torch.zeros(rows, hidden, dtype=dtype), W=torch.zeros(classes, hidden, dtype=dtype),
                b=torch.zeros(classes, dtype=dtype), target=torch.zeros(rows, dtype=torch.int64),
                mask=torch.ones(rows, dtype=torch.bool))


@pytest.mark.parametrize("change,words", [
    (dict(x=torch.zeros(3, 4, dtype=torch.float16)), "fp32 or all be bf16"),
    (dict(x=torch.zeros(3, 4, dtype=torch.bfloat16)), "fp32 or all be bf16"),
    (dict(b=torch.zeros(5, dtype=torch.bfloat16)), "fp32 or all be bf16"),
    (dict(W=torch.zeros(5, 6)), "does not fit"),
    (dict(W=torch.zeros(0, 4)), "does not fit"),
    (dict(W=torch.zeros(4)), "does not fit"),
    (dict(b=torch.zeros(6)), "must be"),
    (dict(target=torch.zeros(4, dtype=torch.int64)), "must be"),
    (dict(target=torch.zeros(3, 4)), "must be"),
    (dict(target=torch.zeros(3, 5, dtype=torch.float64)), "class indices or fp32"),
    (dict(target=torch.zeros(3, dtype=torch.int16)), "class indices or fp32"),
    (dict(mask=torch.ones(3)), "mask must be bool"),
    (dict(mask=torch.ones(2, dtype=torch.bool)), "mask must be bool"),
    (dict(), "one CUDA device"),
])
def test_python_refuses(change, words):
    c = {**_case(), **change}
    with pytest.raises(_lib.GncdeError, match=words):
        engine.linear_cross_entropy(c["x"], c["W"], c["b"], c["target"], c["mask"])


def test_labels_take_no_gradient():
    c = _case()
    y = torch.zeros(3, 5, requires_grad=True)
    with pytest.raises(_lib.GncdeError, match="no gradient with respect to the labels"):
        autograd.linear_cross_entropy(c["x"], c["W"], c["b"], y)


# ---- tensor lists -----------------------------------------------------------------------------------------------
def _list(*entries):
    arr = (_lib.GncdeTensor * max(len(entries), 1))()
    for a, (i, o, n, d) in zip(arr, entries):
        a.inp, a.out, a.numel, a.dtype = i, o, n, d
    return arr


@pytest.mark.parametrize("entry,code", [
    ((P, P, -1, 0), E_SHAPE),
    ((P, P, 1 << 60, 0), E_SHAPE),
    ((P, P, 4, 3), E_UNSUPPORTED),
    ((None, P, 4, 0), E_ARG),
    ((P, None, 4, 0), E_ARG),
    ((P + 2, P, 4, 0), E_ARG),
    ((P, P + 1, 4, 1), E_ARG),
])
def test_list_refuses(entry, code):
    arr = _list((P, P, 4, 0), entry)
    assert LIB.gncde_clip_by_global_norm(2, arr, 1.0, P, P, 1 << 30, None) == code


@pytest.mark.parametrize("max_norm", [0.0, -1.0, float("inf"), float("nan")])
def test_max_norm_must_be_positive_and_finite(max_norm):
    assert LIB.gncde_clip_by_global_norm(1, _list((P, P, 4, 0)), max_norm, P, P, 1 << 30, None) == E_ARG
    with pytest.raises((_lib.GncdeError, RuntimeError), match="max_norm|HIP"):
        engine.clip_by_global_norm([torch.zeros(3)], max_norm)


def test_list_refuses_workspace_and_stats():
    arr = _list((P, None, 4, 0))
    need = LIB.gncde_global_norm_workspace_bytes(1)
    assert need > 0 and LIB.gncde_global_norm_workspace_bytes(-1) == 0
    assert LIB.gncde_global_norm(1, arr, P, P, need - 1, None) == E_WORKSPACE
    assert LIB.gncde_global_norm(1, arr, P, None, need, None) == E_WORKSPACE
    assert LIB.gncde_global_norm(1, arr, None, P, need, None) == E_ARG
    assert LIB.gncde_global_norm(1, None, P, P, need, None) == E_ARG
    assert LIB.gncde_global_norm(-1, arr, P, P, need, None) == E_ARG


@pytest.mark.parametrize("tensors,words", [
    (torch.zeros(3), "a list of tensors"),
    ([], "empty list"),
    ([torch.zeros(3, dtype=torch.float64)], "fp32, bf16 or fp16"),
    ([torch.zeros(3)], "one CUDA device"),
])
def test_python_list_refuses(tensors, words):
    with pytest.raises(_lib.GncdeError, match=words):
        engine._tensor_table("global_norm", tensors)


def _rows(*entries):
    return np.array([[i, o, n, 0] for i, o, n in entries], dtype=np.int64)


@pytest.mark.parametrize("entries,bad", [
    ([(0, 1000, 10), (100, 2000, 10)], False),
    ([(1000, 1000, 10), (2000, 2000, 10)], False),                       # in place
    ([(1000, 1000, 10), (1040, 1040, 10)], False),                       # in place, back to back
    ([(1000, 1000, 10), (1000, 1000, 10)], True),                        # the same tensor twice
    ([(1000, 1000, 10), (1020, 1020, 10)], True),
    ([(0, 1000, 10), (100, 1036, 10)], True),                            # outputs meet
    ([(0, 1000, 10), (1036, 2000, 10)], True),                           # an output meets another's tensor
    ([(1004, 1000, 10)], True),                                          # an output meets its own tensor, shifted
    ([(1000, 1000, 10), (1010, 3000, 2)], True),                         # in place over a tensor read elsewhere
    ([(0, 1000, 0), (100, 1000, 10)], False),                            # nothing in an empty one
])
def test_overlap(entries, bad):
    rows, sizes = _rows(*entries), [4] * len(entries)
    if bad:
        with pytest.raises(_lib.GncdeError, match="share"):
            engine._refuse_overlap("clip", rows, sizes)
    else:
        engine._refuse_overlap("clip", rows, sizes)


def test_list_struct_matches_c(tmp_path):
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gncde.h")
    src = tmp_path / "t.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{header}"\nint main(void) {{ printf("%zu %zu %zu '
                   '%zu", sizeof(GncdeTensor), offsetof(GncdeTensor, out), offsetof(GncdeTensor, numel), '
                   'offsetof(GncdeTensor, dtype)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", str(src), "-o", str(tmp_path / "t")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "t")], capture_output=True, text=True).stdout.split()))
    T = _lib.GncdeTensor
    assert got == [ctypes.sizeof(T), T.out.offset, T.numel.offset, T.dtype.offset]
