"""CPU: argument checks of the linear and grouped entry points, before any CUDA call."""
from __future__ import annotations

import ctypes

import pytest
import torch

import arc
from arc import _lib

BAD, UNS = _lib.ARC_ERR_INVALID_ARGUMENT, _lib.ARC_ERR_UNSUPPORTED


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.cast(buf, ctypes.c_void_p).value + 63) // 64 * 64


def test_linear_checks(native_lib, p):
    f = native_lib.arc_linear_bf16

    def call(x=p, w=p, bias=None, res=None, out=p, z=None, m=4, n=8, k=16, ldx=16, ldw=16, ldr=8, ldo=8, ldz=8, act=0):
        return f(x, w, bias, res, out, z, m, n, k, ldx, ldw, ldr, ldo, ldz, act, None)

    assert call(x=None) == BAD and call(out=None) == BAD
    assert call(m=0) == BAD and call(n=-1) == BAD and call(k=0) == BAD
    assert call(act=5) == BAD and call(act=-1) == BAD
    assert call(ldx=8) == BAD and call(ldw=8) == BAD and call(ldo=7) == BAD
    assert call(res=p, ldr=7) == BAD and call(z=p, ldz=7) == BAD
    assert call(k=12, ldx=12, ldw=16) == UNS and call(x=p + 8) == UNS and call(w=p + 2) == UNS
    assert call(bias=p + 1) == UNS and call(out=p + 1) == UNS


def test_linear_backward_checks(native_lib, p):
    f = native_lib.arc_linear_backward
    size = ctypes.c_size_t(0)
    query = native_lib.arc_linear_backward_workspace_bytes
    assert query(0, 8, 1, 1, ctypes.byref(size)) == BAD
    assert query(64, 9, 1, 0, ctypes.byref(size)) == 0 and size.value >= 64 * 16 * 2
    assert query(64, 9, 0, 0, ctypes.byref(size)) == 0 and size.value == 0
    assert query(64, 9, 0, 1, ctypes.byref(size)) == 0 and size.value >= 9 * 4

    def call(dy=p, x=p, w=p, z=p, dx=p, dw=p, db=p, ws=p, wsb=4096, m=4, n=8, k=16, lddy=8, ldx=16, ldw=16, ldz=8,
             lddx=16, lddw=16, act=2):
        return f(dy, x, w, z, dx, dw, db, ws, wsb, m, n, k, lddy, ldx, ldw, ldz, lddx, lddw, act, None)

    assert call(dy=None) == BAD and call(dx=None, dw=None, db=None) == BAD
    assert call(x=None) == BAD and call(w=None) == BAD and call(z=None) == BAD
    assert call(m=0) == BAD and call(k=0) == BAD and call(act=9) == BAD
    assert call(lddy=7) == BAD and call(ldz=7) == BAD and call(lddx=15) == BAD and call(lddw=15) == BAD
    assert call(ldx=20) == UNS and call(w=p + 2) == UNS
    assert call(ws=None) == BAD and call(wsb=4) == BAD and call(ws=p + 2) == BAD
    assert call(db=p + 1) == UNS


def test_grouped_checks(native_lib, p):
    for name in ("arc_grouped_matmul", "arc_grouped_matmul_dx", "arc_grouped_matmul_dw"):
        f = getattr(native_lib, name)
        dw = name.endswith("dw")

        def call(a=p, b=p, off=p, c=p, t=4, e=2, n=8, k=16, lda=16, ldb=16, ldc=16, stride=128, flags=0):
            return f(a, b, off, c, t, e, n, k, lda, ldb, *((ldc, stride) if dw else (stride, ldc, flags)), None)

        assert call(a=None) == BAD and call(b=None) == BAD and call(c=None) == BAD
        assert call(t=0) == BAD and call(e=0) == BAD and call(n=0) == BAD and call(k=0) == BAD
        assert call(off=None) == BAD  # two groups
        assert call(off=p + 2) == UNS and call(e=1025, stride=1 << 20) == UNS
        assert call(a=p + 2) == UNS and call(b=p + 4) == UNS and call(c=p + 1) == UNS
        assert call(lda=4) == BAD and call(ldb=8, k=16) == BAD and call(stride=64) == BAD
        if not dw:
            assert call(flags=8) == BAD and call(stride=132) == UNS


def test_a8w4_grouped_checks(native_lib, p):
    f = native_lib.arc_a8w4_grouped_gemm

    size = ctypes.c_size_t(0)
    query = native_lib.arc_a8w4_grouped_workspace_bytes
    assert query(4, 0, 128, ctypes.byref(size)) == BAD
    assert query(64, 2, 128, ctypes.byref(size)) == 0 and size.value == 0
    assert query(640, 2, 128, ctypes.byref(size)) == 0 and size.value == 640 * 128 * 2

    def call(a=p, sa=p, wp=p, sb=p, off=p, c=p, t=4, e=2, n=8, k=128, group=128, flags=0):
        return f(a, sa, wp, sb, off, c, None, 0, t, e, n, k, group, flags, None)

    for name in ("a", "sa", "wp", "sb", "off", "c"):
        assert call(**{name: None}) == BAD
    assert call(t=0) == BAD and call(flags=2) == BAD
    assert call(k=64) == UNS and call(n=12) == UNS and call(group=64) == UNS
    assert call(a=p + 8) == UNS and call(wp=p + 8) == UNS and call(c=p + 8) == UNS and call(sa=p + 2) == UNS
    assert call(e=1000, n=1 << 22) == UNS


def test_group_rows_checks(native_lib, p):
    f = native_lib.arc_group_rows
    size = ctypes.c_size_t(0)
    assert native_lib.arc_group_rows_workspace_bytes(16, 1025, ctypes.byref(size)) == BAD
    assert native_lib.arc_group_rows_workspace_bytes(16, 4, ctypes.byref(size)) == 0 and size.value == 0
    assert native_lib.arc_group_rows_workspace_bytes(1 << 20, 4, ctypes.byref(size)) == 0 and size.value > 0

    def call(ids=p, b=8, off=p, rows=p, pos=p, ws=None, wsb=0, slots=16, top=2, e=4):
        return f(ids, b, off, rows, pos, ws, wsb, slots, top, e, None)

    for name in ("ids", "off", "rows", "pos"):
        assert call(**{name: None}) == BAD
    assert call(slots=0) == BAD and call(top=0) == BAD and call(e=0) == BAD
    assert call(b=2) == UNS and call(e=1025) == UNS and call(ids=p + 4) == UNS and call(rows=p + 2) == UNS
    assert call(slots=0x7FFFFFFF) == UNS
    assert call(slots=1 << 20) == BAD  # no workspace


@pytest.fixture(scope="session")
def torch_ops(native_lib):
    """The built PyTorch operators (built here if missing; the build is CPU-only)."""
    from arc import build

    build.build_torch_ops()
    return _lib.torch_ops()


def test_python_refuses_cpu_tensors(torch_ops):
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(3, 8, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        arc.linear(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        arc.grouped_matmul(x, torch.zeros(2, 3, 8, dtype=torch.bfloat16), off)
    with pytest.raises(ValueError, match="CUDA"):
        arc.a8w4_grouped_matmul((torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2)),
                                (torch.zeros(2, 8, 64, dtype=torch.uint8), torch.zeros(2, 8, 1, dtype=torch.bfloat16)), off)
    with pytest.raises(ValueError, match="CUDA"):
        arc.group_rows(torch.zeros(2, 2, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="activation"):
        arc.linear(x, w, activation="tanh")
    with pytest.raises(TypeError):
        arc.linear([1.0], w)
