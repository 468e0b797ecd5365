"""CPU: argument checks of the expert layer and of the linear layer with adapters, before any CUDA call."""
from __future__ import annotations

import ctypes

import pytest
import torch

import arc
from arc import _lib
from linear_bounds import H
from moe_reference import dequantized, moe_reference

BAD, UNS = _lib.ARC_ERR_INVALID_ARGUMENT, _lib.ARC_ERR_UNSUPPORTED


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.cast(buf, ctypes.c_void_p).value + 63) // 64 * 64


def test_moe_checks(native_lib, p, monkeypatch):
    f = native_lib.arc_moe

    def call(x=p, wi=p, si=None, wo=p, so=None, ids=p, idb=8, wt=p, wtb=4, out=p, ws=p, wsb=1 << 30, t=4, top=2, e=8, k=128,
             i=128, n=64, ldx=128, ldi=128, sti=256 * 128, ldo=128, sto=64 * 128, ldout=64, gated=1, act=4):
        return f(x, wi, si, wo, so, ids, idb, wt, wtb, out, ws, wsb, t, top, e, k, i, n, ldx, ldi, sti, ldo, sto, ldout,
                 gated, act, None)

    for name in ("x", "wi", "wo", "ids", "wt", "out"):
        assert call(**{name: None}) == BAD, name
    assert call(si=p) == BAD and call(so=p) == BAD  # scales of one only
    for name in ("t", "top", "e", "k", "i", "n"):
        assert call(**{name: 0}) == BAD, name
    assert call(t=257) == UNS and call(t=256, top=17) == UNS and call(e=1025, sti=1 << 30, sto=1 << 30) == UNS
    for name in ("k", "i", "n"):
        assert call(**{name: (1 << 20) + 128}) == UNS, name
    assert call(act=5) == BAD and call(act=-1) == BAD
    assert call(idb=2) == UNS and call(wtb=8) == UNS
    assert call(ldx=64) == BAD and call(ldi=64) == BAD and call(sti=128 * 128) == BAD and call(gated=0, sti=64 * 128) == BAD
    assert call(ldo=64) == BAD and call(sto=128) == BAD and call(ldout=63) == BAD
    assert call(x=p + 2) == UNS and call(wi=p + 8) == UNS and call(ldx=132) == UNS and call(out=p + 1) == UNS
    assert call(ids=p + 4) == UNS and call(wt=p + 2) == UNS
    assert call(si=p, so=p, k=192) == UNS and call(si=p, so=p, i=64) == UNS and call(si=p, so=p, wi=p + 4) == UNS
    assert call(si=p + 1, so=p) == UNS
    assert call(ws=None) == BAD and call(ws=p + 4) == BAD and call(wsb=100) == BAD
    for plan in ("8:1", "8:3:0", "64:1:0", "8:1:2"):
        monkeypatch.setenv("ARC_EXPERT_PLAN", plan)
        assert call() == BAD, plan


def test_every_allowed_batch_has_a_plan(native_lib, p):
    """Whatever tokens, choices and experts the limits allow, the kernels' shared memory holds them: without a GPU the call
    gets as far as asking for one."""
    if torch.cuda.is_available():
        pytest.skip("a GPU would be given these pointers, which are the host's")
    f = native_lib.arc_moe
    for t in (1, 2, 7, 8, 9, 16, 31, 32, 33, 64, 65, 127, 128, 129, 200, 255, 256):
        for top in (1, 2, 3, 8, 16, 32, 100, 4096 // t):
            for e in (1, 2, 8, 16, 40, 64, 100, 128, 256, 257, 512, 1000, 1024):
                if t * top > 4096:
                    continue
                for scales in (None, p):
                    st = f(p, p, scales, p, scales, p, 8, p, 4, p, p, 1 << 40, t, top, e, 128, 128, 64, 128, 128, 256 * 128, 128,
                           64 * 128, 64, 1, 4, None)
                    assert st not in (BAD, UNS), (t, top, e, scales is not None, native_lib.arc_last_error())


def test_moe_workspace(native_lib):
    size = ctypes.c_size_t(0)
    query = native_lib.arc_moe_workspace_bytes
    assert query(4, 2, 8, 128, 100, ctypes.byref(size)) == 0 and size.value == 8 * 104 * 2
    assert query(128, 2, 8, 128, 100, ctypes.byref(size)) == 0 and size.value == 256 * (104 + 128) * 2  # rows sorted too
    assert query(4, 2, 8, 128, 100, None) == BAD
    for args in ((0, 2, 8, 128, 100), (4, 0, 8, 128, 100), (4, 2, 0, 128, 100), (4, 2, 8, 128, 0), (257, 1, 8, 128, 100)):
        assert query(*args, ctypes.byref(size)) == BAD, args


def test_lora_checks(native_lib, p):
    f = native_lib.arc_lora_linear

    def call(x=p, w=p, a=p, b=p, ids=p, idb=4, sc=None, bias=None, res=None, out=p, ws=p, wsb=1 << 30, m=4, n=64, k=128, r=16,
             l=3, ldx=128, ldw=128, lda=128, sta=16 * 128, ldb=16, stb=64 * 16, ldr=64, ldo=64, act=0):
        return f(x, w, a, b, ids, idb, sc, bias, res, out, ws, wsb, m, n, k, r, l, ldx, ldw, lda, sta, ldb, stb, ldr, ldo, act,
                 None)

    for name in ("x", "w", "a", "b", "ids", "out"):
        assert call(**{name: None}) == BAD, name
    for name in ("m", "n", "k", "r", "l"):
        assert call(**{name: 0}) == BAD, name
    assert call(r=257, ldb=264) == UNS and call(l=1025) == UNS and call(idb=1) == UNS and call(act=7) == BAD
    assert call(ldx=120) == BAD and call(ldw=64) == BAD and call(lda=64) == BAD and call(sta=128) == BAD
    assert call(ldb=8) == BAD and call(stb=64) == BAD and call(ldo=63) == BAD and call(res=p, ldr=63) == BAD
    assert call(x=p + 2) == UNS and call(a=p + 8) == UNS and call(b=p + 2) == UNS and call(ldb=20, stb=64 * 20) == UNS
    assert call(sta=16 * 128 + 4) == UNS and call(out=p + 1) == UNS
    assert call(bias=p + 1) == UNS and call(sc=p + 2) == UNS and call(ids=p + 2) == UNS
    assert call(ws=None) == BAD and call(ws=p + 8) == BAD
    size = ctypes.c_size_t(0)
    query = native_lib.arc_lora_linear_workspace_bytes
    assert query(4, 64, 128, 16, None) == BAD
    for args in ((0, 64, 128, 16), (4, 0, 128, 16), (4, 64, 0, 16), (4, 64, 128, 0)):
        assert query(*args, ctypes.byref(size)) == BAD, args


@pytest.fixture()
def torch_ops(native_lib):
    from arc import build

    build.build_torch_ops()
    return _lib.torch_ops()


def test_python_refuses_cpu_tensors(torch_ops):
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w_in, w_out = torch.zeros(4, 256, 128, dtype=torch.bfloat16), torch.zeros(4, 128, 128, dtype=torch.bfloat16)
    ids, weights = torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2)
    with pytest.raises(ValueError, match="CUDA"):
        arc.moe(x, w_in, w_out, ids, weights)
    with pytest.raises(ValueError, match="activation"):
        arc.moe(x, w_in, w_out, ids, weights, activation="tanh")
    with pytest.raises(ValueError, match="CUDA"):
        arc.lora_linear(x, w_in[0], torch.zeros(3, 16, 128, dtype=torch.bfloat16), torch.zeros(3, 256, 16, dtype=torch.bfloat16),
                        torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="activation"):
        arc.lora_linear(x, w_in[0], x, x, ids, activation="tanh")


def test_the_reference_itself():
    """The 64-bit form the GPU tests compare with, against loops over its definition; and that its bound is one: the plain
    form in 32 bits, h and y rounded to bf16, stays inside it."""
    g = torch.Generator().manual_seed(0)
    t, top, e, k, i, n = 5, 3, 4, 128, 128, 24
    x = torch.randn(t, k, generator=g).to(torch.bfloat16)

    def pair(rows, inner):
        return (torch.randint(0, 256, (e, rows, inner // 2), generator=g, dtype=torch.uint8),
                (0.01 + 0.01 * torch.rand(e, rows, inner // 128, generator=g)).to(torch.bfloat16))

    w_in, w_out = pair(2 * i, k), pair(n, i)
    ids = torch.randint(-1, e, (t, top), generator=g)
    ids[0] = 1  # one expert three times
    weights = torch.rand(t, top, generator=g)
    code = int(w_in[0][1, 7, 3]) >> 4
    assert dequantized(w_in)[1, 7, 7] == (code - 16 if code >= 8 else code) * float(w_in[1][1, 7, 0])
    got, bound = moe_reference(x, w_in, w_out, ids, weights, "silu")
    fi, fo = dequantized(w_in), dequantized(w_out)
    rounded = torch.zeros(t, n)
    for r in range(t):
        want = torch.zeros(n, dtype=torch.float64)
        for j in range(top):
            if ids[r, j] < 0:
                continue
            gate, up = (fi[ids[r, j]] @ x[r].double()).split(i)
            want += weights[r, j].double() * (fo[ids[r, j]] @ (torch.nn.functional.silu(gate) * up))
            gate, up = (fi[ids[r, j]].float() @ x[r].float()).split(i)
            h = (torch.nn.functional.silu(gate) * up).to(torch.bfloat16).float()
            rounded[r] += weights[r, j] * (fo[ids[r, j]].float() @ h)
        assert torch.allclose(got[r], want, rtol=1e-12, atol=1e-13)
    assert ((rounded.to(torch.bfloat16).double() - got).abs() <= bound).all()
    assert bound.max() <= 8 * H * got.abs().max()  # and it is not a loose one
