"""Edges of the grouped products on the B200: extreme scales, offsets that are not offsets."""
from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import arc
from arc._lib import STATUS_BAD_OFFSETS
from linear_bounds import H, SUM, assert_within, normal

pytestmark = pytest.mark.gpu


def _offsets(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kernel", ["narrow", "wide"])
@pytest.mark.parametrize("token,weight", [(-100, 100), (100, -100), (-30, -90), (-25, -108), (-20, -118)])
def test_a8w4_scales_far_apart(cuda_device, monkeypatch, kernel, token, weight):
    """Token scales of 2^token and weight scales of 2^weight: each alone fits fp32, and so does the result.

    Scaling by powers of two is exact, so the bounds are those of scales around one: an fp32 sum over K
    (k + 8 roundings of at most 2^-23 of the terms) and the rounding to bf16, whose last step is 2^-133;
    the sum before the token's scale is a normal number in every case.
    """
    monkeypatch.setenv("ARC_A8W4_GROUPED", kernel)
    g = torch.Generator().manual_seed(1)
    t, e, n, k = 40, 2, 24, 256
    x = torch.randint(-127, 128, (t, k), generator=g).to(torch.int8).cuda()
    wp = torch.randint(0, 256, (e, n, k // 2), generator=g).to(torch.uint8).cuda()
    sa = ((torch.rand(t, generator=g) + 0.5).double() * 2.0 ** token).float().cuda()
    sb = ((torch.rand(e, n, k // 128, generator=g) + 0.5).double() * 2.0 ** weight).to(torch.bfloat16).cuda()
    got = arc.a8w4_grouped_matmul((x, sa), (wp, sb), _offsets(0, 25, 40))
    codes = torch.stack((wp & 15, wp >> 4), -1).flatten(-2).to(torch.int16)
    w = torch.where(codes >= 8, codes - 16, codes).double() * sb.double().repeat_interleave(128, 2)
    xe = x.double() * sa.double()[:, None]
    want = torch.cat((xe[:25] @ w[0].T, xe[25:] @ w[1].T))
    mag = torch.cat((xe[:25].abs() @ w[0].abs().T, xe[25:].abs() @ w[1].abs().T))
    err = (k + 8) * SUM * mag
    assert_within(got, want, err + H * (want.abs() + err) + 2.0 ** -133, f"{kernel} {token} {weight}")
    assert arc.device_status(0) == 0


def test_bad_offsets_of_a_weight_gradient_are_reported(cuda_device):
    """The C entry point for dw alone reads the offsets too, and says when they are none."""
    from arc._lib import lib

    g = torch.Generator().manual_seed(0)
    t, e, n, k = 40, 3, 24, 16
    dy, x = normal(g, t, n), normal(g, t, k)
    dw = torch.empty(e, n, k, dtype=torch.bfloat16, device="cuda")
    for bad in ((0, 30, 10, 40), (-5, 10, 20, 40), (0, 10, 20, 4000), (0, 10, 20, 40)):
        off = _offsets(*bad)
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        status = lib().arc_grouped_matmul_dw(dy.data_ptr(), x.data_ptr(), off.data_ptr(), dw.data_ptr(), t, e, n, k,
                                             n, k, k, n * k, stream)
        assert status == 0
        assert arc.device_status(0) == (STATUS_BAD_OFFSETS if bad != (0, 10, 20, 40) else 0)


def test_forward_gradients_are_refused(cuda_device):
    g = torch.Generator().manual_seed(0)
    x, w, offsets = normal(g, 8, 16), normal(g, 2, 24, 16), _offsets(0, 4, 8)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, forward_ad.make_dual(w, torch.ones_like(w)))):
            for no_grad in (False, True):
                with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="forward"):
                    arc.grouped_matmul(*args, offsets)
        sa = forward_ad.make_dual(torch.ones(8, device="cuda"), torch.ones(8, device="cuda"))
        q = torch.zeros(8, 128, dtype=torch.int8, device="cuda")
        wp = torch.zeros(2, 8, 64, dtype=torch.uint8, device="cuda")
        sb = torch.ones(2, 8, 1, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(RuntimeError, match="forward"):
            arc.a8w4_grouped_matmul((q, sa), (wp, sb), offsets)
        with pytest.raises(RuntimeError, match="forward"):
            arc.a8w4_grouped_matmul((q, torch.ones(8, device="cuda")), (wp, forward_ad.make_dual(sb, sb)), offsets)


def test_operands_that_no_gradient_needs_may_change(cuda_device):
    g = torch.Generator().manual_seed(0)
    x, w, dy, offsets = normal(g, 8, 16), normal(g, 2, 24, 16), normal(g, 8, 24), _offsets(0, 5, 8)
    lx, frozen = x.clone().requires_grad_(), w.clone()
    y = arc.grouped_matmul(lx, frozen, offsets)
    with torch.no_grad():
        lx.mul_(2)  # dx does not need x
    (dx,) = torch.autograd.grad(y, [lx], dy)
    want = torch.cat((dy[:5].double() @ w[0].double(), dy[5:].double() @ w[1].double()))
    assert (dx.double() - want).norm() <= 2 * H * want.norm()
    lw, data = w.clone().requires_grad_(), x.clone()
    y = arc.grouped_matmul(data, lw, offsets)
    with torch.no_grad():
        lw.mul_(2)  # dw does not need w
    (dw,) = torch.autograd.grad(y, [lw], dy)
    want = torch.stack((dy[:5].double().T @ x[:5].double(), dy[5:].double().T @ x[5:].double()))
    assert (dw.double() - want).norm() <= 2 * H * want.norm()
    for changed in (data, offsets):
        y = arc.grouped_matmul(data, lw, offsets)
        changed.mul_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, [lw], dy)


def test_out_that_overlaps_is_refused(cuda_device):
    """Slices of one buffer, weights between the rows of out, and the offsets themselves."""
    g = torch.Generator().manual_seed(0)
    buf, w, offsets = normal(g, 32, 96), normal(g, 2, 32, 32), _offsets(0, 20, 32)
    for c in (0, 8, 31):
        with pytest.raises(ValueError, match="overlap"):
            arc.grouped_matmul(buf[:, :32], w, offsets, out=buf[:, c:c + 32])
    want = arc.grouped_matmul(buf[:, :32].clone(), w, offsets)
    assert torch.equal(arc.grouped_matmul(buf[:, :32], w, offsets, out=buf[:, 32:64]), want)
    flat = torch.zeros(2 * 40 * 96, dtype=torch.bfloat16, device="cuda")
    x = normal(g, 32, 32)
    weights = flat.view(2, 40, 96)[:, :32, :32]
    for bad in (flat.view(80, 96)[8:40, 24:56], flat.view(80, 96)[40:72, 31:63]):
        with pytest.raises(ValueError, match="overlap"):
            arc.grouped_matmul(x, weights, offsets, out=bad)
    weights.copy_(w)
    want = arc.grouped_matmul(x, w, offsets)
    for good in (flat.view(80, 96)[8:40, 32:64], flat.view(80, 96)[32:40, :32]):
        off = _offsets(0, 3, good.shape[0])
        want = arc.grouped_matmul(x[:good.shape[0]], w, off)
        assert torch.equal(arc.grouped_matmul(x[:good.shape[0]], weights, off, out=good), want)
    words = torch.zeros(8, 32, dtype=torch.bfloat16, device="cuda")
    words.view(torch.int32).view(-1)[:3] = torch.tensor([0, 4, 8], dtype=torch.int32)
    inside = words.view(torch.int32).view(-1)[:3]
    with pytest.raises(ValueError, match="overlap"):
        arc.grouped_matmul(x[:8], w, inside, out=words)
    q, sa = torch.zeros(8, 128, dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    wp = torch.zeros(2, 32, 64, dtype=torch.uint8, device="cuda")
    sb = torch.ones(2, 32, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        arc.a8w4_grouped_matmul((q, sa), (wp, sb), inside, out=words)


def test_weight_gradient_of_very_many_rows(cuda_device):
    """A contraction of 2^29 rows takes longer than the limit of an ordinary wait (2 s) and is no fault."""
    from arc._lib import lib

    t, n, k = 2 ** 29 + 37, 8, 8
    dy, x = (torch.zeros(t, c, dtype=torch.bfloat16, device="cuda") for c in (n, k))
    rows = torch.tensor([0, 1, 2 ** 28 + 3, t - 7, t - 6], device="cuda")
    g = torch.Generator().manual_seed(0)
    dy[rows], x[rows] = normal(g, 5, n), normal(g, 5, k)
    dy[t - 5:], x[t - 5:] = float("nan"), float("inf")  # behind the group
    dw = torch.empty(1, n, k, dtype=torch.bfloat16, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    off = _offsets(0, t - 5)
    assert lib().arc_grouped_matmul_dw(dy.data_ptr(), x.data_ptr(), off.data_ptr(), dw.data_ptr(), t, 1, n, k,
                                       n, k, k, n * k, stream) == 0
    assert arc.device_status(0) == 0
    want = dy[rows].double().T @ x[rows].double()
    err = 5 * SUM * (dy[rows].double().abs().T @ x[rows].double().abs())  # all other terms are zero
    assert_within(dw[0], want, err + H * (want.abs() + err), "dw")


@pytest.mark.parametrize("n,k", [(33, 131), (24, 64)])
def test_saved_tensors_may_move(cuda_device, n, k):
    """torch.autograd.graph.save_on_cpu brings the saved tensors back in a layout of its own."""
    g = torch.Generator().manual_seed(0)
    x, w, dy, offsets = normal(g, 40, k), normal(g, 2, n, k, scale=k ** -0.5), normal(g, 40, n), _offsets(0, 25, 40)
    leaves = [t.requires_grad_() for t in (x, w)]
    want = torch.autograd.grad(arc.grouped_matmul(*leaves, offsets), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = arc.grouped_matmul(*leaves, offsets)
    for got, ref in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(got, ref)
