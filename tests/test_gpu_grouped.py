"""Grouped products and the row grouping on the B200 against their definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

import arc
from arc._lib import STATUS_BAD_OFFSETS
from linear_bounds import H, SUM, assert_within, normal

pytestmark = pytest.mark.gpu

# Rows of each group, rows behind the last one.
SPLITS = [([5], 0), ([0, 0, 0], 4), ([1, 0, 1], 0), ([16, 17, 0, 15, 33], 3), ([0, 130, 300, 1, 0], 9),
          ([64, 64, 64, 64], 0), ([257, 63, 16, 48, 15, 1], 2)]
PLANS = ["pair:1", "16:1", "16:2", "32:1", "64:4", "128:1", "128:8"]


def _offsets(sizes):
    return torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def _inputs(sizes, behind, n, k, seed=0, poison=True):
    """Rows behind the last group hold NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    t = sum(sizes) + behind
    x, w, dy = normal(g, t, k), normal(g, len(sizes), n, k, scale=k ** -0.5), normal(g, t, n)
    if poison and behind:
        x[sum(sizes):] = float("nan")
        dy[sum(sizes):] = float("inf")
    return x, w, dy, _offsets(sizes)


def _spans(sizes):
    ends = [0, *torch.tensor(sizes).cumsum(0).tolist()]
    return list(zip(ends, ends[1:]))


def _reference(x, w, dy, sizes):
    """{name: (value, bound)} in float64; rows of no group are zero."""
    t, k = x.shape
    e, n, _ = w.shape
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"y": (new(t, n), new(t, n)), "dx": (new(t, k), new(t, k)), "dw": (new(e, n, k), new(e, n, k))}
    for i, (a, b) in enumerate(_spans(sizes)):
        xe, we, de = x[a:b].double(), w[i].double(), dy[a:b].double()
        for name, at, v, mag, terms in (("y", slice(a, b), xe @ we.T, xe.abs() @ we.abs().T, k),
                                        ("dx", slice(a, b), de @ we, de.abs() @ we.abs(), n),
                                        ("dw", i, de.T @ xe, de.abs().T @ xe.abs(), b - a)):
            err = terms * SUM * mag
            out[name][0][at], out[name][1][at] = v, err + H * (v.abs() + err) + 1e-30
    return out


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("sizes,behind", SPLITS)
@pytest.mark.parametrize("n,k", [(136, 200), (300, 64)])
def test_grouped_forward(cuda_device, monkeypatch, plan, sizes, behind, n, k):
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    x, w, dy, offsets = _inputs(sizes, behind, n, k)
    want, bound = _reference(x, w, dy, sizes)["y"]
    assert_within(arc.grouped_matmul(x, w, offsets), want, bound, "fresh")
    out = torch.full((x.shape[0], n), 5.0, dtype=torch.bfloat16, device="cuda")
    assert arc.grouped_matmul(x, w, offsets, out=out) is out
    assert (out[sum(sizes):] == 5).all(), "rows of no group were written"
    assert_within(out[:sum(sizes)], want[:sum(sizes)], bound[:sum(sizes)], "out")
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("plan", [None, "pair:1", "16:2", "64:1"])
@pytest.mark.parametrize("sizes,behind", SPLITS)
@pytest.mark.parametrize("n,k", [(136, 200), (77, 320)])
def test_grouped_gradients(cuda_device, monkeypatch, plan, sizes, behind, n, k):
    if plan:
        monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    x, w, dy, offsets = _inputs(sizes, behind, n, k, seed=4)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = arc.grouped_matmul(lx, lw, offsets)
    y.backward(dy)
    want = _reference(x, w, dy, sizes)
    assert_within(y.detach(), *want["y"], "y")
    assert_within(lx.grad, *want["dx"], "dx")
    assert_within(lw.grad, *want["dw"], "dw")
    assert arc.device_status(0) == 0


def test_poisoned_neighbours(cuda_device):
    """A group full of NaN and infinities leaves its neighbours' results and gradients alone."""
    sizes = [37, 20, 75]
    x, w, dy, offsets = _inputs(sizes, 0, 136, 72, seed=8)
    want = _reference(x, w, dy, sizes)
    x[37:57], dy[37:57] = float("nan"), float("-inf")
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = arc.grouped_matmul(lx, lw, offsets)
    y.backward(dy)
    for name, got in (("y", y.detach()), ("dx", lx.grad)):
        for a, b in ((0, 37), (57, 132)):
            assert_within(got[a:b], want[name][0][a:b], want[name][1][a:b], name)
    for e in (0, 2):
        assert_within(lw.grad[e], want["dw"][0][e], want["dw"][1][e], "dw")


def test_many_small_groups(cuda_device):
    g = torch.Generator().manual_seed(0)
    sizes = torch.randint(0, 4, (1024,), generator=g).tolist()
    x, w, dy, offsets = _inputs(sizes, 1, 16, 64)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = arc.grouped_matmul(lx, lw, offsets)
    y.backward(dy)
    want = _reference(x, w, dy, sizes)
    for name, got in (("y", y.detach()), ("dx", lx.grad), ("dw", lw.grad)):
        assert_within(got, *want[name], name)


def test_grouped_layouts(cuda_device):
    """Strided x, out and weight groups; rows before the first group; an expanded gradient."""
    g = torch.Generator().manual_seed(2)
    wide_x, wide_w = normal(g, 60, 100), normal(g, 3, 50, 88, scale=0.1)
    x, w = wide_x[:, 16:88], wide_w[:, 3:40, 8:80]
    offsets = torch.tensor([6, 20, 20, 51], dtype=torch.int32, device="cuda")
    buf = torch.full((60, 45), 3.0, dtype=torch.bfloat16, device="cuda")
    arc.grouped_matmul(x, w, offsets, out=buf[:, 4:41])
    fresh = arc.grouped_matmul(x, w, offsets)
    want = torch.zeros(60, 37, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for e, (a, b) in enumerate(((6, 20), (20, 20), (20, 51))):
        want[a:b] = x[a:b].double() @ w[e].double().T
        bound[a:b] = 72 * SUM * (x[a:b].double().abs() @ w[e].double().abs().T) * (1 + H) + H * want[a:b].abs()
    assert_within(fresh, want, bound, "fresh")
    assert torch.equal(buf[6:51, 4:41], fresh[6:51])
    assert (buf[:6] == 3).all() and (buf[51:] == 3).all() and (buf[:, :4] == 3).all() and (buf[:, 41:] == 3).all()
    lx = x.clone().requires_grad_()
    arc.grouped_matmul(lx, w, offsets).sum().backward()
    assert (lx.grad[:6] == 0).all() and (lx.grad[51:] == 0).all()
    assert arc.grouped_matmul(x[:0], w, torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 37)


@pytest.mark.parametrize("plan", [None, "pair:1", "16:1"])
@pytest.mark.parametrize("n", [96, 33])
def test_mostly_padding(cuda_device, monkeypatch, plan, n):
    """A buffer of which the groups fill little: the rest is zeroed, or left alone."""
    if plan:
        monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    g = torch.Generator().manual_seed(1)
    x, w = normal(g, 3000, 64), normal(g, 4, n, 64)
    offsets = torch.tensor([7, 10, 10, 40, 41], dtype=torch.int32, device="cuda")
    y = arc.grouped_matmul(x, w, offsets)
    assert (y[:7] == 0).all() and (y[41:] == 0).all() and (y[7:41] != 0).any(1).all()
    out = torch.full_like(y, 4.0)
    arc.grouped_matmul(x, w, offsets, out=out)
    assert (out[:7] == 4).all() and (out[41:] == 4).all() and torch.equal(out[7:41], y[7:41])
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(arc.grouped_matmul(lx, lw, offsets), [lx, lw], torch.ones_like(y))
    assert (dx[:7] == 0).all() and (dx[41:] == 0).all() and (dw[1] == 0).all()


def test_bad_offsets_are_reported(cuda_device):
    """Offsets outside the rows stay in bounds and set the status bit."""
    x, w, _, _ = _inputs([40], 0, 64, 64)
    w = w.expand(3, 64, 64).contiguous()
    for bad in ([0, 30, 10, 40], [-5, 10, 20, 40], [0, 10, 20, 4000]):
        arc.grouped_matmul(x, w, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert arc.device_status(0) == STATUS_BAD_OFFSETS
    assert arc.device_status(0) == 0


# ---------------------------------------------------------------------------------- A8W4
def _a8w4(sizes, behind, n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    t, e = sum(sizes) + behind, len(sizes)
    x = torch.randint(-127, 128, (t, k), generator=g).to(torch.int8).cuda()
    sa = (torch.rand(t, generator=g) + 0.5).cuda()
    wp = torch.randint(0, 256, (e, n, k // 2), generator=g).to(torch.uint8).cuda()
    sb = (torch.rand(e, n, k // 128, generator=g) + 0.1).to(torch.bfloat16).cuda()
    if behind:
        sa[sum(sizes):] = float("nan")
    return (x, sa), (wp, sb), _offsets(sizes)


@pytest.fixture(params=["narrow", "wide"])
def a8w4_kernel(request, monkeypatch):
    """Both kernels on every size: int32 partial sums, or scales in the fp16 operand."""
    monkeypatch.setenv("ARC_A8W4_GROUPED", request.param)
    return request.param


def _check_a8w4(kernel, a, b, sizes, offsets, prepacked=False):
    """Every group's rows against the definition in 64 bits. int32 partial sums are exact and the fp32
    scale sum is off by at most (G + 8) 2^-23 of its terms' magnitude, plus the rounding beside the bias
    kept in the accumulators (2^-24 of four terms of 1.5 * 2^23 / 16). Scales in the operand: an fp32 sum
    over K of exact products, and 2^-29 of the row's largest scale for a code whose scale fp16 rounds."""
    (x, sa), (wp, sb) = a, b
    e, n, k2 = wp.shape
    k = 2 * k2
    packed = arc.prepack_weights(wp.view(-1, k2)).view_as(wp) if prepacked else wp
    got = arc.a8w4_grouped_matmul(a, (packed, sb), offsets, prepacked=prepacked)
    total = sum(sizes)
    assert (got[total:] == 0).all()
    codes = torch.stack((wp & 15, wp >> 4), -1).flatten(-2).to(torch.int64)
    codes = torch.where(codes >= 8, codes - 16, codes).double()
    for i, (r0, r1) in enumerate(_spans(sizes)):
        if r0 == r1:
            continue
        xe, scale = x[r0:r1].double(), sa[r0:r1].double()[:, None]
        w = codes[i] * sb[i].double().repeat_interleave(128, 1)
        want = scale * (xe @ w.T)
        if kernel == "narrow":
            p = torch.einsum("tgk,ngk->tng", xe.view(r1 - r0, -1, 128), codes[i].view(n, -1, 128))
            mag = (p * sb[i].double()).abs().sum(-1)
            bias = 4 * 1.5 * 2.0 ** 23 / 16 * sb[i].double().abs().amax(-1) * 2.0 ** -24
            err = scale * ((k // 128 + 8) * SUM * mag + (k // 128) * bias)
        else:
            small = 2.0 ** -29 * sb[i].double().abs().amax(-1)
            err = scale * ((k + 4) * SUM * (xe.abs() @ w.abs().T) + xe.abs().sum(-1, keepdim=True) * small)
        assert_within(got[r0:r1], want, err + H * (want.abs() + err) + 1e-38, f"group {i}")
    out = torch.full_like(got, 2.0)
    arc.a8w4_grouped_matmul(a, (packed, sb), offsets, out=out, prepacked=prepacked)
    assert torch.equal(out[:total], got[:total]) and (out[total:] == 2).all()
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("sizes,behind", [*SPLITS, ([300, 0, 200], 1), ([20, 30, 25], 0), ([50, 60], 5)])
@pytest.mark.parametrize("n,k", [(8, 128), (264, 384), (520, 1024)])
@pytest.mark.parametrize("prepacked", [False, True])
def test_a8w4_grouped(cuda_device, a8w4_kernel, sizes, behind, n, k, prepacked):
    a, b, offsets = _a8w4(sizes, behind, n, k)
    _check_a8w4(a8w4_kernel, a, b, sizes, offsets, prepacked)


@pytest.mark.parametrize("k", [1024, 640])
def test_a8w4_scales(cuda_device, a8w4_kernel, k):
    """Scales that differ by many powers of two inside a row, zero, negative, tiny and huge ones."""
    a, (wp, sb), offsets = _a8w4([40, 300], 0, 64, k)
    g = torch.arange(k // 128, device="cuda")
    sb[:, :8] *= torch.exp2(-4.0 * g).to(torch.bfloat16)
    sb[:, 8:16] *= torch.exp2(-4.0 * g.flip(0)).to(torch.bfloat16)
    sb[:, 16:24] = 0
    sb[:, 24:32, 1] = 0
    sb[:, 32:40] *= -1
    sb[:, 40:48] *= 2.0 ** -100
    sb[:, 48:56] *= 2.0 ** 60
    _check_a8w4(a8w4_kernel, a, (wp, sb), [40, 300], offsets)


def test_a8w4_kernels_are_chosen_by_rows(cuda_device):
    for sizes in ([128, 100], [400, 300], [1, 0, 1500]):
        a, b, offsets = _a8w4(sizes, 0, 136, 256)
        _check_a8w4("wide" if sum(sizes) > 128 * len(sizes) else "narrow", a, b, sizes, offsets)


def _a8w4_on_gpu(a, b, offsets):
    """The product in fp64 on the GPU, group by group, and the magnitude of its terms."""
    (x, sa), (wp, sb) = a, b
    ends = offsets.tolist()
    want = torch.zeros(x.shape[0], wp.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    for i, (r0, r1) in enumerate(zip(ends, ends[1:])):
        codes = torch.stack((wp[i] & 15, wp[i] >> 4), -1).flatten(-2).to(torch.int16)
        w = torch.where(codes >= 8, codes - 16, codes).double() * sb[i].double().repeat_interleave(128, 1)
        xe = x[r0:r1].double() * sa[r0:r1].double()[:, None]
        want[r0:r1], mag[r0:r1] = xe @ w.T, xe.abs() @ w.abs().T
    return want, mag


@pytest.mark.parametrize("sizes,n,k", [([763, 578, 517, 684, 346, 455, 153, 597], 4096, 1024),
                                       ([300] * 24, 2056, 640), ([900, 100], 14336, 128), ([257] * 16, 1024, 2048),
                                       ([2] * 32, 4096, 1152), ([20] * 32, 4096, 1152), ([40] * 32, 4096, 1152),
                                       ([80, 1, 0, 128] * 8, 2048, 1152), ([1] * 512, 512, 256)])
def test_a8w4_many_tiles_per_block(cuda_device, a8w4_kernel, sizes, n, k):
    """Every block walks several tiles: the pipelines run on from tile to tile. The result is the
    same each time, bit for bit, and right."""
    g = torch.Generator(device="cuda").manual_seed(k)
    t, e = sum(sizes), len(sizes)
    a = (torch.randint(-127, 128, (t, k), generator=g, device="cuda").to(torch.int8),
         torch.rand(t, generator=g, device="cuda") + 0.5)
    b = (torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda").to(torch.uint8),
         (torch.rand(e, n, k // 128, generator=g, device="cuda") + 0.1).to(torch.bfloat16))
    offsets = _offsets(sizes)
    first = arc.a8w4_grouped_matmul(a, b, offsets)
    want, mag = _a8w4_on_gpu(a, b, offsets)
    err = (k + 8) * SUM * mag  # covers both kernels' sums
    assert_within(first, want, err + H * (want.abs() + err), "first")
    for _ in range(12):
        assert torch.equal(arc.a8w4_grouped_matmul(a, b, offsets), first)
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("sizes,n,k", [([763, 578, 517, 684, 0, 455, 153, 597], 2048, 1024), ([300] * 24, 1032, 520),
                                       ([17, 3, 9, 30] * 16, 2048, 1024)])
def test_grouped_many_tiles_per_block(cuda_device, sizes, n, k):
    x, w, dy, offsets = _inputs(sizes, 0, n, k)
    want = _reference(x, w, dy, sizes)
    first = None
    for _ in range(8):
        lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = arc.grouped_matmul(lx, lw, offsets)
        got = (y.detach(), *torch.autograd.grad(y, [lx, lw], dy))
        if first is None:
            first = got
            for v, name in zip(got, ("y", "dx", "dw")):
                assert_within(v, *want[name], name)
        for a, b in zip(got, first):
            assert torch.equal(a, b)


def test_a8w4_one_group_is_a8w4_matmul(cuda_device):
    a, (wp, sb), offsets = _a8w4([100], 0, 256, 512)
    assert torch.equal(arc.a8w4_grouped_matmul(a, (wp, sb), offsets), arc.a8w4_matmul(a, (wp[0], sb[0])))


# ---------------------------------------------------------------------------------- group_rows
def _group_rows_reference(ids, groups):
    flat = ids.reshape(-1).cpu().to(torch.int64)
    key = torch.where((flat < 0) | (flat >= groups), groups, flat)
    order = torch.sort(key, stable=True).indices
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel())
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), torch.bincount(key, minlength=groups + 1)[:groups].cumsum(0)))
    return offsets, order // (ids.shape[1] if ids.dim() == 2 else 1), positions.view(ids.shape)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,top,groups", [(1, 1, 1), (1, 8, 64), (3, 2, 5), (33, 3, 1024), (1024, 8, 64),
                                               (1025, 8, 256), (8193, 1, 7), (20000, 8, 1000), (70001, 6, 128)])
def test_group_rows(cuda_device, dtype, tokens, top, groups):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, groups + 1, (tokens, top), generator=g).to(dtype).cuda()
    if tokens > 3:
        ids[1] = ids[0]  # the same choice several times
        ids[-1] = torch.iinfo(dtype).min
        ids[-2] = torch.iinfo(dtype).max
    for got, want in zip(arc.group_rows(ids, groups), _group_rows_reference(ids, groups)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu().to(torch.int64), want)


def test_group_rows_extremes(cuda_device):
    for ids in (torch.zeros(40000, dtype=torch.int64), torch.full((9000, 2), -1), torch.full((100, 2), 3)):
        ids = ids.cuda()
        for got, want in zip(arc.group_rows(ids, 4), _group_rows_reference(ids, 4)):
            assert torch.equal(got.cpu().to(torch.int64), want)
    offsets, rows, positions = arc.group_rows(torch.empty(0, 8, dtype=torch.int32, device="cuda"), 4)
    assert offsets.tolist() == [0] * 5 and rows.numel() == 0 and positions.shape == (0, 8)


# ---------------------------------------------------------------------------------- together
def test_expert_layer(cuda_device):
    """Routing, two grouped products with an activation between and the way back, with gradients."""
    g = torch.Generator().manual_seed(11)
    tokens, top, e, k, n = 90, 2, 6, 64, 96
    x, w1, w2 = normal(g, tokens, k), normal(g, e, n, k, scale=0.1), normal(g, e, k, n, scale=0.1)
    ids = torch.rand(tokens, e, generator=g).topk(top, 1).indices.cuda()
    ids[-3:] = -1
    weights = torch.rand(tokens, top, generator=g).cuda()
    dy = torch.randn(tokens, k, generator=g).cuda()

    def layer(xx, a, b, product):
        offsets, rows, positions = arc.group_rows(ids, e)
        h = torch.nn.functional.silu(product(xx[rows.long()], a, offsets))
        y = product(h, b, offsets)
        return (y[positions.long()].to(dy.dtype if y.dtype != torch.float64 else torch.float64) * weights[..., None]).sum(1)

    def plain(v, m, offsets):
        ends = offsets.tolist()
        parts = [v[p:q] @ m[i].T for i, (p, q) in enumerate(zip(ends, ends[1:]))]
        return torch.cat((*parts, v.new_zeros(v.shape[0] - ends[-1], m.shape[1])))

    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    got = layer(*leaves, arc.grouped_matmul)
    got.backward(dy)
    exact = [t.double().requires_grad_() for t in (x, w1, w2)]
    want = layer(*exact, plain)
    want.backward(dy.double())
    # Five bf16 roundings on the way (h before and after silu, y, and two in the gradients):
    # each at most 2^-8 of what it rounds, relative to the result's norm.
    for a, b in ((got.detach(), want.detach()), *((p.grad, q.grad) for p, q in zip(leaves, exact))):
        assert (a.double() - b).norm() <= 5 * 2.0 ** -8 * b.norm()
    assert (got[-3:] == 0).all()


def test_graph_replay_with_new_routing(cuda_device):
    g = torch.Generator().manual_seed(3)
    e, n, k, tokens = 8, 128, 128, 64
    x, w = normal(g, tokens, k), normal(g, e, n, k, scale=0.1)
    ids = torch.randint(0, e, (tokens, 2), generator=g).cuda()
    (qx, sa), (wp, sb), _ = _a8w4([tokens * 2] + [0] * (e - 1), 0, n, k)

    def step():
        offsets, rows, positions = arc.group_rows(ids, e)
        return (arc.grouped_matmul(x[rows.long()], w, offsets), arc.a8w4_grouped_matmul((qx, sa), (wp, sb), offsets),
                offsets, positions)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        ids.copy_(torch.randint(-1, 3 * seed, (tokens, 2), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        for a, b in zip(step(), captured):
            assert torch.equal(a, b)
    assert arc.device_status(0) == 0


def test_refusals(cuda_device):
    x, w, _, offsets = _inputs([4, 4], 0, 24, 16)
    with pytest.raises(ValueError, match="offsets"):
        arc.grouped_matmul(x, w, offsets[:2])
    with pytest.raises(TypeError, match="offsets"):
        arc.grouped_matmul(x, w, offsets.long())
    with pytest.raises(ValueError, match="3-D"):
        arc.grouped_matmul(x, w[0], offsets)
    with pytest.raises(ValueError, match="Inner"):
        arc.grouped_matmul(x[:, :8], w, offsets)
    with pytest.raises(ValueError, match="gradient"):
        arc.grouped_matmul(x, w.clone().requires_grad_(), offsets, out=x)
    with pytest.raises(ValueError, match="groups"):
        arc.group_rows(torch.zeros(4, dtype=torch.int64, device="cuda"), 1025)
    with pytest.raises(TypeError, match="int32 or int64"):
        arc.group_rows(torch.zeros(4, device="cuda"), 4)
    a, b, off = _a8w4([4, 4], 0, 8, 128)
    with pytest.raises(ValueError):
        arc.a8w4_grouped_matmul(a, (b[0][:1], b[1]), off)
    with pytest.raises(TypeError):
        arc.a8w4_grouped_matmul((a[0].float(), a[1]), b, off)


def test_out_is_refused_where_it_would_be_wrong(cuda_device):
    x, w, _, offsets = _inputs([20, 12], 0, 32, 32)
    with pytest.raises(ValueError, match="overlap"):
        arc.grouped_matmul(x, w, offsets, out=x)
    with pytest.raises(ValueError, match="gradient"):
        arc.grouped_matmul(x, w, offsets, out=x.clone().requires_grad_())


@pytest.mark.parametrize("rows", [2, 40])
def test_weights_past_two_to_the_31st_element(cuda_device, rows):
    """Weights and their gradient of more than 2^31 elements, by the streaming and the pair kernel."""
    e, n, k = 33, 8192, 8200
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = (torch.randn(e * rows, c, generator=g, device="cuda").to(torch.bfloat16) for c in (k, n))
    w = torch.empty(e, n, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g).requires_grad_()
    lx = x.clone().requires_grad_()
    y = arc.grouped_matmul(lx, w, _offsets([rows] * e))
    dx, dw = torch.autograd.grad(y, [lx, w], dy)
    for i in (0, 15, e - 1):
        at = slice(i * rows, (i + 1) * rows)
        want = _reference(x[at], w.detach()[i:i + 1], dy[at], [rows])
        assert_within(y.detach()[at], *want["y"], "y")
        assert_within(dx[at], *want["dx"], "dx")
        assert_within(dw[i:i + 1], *want["dw"], "dw")
    assert arc.device_status(0) == 0


def test_a8w4_codes_past_two_to_the_31st_byte(cuda_device, a8w4_kernel):
    e, n, k, rows = 65, 8192, 8192, 3
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randint(-127, 128, (e * rows, k), generator=g, device="cuda").to(torch.int8)
    sa = torch.rand(e * rows, generator=g, device="cuda") + 0.5
    wp = torch.empty(e, n, k // 2, dtype=torch.uint8, device="cuda").random_(0, 256, generator=g)
    sb = (torch.rand(e, n, k // 128, generator=g, device="cuda") + 0.1).to(torch.bfloat16)
    got = arc.a8w4_grouped_matmul((x, sa), (wp, sb), _offsets([rows] * e))
    for i in (0, 31, e - 1):
        at = slice(i * rows, (i + 1) * rows)
        want, mag = _a8w4_on_gpu((x[at], sa[at]), (wp[i:i + 1], sb[i:i + 1]), _offsets([rows]))
        err = (k + 8) * SUM * mag
        assert_within(got[at], want, err + H * (want.abs() + err), f"group {i}")
    assert arc.device_status(0) == 0
