"""The linear layer on the B200 against its definition in 64 bits, forward and gradients."""
from __future__ import annotations

import pytest
import torch

import arc
from arc import _lib
from linear_bounds import act64, assert_within, linear_forward, linear_gradients, normal

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
PLANS = ["pair:1", "pair:2", "pair128:1", "pair128:2", "16:1", "16:4", "32:2", "64:1", "128:8", "128:1"]


def _inputs(m, n, k, seed=0, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    return (normal(g, m, k), normal(g, n, k, scale=k ** -0.5), normal(g, n) if bias else None,
            normal(g, m, n) if residual else None)


def _check(m, n, k, act, bias=True, residual=True, seed=0):
    x, w, b, r = _inputs(m, n, k, seed, bias, residual)
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    assert arc.linear(x, w, b, r, activation=act, out=out) is out
    y, bound, _, _ = linear_forward(x, w, b, r, act)
    assert_within(out, y, bound, f"linear {m}x{n}x{k} {act}")
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (16, 128, 512), (17, 129, 520), (128, 256, 64), (130, 264, 1000),
                                   (257, 515, 328)])
def test_every_plan(cuda_device, monkeypatch, plan, m, n, k):
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    _check(m, n, k, "gelu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("m,n,k", [(3, 200, 136), (600, 300, 72)])
def test_epilogues(cuda_device, m, n, k, act, bias, residual):
    _check(m, n, k, act, bias, residual)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (16, 14336, 4096), (333, 1003, 2056), (2048, 4096, 512)])
def test_real_sizes(cuda_device, m, n, k):
    _check(m, n, k, "silu")


@pytest.mark.parametrize("plan", ["pair:1", "pair:2", "pair128:1", "pair128:2", "16:4", "128:1"])
def test_strided_operands(cuda_device, monkeypatch, plan):
    """Column slices of wider matrices; an output whose rows are not 16-byte aligned."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    g = torch.Generator().manual_seed(3)
    x = normal(g, 70, 600)[:, 16:536]
    w = normal(g, 99, 640, scale=0.05)[:, 8:528]
    r = normal(g, 70, 150)[:, 1:100]
    b = normal(g, 200)[1:100]
    buf = torch.full((70, 151), 7.0, dtype=torch.bfloat16, device="cuda")
    arc.linear(x, w, b, r, activation="relu", out=buf[:, 3:102])
    y, bound, _, _ = linear_forward(x, w, b, r, "relu")
    assert_within(buf[:, 3:102], y, bound, "strided")
    assert (buf[:, :3] == 7).all() and (buf[:, 102:] == 7).all()
    # transposed operands are laid out first
    assert_within(arc.linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r, activation="relu"), y, bound, "copied")


def test_in_place_residual(cuda_device):
    x, w, b, r = _inputs(40, 96, 64)
    y, bound, _, _ = linear_forward(x, w, b, r, None)
    assert_within(arc.linear(x, w, b, r, out=r), y, bound, "in place")


@pytest.mark.parametrize("act", ACTS)
def test_special_values(cuda_device, act):
    """Infinities and NaN go through the epilogue as through the formula; finite rows stay finite."""
    x = torch.zeros(5, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.eye(8, dtype=torch.bfloat16, device="cuda")
    r = torch.zeros(5, 8, dtype=torch.bfloat16, device="cuda")
    b = torch.tensor([300.0, -300.0, 3e38, -3e38, 0.0, -4.0, -9.0, 9.0], device="cuda").to(torch.bfloat16)
    r[1, 0] = float("inf")
    r[2, 0] = float("nan")
    got = arc.linear(x, w, b, r, activation=act).double()
    want = act64(b.double(), act).expand(5, 8) + r.double()
    if act == "gelu_tanh":  # z^3 overflows fp32 there, with the right limit
        want[:, 3] = r.double()[:, 3]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert torch.allclose(got[fine], want[fine], rtol=2.0 ** -8 + 2.0 ** -16, atol=2.0 ** -19)


def _leaves(*ts):
    return [t.detach().clone().requires_grad_() if t is not None else None for t in ts]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (5, 33, 40), (200, 120, 136), (64, 1003, 72), (700, 520, 264)])
def test_gradients(cuda_device, m, n, k, act):
    x, w, b, r = _inputs(m, n, k, seed=m)
    dy = normal(torch.Generator().manual_seed(9), m, n)
    lx, lw, lb, lr = _leaves(x, w, b, r)
    y = arc.linear(lx, lw, lb, lr, activation=act)
    y.backward(dy)
    want, bound, z, zerr = linear_forward(x, w, b, r, act)
    assert_within(y.detach(), want, bound, "y")
    grads = linear_gradients(x, w, z, zerr, dy, act)
    for name, leaf in (("dx", lx), ("dw", lw), ("dbias", lb)):
        assert_within(leaf.grad, *grads[name], f"{name} {act}")
    assert torch.equal(lr.grad, dy)
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("m,n,k", [(300, 264, 136), (1000, 260, 520), (4100, 72, 64), (520, 300, 2056)])
def test_split_contractions(cuda_device, m, n, k):
    """Few tiles and long contractions, in every product of a training step; the same bits each time."""
    x, w, b, _ = _inputs(m, n, k, seed=m, residual=False)
    dy = normal(torch.Generator().manual_seed(9), m, n)
    first = None
    for _ in range(4):
        leaves = _leaves(x, w, b)
        y = arc.linear(*leaves, activation="silu")
        got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
        if first is None:
            first = got
            want, bound, z, zerr = linear_forward(x, w, b, None, "silu")
            assert_within(got[0], want, bound, "y")
            grads = linear_gradients(x, w, z, zerr, dy, "silu")
            for v, name in zip(got[1:], ("dx", "dw", "dbias")):
                assert_within(v, *grads[name], name)
        for a, c in zip(got, first):
            assert torch.equal(a, c)
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(cuda_device, act):
    """The kernels' gradients along a direction against central differences of the 64-bit form."""
    m, n, k, h = 24, 40, 48, 1e-5
    x, w, b, _ = _inputs(m, n, k, seed=5, residual=False)
    g = torch.Generator().manual_seed(6)
    dy = normal(g, m, n)
    lx, lw, lb = _leaves(x, w, b)
    arc.linear(lx, lw, lb, activation=act).backward(dy)
    y, _, z, zerr = linear_forward(x, w, b, None, act)
    grads = linear_gradients(x, w, z, zerr, dy, act)

    def loss(xx, ww, bb):
        return (act64(xx @ ww.T + bb, act) * dy.double()).sum()

    for i, (name, leaf) in enumerate((("dx", lx), ("dw", lw), ("dbias", lb))):
        args = [x.double(), w.double(), b.double()]
        d = torch.randn(leaf.shape, generator=g).double().cuda()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        diff = (loss(*up) - loss(*down)) / (2 * h)
        # the kernels' bound along d, and the differences' own error (h^2 and cancellation)
        tol = (grads[name][1] * d.abs()).sum() + 1e-4
        assert (leaf.grad.double() * d).sum().sub(diff).abs() <= tol, name


def test_partial_gradients_and_layouts(cuda_device):
    """Only some inputs need gradients; the output gradient is expanded, transposed or sliced."""
    m, n, k = 50, 33, 64
    x, w, b, _ = _inputs(m, n, k, residual=False)
    _, _, z, zerr = linear_forward(x, w, b, None, "silu")
    g = torch.Generator().manual_seed(1)
    wide = normal(g, m, n + 7)
    for dy in (torch.ones((), dtype=torch.bfloat16, device="cuda").expand(m, n), normal(g, n, m).t(), wide[:, 5:5 + n]):
        want = linear_gradients(x, w, z, zerr, dy, "silu")
        for need in ("dx", "dw", "dbias"):
            lx, lw, lb = (t.clone().requires_grad_(need == s) for t, s in ((x, "dx"), (w, "dw"), (b, "dbias")))
            (got,) = torch.autograd.grad(arc.linear(lx, lw, lb, activation="silu"),
                                         [{"dx": lx, "dw": lw, "dbias": lb}[need]], dy)
            assert_within(got, *want[need], need)
    lx, lw, lb = _leaves(x, w, b)
    y = arc.linear(lx, lw, lb)  # no activation: dy itself goes into the products
    got = torch.autograd.grad(y, [lx, lw, lb], wide[:, 5:5 + n])
    _, _, z, zerr = linear_forward(x, w, b, None, None)
    want = linear_gradients(x, w, z, zerr, wide[:, 5:5 + n], None)
    for v, name in zip(got, ("dx", "dw", "dbias")):
        assert_within(v, *want[name], name)


def test_single_row_and_column_layouts(cuda_device):
    """One row or one column: the other stride may be anything."""
    x, w, b, r = _inputs(1, 24, 64)
    y, bound, _, _ = linear_forward(x, w, b, r, "relu")
    odd = [t.as_strided(t.shape, (3, 1)) for t in (x, r)]
    assert_within(arc.linear(odd[0], w, b, odd[1], activation="relu"), y, bound, "row")
    out = torch.empty(24, dtype=torch.bfloat16, device="cuda").as_strided((1, 24), (5, 1))
    assert_within(arc.linear(x, w, b, r, activation="relu", out=out), y, bound, "out")
    lx, lw, lb = _leaves(x, w, b)
    arc.linear(lx, lw, lb).backward(odd[1])
    _, _, z, zerr = linear_forward(x, w, b, None, None)
    for leaf, name in ((lx, "dx"), (lw, "dw"), (lb, "dbias")):
        assert_within(leaf.grad, *linear_gradients(x, w, z, zerr, r, None)[name], name)
    x, w, b, r = _inputs(9, 1, 64)
    y, bound, _, _ = linear_forward(x, w, b, r, None)
    assert_within(arc.linear(x, w, b, r.t().contiguous().t()), y, bound, "column")


def test_no_rows(cuda_device):
    x, w, b, _ = _inputs(4, 24, 16, residual=False)
    assert arc.linear(x[:0], w, b).shape == (0, 24)
    lx, lw, lb = _leaves(x[:0], w, b)
    arc.linear(lx, lw, lb, activation="gelu").sum().backward()
    assert lx.grad.shape == (0, 16) and (lw.grad == 0).all() and (lb.grad == 0).all()


@pytest.mark.parametrize("m", [2, 300])
def test_graph_and_streams(cuda_device, m):
    """Capture and replay on another stream, with new inputs, forward and backward."""
    x, w, b, r = _inputs(m, 264, 136)
    dy = normal(torch.Generator().manual_seed(2), m, 264)
    lx, lw, lb = _leaves(x, w, b)

    def step():
        y = arc.linear(lx, lw, lb, r, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, [lx, lw, lb], dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for t in captured:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(eager, captured):
        assert torch.equal(a, c)
    with torch.no_grad():
        lx.mul_(0.5)
    graph.replay()
    for a, c in zip(step(), captured):
        assert torch.equal(a, c)
    assert arc.device_status(0) == 0


def test_two_streams_at_once(cuda_device):
    cases = [_inputs(m, 512, 1024, seed=m) for m in (4, 300)]
    want = [arc.linear(*c, activation="silu") for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(8):
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(arc.linear(*c, activation="silu"))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert torch.equal(t, want[i % 2])


def test_second_derivatives_are_refused(cuda_device):
    x, w, b, _ = _inputs(4, 24, 16, residual=False)
    lx, lw, lb = _leaves(x, w, b)
    dy = torch.ones(4, 24, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(arc.linear(lx, lw, lb, activation="gelu"), [lx], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dx.sum().backward()


def test_unused_gradients_and_no_grad(cuda_device):
    x, w, b, r = _inputs(4, 24, 16)
    lx, lw = _leaves(x, w)
    with torch.no_grad():
        assert not arc.linear(lx, lw, b, r).requires_grad
    out = torch.empty_like(r)
    with torch.no_grad():
        arc.linear(lx, lw, b, r, out=out)
    lr = r.clone().requires_grad_()
    arc.linear(x, w, b, lr).backward(r)  # only the residual's
    assert torch.equal(lr.grad, r)
    # twice through the same leaves accumulates
    arc.linear(lx, lw, b).backward(r)
    first = lw.grad.clone()
    arc.linear(lx, lw, b).backward(r)
    assert torch.equal(lw.grad, first + first)


def test_refusals(cuda_device):
    x, w, b, r = _inputs(4, 24, 16)
    with pytest.raises(ValueError, match="activation"):
        arc.linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="Inner"):
        arc.linear(x, w[:, :8])
    with pytest.raises(TypeError):
        arc.linear(x.float(), w)
    with pytest.raises(ValueError, match="bias"):
        arc.linear(x, w, b[:8])
    with pytest.raises(ValueError, match="residual"):
        arc.linear(x, w, b, r[:2])
    with pytest.raises(ValueError, match="2-D"):
        arc.linear(x[None], w)
    with pytest.raises(ValueError, match="out"):
        arc.linear(x, w, out=torch.empty(4, 23, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="gradient"):
        arc.linear(x.clone().requires_grad_(), w, out=r)


def test_any_contraction_size(cuda_device):
    """Rows that are not 16-byte aligned are laid out first."""
    for k in (1, 7, 12, 131):
        _check(9, 24, k, "gelu")
        x, w, b, _ = _inputs(9, 24, k, residual=False)
        dy = normal(torch.Generator().manual_seed(9), 9, 24)
        leaves = _leaves(x, w, b)
        got = torch.autograd.grad(arc.linear(*leaves, activation="gelu"), leaves, dy)
        _, _, z, zerr = linear_forward(x, w, b, None, "gelu")
        want = linear_gradients(x, w, z, zerr, dy, "gelu")
        for v, name in zip(got, ("dx", "dw", "dbias")):
            assert_within(v, *want[name], name)


def test_second_derivatives_by_operands_are_refused(cuda_device):
    """dx depends on w and dw on x, also where dy is a constant."""
    x, w, _, _ = _inputs(4, 24, 16, bias=False, residual=False)
    lx, lw = _leaves(x, w)
    (dx,) = torch.autograd.grad(arc.linear(lx, lw).sum(), [lx], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        (dx * dx).sum().backward()


def test_out_is_refused_where_it_would_be_wrong(cuda_device):
    x, w, b, r = _inputs(32, 32, 32)
    for bad in (x, w, x.view(-1).view(32, 32)):  # views included
        with pytest.raises(ValueError, match="overlap"):
            arc.linear(x, w, b, out=bad)
    buf = torch.zeros(33 * 32, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="residual"):
        arc.linear(x, w, b, buf[:1024].view(32, 32), out=buf[32:].view(32, 32))
    with pytest.raises(ValueError, match="gradient"):
        arc.linear(x, w, b, out=r.clone().requires_grad_())
    # Side by side in one buffer is no overlap.
    both = torch.zeros(32, 64, dtype=torch.bfloat16, device="cuda")
    both[:, :32] = x
    arc.linear(both[:, :32], w, b, out=both[:, 32:])
    y, bound, _, _ = linear_forward(x, w, b, None, None)
    assert_within(both[:, 32:], y, bound, "side by side")
    # A tensor that a graph has saved is not overwritten unnoticed.
    h = x.clone()
    y = arc.linear(h, w.clone().requires_grad_())
    arc.linear(x, w, out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("m,n", [(70_001, 32_776), (32_776, 70_001)])
def test_past_two_to_the_31st_element(cuda_device, m, n):
    """Outputs, z and dz of more than 2^31 elements; dy is zero but for a few rows."""
    k = 64
    x, w, b, _ = _inputs(m, n, k, residual=False)
    rows = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
    leaves = _leaves(x, w, b)
    y = arc.linear(*leaves, activation="silu")
    want, bound, z, zerr = linear_forward(x[rows], w, b, None, "silu")
    assert_within(y.detach()[rows], want, bound, "y")
    some = normal(torch.Generator().manual_seed(1), 5, n)
    dy = torch.zeros_like(y).index_copy_(0, rows, some)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    grads = linear_gradients(x[rows], w, z, zerr, some, "silu")
    assert_within(dx[rows], *grads["dx"], "dx")
    assert_within(dw, *grads["dw"], "dw")
    assert_within(db, *grads["dbias"], "dbias")
    assert dx.count_nonzero() == dx[rows].count_nonzero()
    assert arc.device_status(0) == 0


def test_kernel_name(cuda_device, monkeypatch):
    name = lambda *s: arc.kernel_name(_lib.OP_LINEAR, *s)  # noqa: E731
    assert name(4096, 14336, 4096) == "gemm_linear_pair_kernel<0, 0, 0, 0, 256>"
    assert name(16, 14336, 4096) == "gemm_linear_stream_kernel<16, 0>"
    monkeypatch.setenv("ARC_LINEAR_PLAN", "pair:2")
    assert name(16, 14336, 4096) == "gemm_linear_pair_kernel<0, 0, 0, 1, 256>"


@pytest.mark.parametrize("plan", ["pair:1", "pair:2", "pair128:1", "pair128:2", "32:2"])
@pytest.mark.parametrize("m,n,k", [(300, 264, 136), (1000, 1500, 520), (2600, 2056, 264)])
def test_row_gradient_by_every_plan(cuda_device, monkeypatch, plan, m, n, k):
    """The row gradient takes the forward product's kernels with w read MN-major; several tiles per pair."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    x, w, _, _ = _inputs(m, k, n, bias=False, residual=False)
    dy = normal(torch.Generator().manual_seed(2), m, k)
    lx = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(arc.linear(lx, w), [lx], dy)
    z = x.double() @ w.double().T
    want = linear_gradients(x, w, z, torch.zeros_like(z), dy, None)
    assert_within(dx, *want["dx"], "dx")
    _check(m, n, k, "silu")
    assert arc.device_status(0) == 0
