"""arc.lora_linear on the B200 against its definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import arc
from linear_bounds import F, H, SUM, act64, assert_within, normal

pytestmark = pytest.mark.gpu

PLANS = ["16:1", "16:4", "32:2", "64:8", "128:1", "128:4", "pair:1", "pair:2", "pair128:1", "pair128:2"]


def reference(x, w, a, b, ids, bias=None, residual=None, scales=None, act=None):
    """(y, bound): as linear_bounds.linear_forward, with u's sum (k terms), its scale and its rounding to bf16 on top,
    and the r products of u in the sum."""
    xd, wd = x.double(), w.double()
    k, r = x.shape[1], a.shape[1]
    z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    zerr = torch.zeros_like(z)
    for i in range(a.shape[0]):
        rows = torch.nonzero(ids == i)[:, 0]
        if rows.numel() == 0:
            continue
        s = 1.0 if scales is None else scales[i].double()
        u = s * (xd[rows] @ a[i].double().T)
        uerr = abs(s) * k * SUM * (xd[rows].abs() @ a[i].double().abs().T) + 2.0 ** -22 * u.abs()
        uerr = uerr + H * (u.abs() + uerr) + 1e-38
        z[rows] += u @ b[i].double().T
        mag[rows] += (u.abs() + uerr) @ b[i].double().abs().T
        zerr[rows] += uerr @ b[i].double().abs().T
    zerr = zerr + (k + r) * SUM * mag
    if bias is not None:
        z = z + bias.double()
        zerr = zerr + 2.0 ** -23 * (z.abs() + bias.double().abs())
    y = act64(z, act)
    yerr = 1.2 * zerr + F * y.abs() + 2.0 ** -22 * z.abs()
    if residual is not None:
        y = y + residual.double()
    return y, yerr + H * (y.abs() + yerr) + F * y.abs() + 1e-30


def _inputs(m, n, k, r, count, seed=0, runs=False, without=0.2):
    g = torch.Generator().manual_seed(seed)
    x, w = normal(g, m, k), normal(g, n, k, scale=k ** -0.5)
    a, b = normal(g, count, r, k, scale=k ** -0.5), normal(g, count, n, r, scale=r ** -0.5)
    if runs:
        cuts = torch.randint(0, m + 1, (runs - 1,), generator=g).sort().values.tolist()
        owner = torch.randint(-1, count, (runs,), generator=g)
        ids = torch.repeat_interleave(owner, torch.tensor([q - p for p, q in zip([0] + cuts, cuts + [m])]))
    else:
        ids = torch.randint(0, count, (m,), generator=g)
        ids[torch.rand(m, generator=g) < without] = -1
    scales = (0.25 + torch.rand(count, generator=g)).cuda()
    return x, w, a, b, ids.to(torch.int32).cuda(), normal(g, n), normal(g, m, n), scales


def _check(args, act=None, what=""):
    x, w, a, b, ids, bias, residual, scales = args
    want, bound = reference(x, w, a, b, ids, bias, residual, scales, act)
    got = arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales, activation=act)
    assert_within(got, want, bound, what)
    assert arc.device_status(0) == 0
    return got


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("m,n,k,r,count", [(1, 136, 512, 16, 4), (37, 300, 520, 24, 7), (300, 264, 1032, 8, 40),
                                           (530, 136, 512, 72, 3)])
def test_plans(cuda_device, monkeypatch, plan, m, n, k, r, count):
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    _check(_inputs(m, n, k, r, count, seed=m), "gelu", plan)
    _check(_inputs(m, n, k, r, count, seed=m + 1, runs=5), None, plan + " runs")


@pytest.mark.parametrize("r", [1, 8, 13, 16, 32, 40, 64, 65, 128, 200, 256])
def test_ranks(cuda_device, r):
    _check(_inputs(50, 200, 264, r, 5, seed=r), "silu", r)
    _check(_inputs(700, 512, 264, r, 5, seed=r, runs=6), "silu", r)


@pytest.mark.parametrize("m,n,k,r,count", [(1, 4096, 4096, 16, 8), (2, 8, 8, 8, 1), (16, 1024, 72, 16, 1024), (33, 77, 2056, 16, 64),
                                           (64, 512, 4096, 64, 64), (257, 1000, 328, 16, 300), (1100, 520, 136, 32, 9)])
def test_shapes(cuda_device, m, n, k, r, count):
    _check(_inputs(m, n, k, r, count, seed=3), "gelu_tanh")


def test_every_row_its_own_adapter(cuda_device):
    x, w, a, b, ids, bias, residual, scales = _inputs(256, 128, 136, 8, 256, seed=6)
    ids = torch.randperm(256, generator=torch.Generator().manual_seed(1)).cuda()  # int64
    for plan in (None, "pair:1"):
        with pytest.MonkeyPatch.context() as mp:
            if plan:
                mp.setenv("ARC_LINEAR_PLAN", plan)
            _check((x, w, a, b, ids, bias, residual, scales), "relu")


def test_without_adapters_it_is_linear(cuda_device):
    """No row has one: bit for bit arc.linear's result. Ids outside [0, L) count as none, adapters full of NaN that no
    row has are not read."""
    for m in (5, 600):
        x, w, a, b, ids, bias, residual, scales = _inputs(m, 264, 520, 16, 4)
        a[:], b[:], scales[:] = float("nan"), float("inf"), float("nan")
        ids[:] = -1
        ids[::2] = 4
        got = arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales, activation="silu")
        assert torch.equal(got, arc.linear(x, w, bias, residual, activation="silu"))


def test_nan_stays_in_its_rows(cuda_device):
    for m, plan in ((40, None), (300, "pair:1")):
        x, w, a, b, ids, bias, residual, scales = _inputs(m, 136, 264, 16, 5, seed=9, without=0.1)
        want, bound = reference(x, w, a, b, ids, bias, residual, scales, None)
        a[2], b[3, :, 5] = float("nan"), float("inf")
        with pytest.MonkeyPatch.context() as mp:
            if plan:
                mp.setenv("ARC_LINEAR_PLAN", plan)
            got = arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales)
        keep = (ids != 2) & (ids != 3)
        assert_within(got[keep], want[keep], bound[keep], "other adapters")
        assert got[ids == 2].isnan().all() and not got[ids == 3].isfinite().all()


@pytest.mark.parametrize("plan", PLANS)
def test_nan_stays_in_its_rows_whatever_the_plan(cuda_device, monkeypatch, plan):
    """Adapters of NaN and infinities, and a row of NaN, beside the others of their tile; the rank passes one block of 64."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    for r in (16, 72):
        x, w, a, b, ids, bias, residual, scales = _inputs(150, 136, 520, r, 9, seed=r, without=0.1)
        want, bound = reference(x, w, a, b, ids, bias, residual, scales, None)
        a[2], b[3], scales[4] = float("nan"), float("inf"), float("inf")
        x[70] = float("nan")
        got = arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales)
        keep = (ids < 2) | (ids > 4)
        keep[70] = False
        assert_within(got[keep], want[keep], bound[keep], plan)
        assert got[70].isnan().all() and got[ids == 2].isnan().all() and not got[ids == 3].isfinite().all()


def test_adapters_beyond_32_bits_of_elements(cuda_device):
    """The last adapters of a and b lie more than 2^32 elements behind the first."""
    n, k, r, count = 32768, 32768, 136, 1024
    a = torch.empty(count, r, k, dtype=torch.bfloat16, device="cuda")
    b = torch.empty(count, n, r, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(3)
    last_a, last_b = normal(g, 1, r, 8), normal(g, 1, n, r, scale=r ** -0.5)
    a[-1].zero_()
    a[-1, :, -8:] = last_a[0]
    b[-1] = last_b[0]
    w = torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda").expand(n, k).contiguous()
    for m in (3, 300):
        x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
        x[:, -8:] = normal(g, m, 8)
        ids = torch.full((m,), count - 1, device="cuda")
        ids[1] = -1
        want, bound = reference(x[:, -8:], w[:, -8:], last_a, last_b, torch.where(ids > 0, 0, -1))
        got = arc.lora_linear(x, w, a, b, ids)
        assert_within(got, want, bound, m)
        assert (got[1] == 0).all()


def test_two_streams_at_once(cuda_device):
    calls = [_inputs(9, 264, 520, 16, 6, seed=1), _inputs(600, 264, 520, 16, 6, seed=2, runs=7), _inputs(40, 512, 1032, 72, 6)]

    def call(v):
        return arc.lora_linear(*v[:7], scales=v[7], activation="silu")

    want = [call(v) for v in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(10):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(((turn + j) % 3, call(calls[(turn + j) % 3])))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[j]) for j, v in got) and arc.device_status(0) == 0


def test_plain_call_strides_and_out(cuda_device):
    """No bias, residual or scales; operands and out inside wider buffers; the residual as out."""
    g = torch.Generator().manual_seed(2)
    x, w, a, b, ids, bias, residual, scales = _inputs(21, 100, 72, 16, 6, seed=8)
    want, bound = reference(x, w, a, b, ids)
    assert_within(arc.lora_linear(x, w, a, b, ids), want, bound, "plain")
    wx, ww, wa, wb = normal(g, 21, 96), normal(g, 120, 88), normal(g, 7, 20, 80), normal(g, 6, 110, 40)
    wx[:, 8:80], ww[8:108, 16:88], wa[1:, 2:18, 8:80], wb[:, 5:105, 24:40] = x, w, a, b
    buf = torch.full((21, 130), 3.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, 7:107]
    got = arc.lora_linear(wx[:, 8:80], ww[8:108, 16:88], wa[1:, 2:18, 8:80], wb[:, 5:105, 24:40], ids, out=out)
    assert got is out
    assert_within(got, want, bound, "strided")
    assert (buf[:, :7] == 3).all() and (buf[:, 107:] == 3).all()
    stacked = b.permute(1, 0, 2).contiguous().permute(1, 0, 2)  # adapters side by side
    assert_within(arc.lora_linear(x, w, a, stacked, ids), want, bound, "stacked")
    want, bound = reference(x, w, a, b, ids, bias, residual, scales, "silu")
    assert arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales, activation="silu", out=residual) is residual
    assert_within(residual, want, bound, "in place")


def test_captured_and_other_streams(cuda_device):
    small, large = _inputs(9, 264, 520, 16, 6, seed=1), _inputs(600, 264, 520, 16, 6, seed=2, runs=7)

    def call(v):
        return arc.lora_linear(*v[:7], scales=v[7], activation="silu")

    want = [call(v) for v in (small, large)]
    for _ in range(3):
        assert all(torch.equal(call(v), u) for v, u in zip((small, large), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [call(v) for v in (small, large)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(on_side, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [call(v) for v in (small, large, small)]
    for seed in (5, 6):
        fresh = _inputs(9, 264, 520, 16, 6, seed=seed)
        small[0].copy_(fresh[0]), small[4].copy_(fresh[4])
        graph.replay()
        now = call(small)
        assert torch.equal(captured[0], now) and torch.equal(captured[2], now) and torch.equal(captured[1], want[1])


def test_empty(cuda_device):
    x, w, a, b, ids, *_ = _inputs(3, 16, 64, 8, 2)
    assert arc.lora_linear(x[:0], w, a, b, ids[:0]).shape == (0, 16)


def test_refusals(cuda_device):
    x, w, a, b, ids, bias, residual, scales = _inputs(4, 64, 128, 16, 3)
    for args in ((x[:, :64], w, a, b, ids), (x, w, a[:2], b, ids), (x, w, a, b[:, :32], ids), (x, w, a, b[:, :, :8], ids),
                 (x, w, a, b, ids[:3]), (x, w, a, b, ids.cpu()), (x, w, a, b, ids[:, None]), (x, w[0], a, b, ids),
                 (x, w, a[:0], b[:0], ids), (x, w, a, b, ids, bias[:5]), (x, w, a, b, ids, bias, residual[:2])):
        with pytest.raises(ValueError):
            arc.lora_linear(*args)
    for args in ((x.float(), w, a, b, ids), (x, w, a.half(), b, ids), (x, w, a, b, ids.float())):
        with pytest.raises(TypeError):
            arc.lora_linear(*args)
    for bad in (scales[:2], scales.cpu()):
        with pytest.raises(ValueError):
            arc.lora_linear(x, w, a, b, ids, scales=bad)
    with pytest.raises(TypeError):
        arc.lora_linear(x, w, a, b, ids, scales=scales.double())
    with pytest.raises(ValueError):
        arc.lora_linear(x, w, a, b, ids, activation="tanh")
    with pytest.raises(ValueError, match="rank"):
        arc.lora_linear(x, w, a.repeat(1, 17, 1), b.repeat(1, 1, 17), ids)
    square = torch.empty(4, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        arc.lora_linear(square, normal(torch.Generator(), 128, 128), a, normal(torch.Generator(), 3, 128, 16), ids, out=square)
    with pytest.raises(RuntimeError, match="no gradient"):
        arc.lora_linear(x, w, a.clone().requires_grad_(), b, ids)
    with torch.no_grad():
        arc.lora_linear(x, w, a.clone().requires_grad_(), b, ids)


def test_decode_step(cuda_device):
    """A layer's step as a server runs it: the projection with adapters, then the experts, then the projection again, in
    one graph, equals the eager calls bit for bit."""
    t, k, e, i = 12, 256, 8, 128
    x, w, a, b, ids, bias, _, scales = _inputs(t, k, k, 16, 5, seed=4)
    g = torch.Generator().manual_seed(7)
    w_in, w_out = normal(g, e, 2 * i, k, scale=k ** -0.5), normal(g, e, k, i, scale=i ** -0.5)
    router = normal(g, e, k, scale=k ** -0.5)

    def step():
        h = arc.lora_linear(x, w, a, b, ids, bias, x, scales=scales, activation="silu")
        best = arc.linear(h, router).float().topk(2, dim=1)
        h = arc.moe(h, w_in, w_out, best.indices, torch.softmax(best.values, 1))
        return arc.lora_linear(h, w, a, b, ids, bias, h, scales=scales)

    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and arc.device_status(0) == 0
