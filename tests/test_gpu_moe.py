"""arc.moe on the B200 against its definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import arc
from linear_bounds import assert_within, normal
from moe_reference import moe_reference

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def _int4(g, e, n, k):
    packed = torch.randint(0, 256, (e, n, k // 2), generator=g, dtype=torch.uint8).cuda()
    scales = ((0.5 + torch.rand(e, n, k // 128, generator=g)) * (0.2 * k ** -0.5)).to(torch.bfloat16).cuda()
    return packed, scales


def _inputs(t, top, e, k, i, n=None, kind="bf16", gated=True, seed=0, skew=0.7, repeat=False):
    g = torch.Generator().manual_seed(seed)
    n = k if n is None else n
    rows = 2 * i if gated else i
    x = normal(g, t, k)
    if kind == "bf16":
        w_in, w_out = normal(g, e, rows, k, scale=k ** -0.5), normal(g, e, n, i, scale=i ** -0.5)
    else:
        w_in, w_out = _int4(g, e, rows, k), _int4(g, e, n, i)
    if repeat:
        ids = torch.randint(0, e, (t, top), generator=g)
    else:
        ids = (torch.randn(t, e, generator=g) + skew * torch.randn(e, generator=g)).topk(top, dim=1).indices
    weights = torch.softmax(torch.randn(t, top, generator=g), dim=1)
    return x, w_in, w_out, ids.cuda(), weights.cuda()


def _check(args, act, what="", **kw):
    want, bound = moe_reference(*args, act)
    got = arc.moe(*args, activation=act, **kw)
    assert_within(got, want, bound, what)
    assert arc.device_status(0) == 0
    return got


# tokens, top, experts, K, I: one token and many, odd sizes, one expert, passes of an expert that run over,
# contractions shorter than a box and no multiple of one.
SHAPES = [(1, 1, 1, 64, 64), (1, 8, 64, 512, 256), (2, 2, 4, 8, 8), (5, 3, 10, 136, 72), (16, 8, 64, 256, 128),
          (7, 1, 3, 1032, 520), (33, 4, 8, 200, 104), (100, 2, 3, 264, 136), (256, 8, 16, 128, 64), (3, 16, 1024, 72, 40), (256, 16, 1024, 64, 32), (256, 8, 200, 136, 72)]
SHAPES4 = [(1, 1, 1, 128, 128), (1, 8, 64, 512, 256), (5, 3, 10, 384, 128), (16, 8, 64, 256, 384), (33, 4, 8, 640, 128),
           (100, 2, 3, 256, 128), (256, 8, 16, 128, 256), (256, 16, 600, 128, 128), (250, 4, 100, 256, 128)]


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_bf16(cuda_device, shape, gated):
    _check(_inputs(*shape, gated=gated), "silu")


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("shape", SHAPES4)
def test_int4(cuda_device, shape, gated):
    _check(_inputs(*shape, kind="int4", gated=gated), "silu")


@pytest.mark.parametrize("kind,columns", [("bf16", 8), ("bf16", 16), ("bf16", 32), ("int4", 8), ("int4", 16)])
@pytest.mark.parametrize("splits,ordered", [(1, 0), (2, 1), (4, 0), (8, 1)])
def test_plans(cuda_device, monkeypatch, kind, columns, splits, ordered):
    """Every instantiation and cluster size, with experts of more choices than a pass holds."""
    monkeypatch.setenv("ARC_EXPERT_PLAN", f"{columns}:{splits}:{ordered}")
    for t in (3, 70):
        _check(_inputs(t, 2, 5, 640, 512, n=456, kind=kind, seed=t), "gelu", t)
    x, w_in, w_out, ids, weights = _inputs(40, 6, 4, 128, 256, kind=kind, repeat=True, seed=5)
    ids[3], ids[4, 1:] = -1, 7
    _check((x, w_in, w_out, ids, weights), "silu", "absent and repeated")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [True, False])
def test_activations(cuda_device, act, gated):
    _check(_inputs(9, 3, 6, 256, 128, gated=gated), act)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_features_out_and_types(cuda_device, kind):
    """N other than K, int32 ids, bf16 weights of the choices."""
    for n in (8, 33, 1001):
        x, w_in, w_out, ids, weights = _inputs(6, 3, 8, 256, 128, n=n, kind=kind)
        _check((x, w_in, w_out, ids.int(), weights.to(torch.bfloat16)), "silu", n)


def test_absent_and_repeated_experts(cuda_device):
    x, w_in, w_out, ids, weights = _inputs(40, 6, 4, 136, 72, repeat=True, seed=5)  # six of four: repeats
    ids[3], ids[4, 1:], ids[5, 0], ids[6, 2] = -1, 1 << 40, 4, -5
    got = _check((x, w_in, w_out, ids, weights), "silu")
    assert (got[3] == 0).all()
    ids[:] = -1
    assert (arc.moe(x, w_in, w_out, ids, weights) == 0).all()
    ids[:] = 2  # one expert six times, for all tokens
    _check((x, w_in, w_out, ids, weights), "silu")


def test_unchosen_experts_are_not_read(cuda_device):
    """NaN in unchosen experts, in tokens that choose nobody and in other tokens' rows stay where they are."""
    x, w_in, w_out, ids, weights = _inputs(11, 2, 9, 200, 104, seed=2)
    ids[ids == 4] = 5
    w_in[4], w_out[4] = float("nan"), float("inf")
    x[7] = float("nan")
    ids[7] = -1
    weights[7] = float("inf")
    x2 = x.clone()
    x2[7] = 0
    want, bound = moe_reference(x2, torch.nan_to_num(w_in), torch.nan_to_num(w_out, posinf=0.), ids, weights, "silu")
    got = arc.moe(x, w_in, w_out, ids, weights)
    keep = [i for i in range(11) if i != 7]
    assert_within(got[keep], want[keep], bound[keep], "others")
    assert (got[7] == 0).all()
    # A token full of NaN that does choose spoils its own row alone.
    ids[7] = torch.tensor([0, 1])
    got = arc.moe(x, w_in, w_out, ids, torch.nan_to_num(weights, posinf=1.0))
    assert got[7].isnan().all()
    assert_within(got[keep], want[keep], bound[keep], "beside a NaN token")


def test_int4_nan_stays_in_its_token(cuda_device):
    """Scales full of NaN of experts that nobody chooses are not read, and a token of infinities spoils its own row alone."""
    for t in (7, 40):
        x, w_in, w_out, ids, weights = _inputs(t, 2, 9, 256, 128, kind="int4", seed=t)
        ids[ids == 4] = 5
        want, bound = moe_reference(x, w_in, w_out, ids, weights, "silu")
        w_in[1][4], w_out[1][4] = float("nan"), float("inf")
        x[3] = float("inf")
        got = arc.moe(x, w_in, w_out, ids, weights)
        keep = [i for i in range(t) if i != 3]
        assert not got[3].isfinite().any()
        assert_within(got[keep], want[keep], bound[keep], t)


@pytest.mark.parametrize("power", [-50, -20, 20, 50])
def test_int4_large_and_small_activations(cuda_device, power):
    """The kernel's scaled codes keep a sum's relative precision: without an activation or a gate y is linear in x. (What
    the end of fp32's range takes, 2^-80 a product, is below the bound's 2^-23 of products of 2^-50.)"""
    x, w_in, w_out, ids, weights = _inputs(9, 2, 6, 256, 128, kind="int4", gated=False, seed=3)
    _check((x * 2.0 ** power, w_in, w_out, ids, weights), None, power)


@pytest.mark.parametrize("t,top,e", [(1, 4096, 1024), (1, 33, 40), (2, 100, 8), (40, 102, 300)])
def test_many_choices_of_a_token(cuda_device, t, top, e):
    _check(_inputs(t, top, e, 72, 40, repeat=True, seed=top), "silu")


def test_weights_beyond_32_bits_of_elements(cuda_device):
    """The last of the experts, 2^33 and 2^32 elements into the weights."""
    e, k, i = 17, 16384, 16384
    w_in, w_out = (torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((e, 2 * i, k), (e, k, i)))
    small_in, small_out = normal(torch.Generator().manual_seed(1), 64, k, scale=k ** -0.5), normal(torch.Generator(), 2, k)
    # h is nonzero in the last 32 gate and up rows alone, and in the last columns of w_out's rows.
    w_in[-1].zero_(), w_out[-1].zero_()
    w_in[-1, i - 32:i], w_in[-1, 2 * i - 32:] = small_in[:32], small_in[32:]
    w_out[-1, :, i - 2:] = small_out.T
    x = normal(torch.Generator().manual_seed(2), 2, k)
    ids, weights = torch.tensor([[e - 1], [-1]], device="cuda"), torch.ones(2, 1, device="cuda")
    got = arc.moe(x, w_in, w_out, ids, weights)
    w = torch.cat((small_in[30:32], small_in[62:]))[None]
    want, bound = moe_reference(x[:1], w, small_out.T.contiguous()[None], torch.zeros_like(ids[:1]), weights[:1], "silu")
    assert_within(got[:1], want, bound, "the last expert")
    assert (got[1] == 0).all()


def test_two_streams_at_once(cuda_device):
    calls = [_inputs(4, 2, 8, 512, 256, seed=1), _inputs(70, 4, 8, 512, 256, seed=2), _inputs(4, 2, 8, 512, 256, kind="int4")]
    want = [arc.moe(*v) for v in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for turn in range(10):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(((turn + j) % 3, arc.moe(*calls[(turn + j) % 3])))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[j]) for j, v in got) and arc.device_status(0) == 0


def test_strides_and_out(cuda_device):
    g = torch.Generator().manual_seed(3)
    x, w_in, w_out, ids, weights = _inputs(6, 2, 5, 72, 40, seed=1)
    want, bound = moe_reference(x, w_in, w_out, ids, weights, "silu")
    wide = normal(g, 6, 200)
    wide[:, 8:80] = x
    win = normal(g, 7, 90, 88)
    win[1:6, :80, 8:80] = w_in
    wout = normal(g, 5, 80, 56)
    wout[:, 4:76, 16:56] = w_out
    buf = torch.full((6, 100), 3.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, 5:77]
    ids_t = ids.T.contiguous().T
    got = arc.moe(wide[:, 8:80], win[1:6, :80, 8:80], wout[:, 4:76, 16:56], ids_t, weights.T.contiguous().T, out=out)
    assert got is out
    assert_within(got, want, bound, "strided")
    assert (buf[:, :5] == 3).all() and (buf[:, 77:] == 3).all()
    # Rows that TMA cannot read are copied.
    odd = normal(g, 6, 75)
    odd[:, 1:73] = x
    assert_within(arc.moe(odd[:, 1:73], w_in.transpose(1, 2).contiguous().transpose(1, 2), w_out, ids, weights), want,
                  bound, "copied")
    # K that is no multiple of 8
    x3, w3 = x[:, :69], w_in[:, :, :69]
    _check((x3, w3, w_out, ids, weights), "silu")


def test_repeatable_and_independent_of_the_batch(cuda_device):
    args = _inputs(64, 4, 16, 512, 256, seed=9)
    first = arc.moe(*args)
    for _ in range(5):
        assert torch.equal(arc.moe(*args), first)


def test_captured_and_other_streams(cuda_device):
    a, b = _inputs(4, 2, 8, 256, 128, seed=1), _inputs(9, 3, 8, 512, 128, kind="int4", seed=2)
    want = [arc.moe(*v) for v in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [arc.moe(*v) for v in (a, b)]
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(on_side, want):
        assert torch.equal(u, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [arc.moe(*v) for v in (a, b, a)]
    for seed in (5, 6):
        fresh = _inputs(4, 2, 8, 256, 128, seed=seed)
        a[0].copy_(fresh[0]), a[3].copy_(fresh[3]), a[4].copy_(fresh[4])
        graph.replay()
        want = arc.moe(*a)
        assert torch.equal(captured[0], want) and torch.equal(captured[2], want)
        assert torch.equal(captured[1], arc.moe(*b))


def test_empty(cuda_device):
    x, w_in, w_out, ids, weights = _inputs(4, 2, 8, 64, 64)
    assert arc.moe(x[:0], w_in, w_out, ids[:0], weights[:0]).shape == (0, 64)
    out = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda")
    assert (arc.moe(x, w_in, w_out, ids[:, :0], weights[:, :0], out=out) == 0).all() and (out == 0).all()


def test_refusals(cuda_device):
    x, w_in, w_out, ids, weights = _inputs(4, 2, 8, 256, 128)
    q_in, q_out = _inputs(4, 2, 8, 256, 128, kind="int4")[1:3]
    for bad in (x.float(), x.cpu()):
        with pytest.raises((TypeError, ValueError)):
            arc.moe(bad, w_in, w_out, ids, weights)
    for args in ((x[:, :128], w_in, w_out, ids, weights), (x, w_in[:7], w_out, ids, weights),
                 (x, w_in[:, :200], w_out, ids, weights), (x, w_in, w_out, ids[:3], weights),
                 (x, w_in, w_out, ids, weights[:, :1]), (x, w_in, q_out, ids, weights), (x, q_in, w_out, ids, weights),
                 (x, (q_in[0], q_in[1][:, :, :1]), q_out, ids, weights), (x, w_in, w_out, ids.cpu(), weights),
                 (x, w_in[0], w_out, ids, weights)):
        with pytest.raises(ValueError):
            arc.moe(*args)
    for args in ((x, w_in, w_out, ids.to(torch.int16), weights), (x, w_in, w_out, ids, weights.half()),
                 (x, w_in.half(), w_out, ids, weights)):
        with pytest.raises(TypeError):
            arc.moe(*args)
    with pytest.raises(ValueError):
        arc.moe(x, w_in, w_out, ids, weights, activation="tanh")
    big = _inputs(257, 1, 8, 256, 128)
    with pytest.raises(ValueError, match="at most"):
        arc.moe(*big)
    with pytest.raises(ValueError, match="overlap"):
        arc.moe(x, w_in, w_out, ids, weights, out=x)
    with pytest.raises(ValueError):
        arc.moe(x, w_in, w_out, ids, weights, out=torch.empty(4, 255, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        arc.moe(x.clone().requires_grad_(), w_in, w_out, ids, weights)
    with torch.no_grad():
        arc.moe(x.clone().requires_grad_(), w_in, w_out, ids, weights)


def test_beside_the_grouped_products(cuda_device):
    """The layer put together from group_rows and grouped_matmul, with h rounded in between, agrees."""
    t, top, e, k, i = 48, 4, 16, 256, 128
    x, w_in, w_out, ids, weights = _inputs(t, top, e, k, i, seed=4)
    offsets, rows, positions = arc.group_rows(ids, e)
    z = arc.grouped_matmul(x[rows.long()], w_in, offsets).float()
    h = (torch.nn.functional.silu(z[:, :i]) * z[:, i:]).to(torch.bfloat16)
    ys = arc.grouped_matmul(h, w_out, offsets).float()
    y = (ys[positions.long()] * weights[..., None]).sum(1)
    got = arc.moe(x, w_in, w_out, ids, weights).float()
    # the composition rounds z and ys as well: five roundings of at most 2^-8 each, of terms that partly cancel
    assert (got - y).norm() <= 5 * 2.0 ** -8 * y.norm()
