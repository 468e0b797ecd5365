"""arc.moe and arc.lora_linear on the B200: what their documentation promises beyond the values themselves."""
from __future__ import annotations

import pytest
import torch

import arc
from arc import _lib
from int4_bounds import moe_int4_linear
from linear_bounds import assert_within, normal
from moe_reference import moe_reference
from test_gpu_lora import reference as lora_reference

pytestmark = pytest.mark.gpu


def _cancelling_experts(g, kind, e, k, i, n):
    """Experts whose rows of w_in come twice and whose columns of w_out come twice with opposite signs: every result is zero but for
    the rounding of its sums, so that a sum's error is all that shows."""
    half = i // 2
    if kind == "bf16":
        rows, cols = normal(g, e, 2, half, k, scale=k ** -0.5), normal(g, e, n, half, scale=i ** -0.5)
        return torch.cat((rows, rows), 2).flatten(1, 2), torch.cat((cols, -cols), 2)
    codes, signed = torch.randint(-8, 8, (e, 2, half, k), generator=g), torch.randint(-7, 8, (e, n, half), generator=g)
    codes, signed = torch.cat((codes, codes), 2).flatten(1, 2), torch.cat((signed, -signed), 2)

    def pack(c, scale):
        c = (c & 15).to(torch.uint8)
        return (c[..., 0::2] | c[..., 1::2] << 4).cuda(), torch.full((e, c.shape[1], c.shape[2] // 128), scale,
                                                                    dtype=torch.bfloat16, device="cuda")

    return pack(codes, 0.2 * k ** -0.5), pack(signed, 0.2 * i ** -0.5)


# Contractions of 6 and 10 boxes, 7 and 5, 3 and 3: no multiple of the four parts that share them, nor of the blocks of a
# cluster. 6 tokens are sorted by one warp, 40 by eight.
@pytest.mark.parametrize("kind,k,i", [("bf16", 328, 584), ("int4", 896, 640), ("int4", 384, 384)])
@pytest.mark.parametrize("t", [6, 40])
@pytest.mark.parametrize("splits,ordered", [(None, None), (1, 0), (2, 1), (4, 0), (8, 1)])
def test_a_token_beside_others(cuda_device, monkeypatch, kind, k, i, t, splits, ordered):
    """One token's row, choices and weights beside different tokens and in different rows: the same bits for the same
    batch, and within the error of its sums in every one, under each plan."""
    g = torch.Generator().manual_seed(t + k)
    e, top, n = 11, 3, 392
    w_in, w_out = _cancelling_experts(g, kind, e, k, i, n)
    x1, weights1, ids1 = normal(g, 1, k), torch.rand(1, top, generator=g).cuda(), torch.tensor([[7, 2, 10]], device="cuda")
    want, bound = moe_reference(x1, w_in, w_out, ids1, weights1, "silu")
    for columns in (8, 16) if splits else (0,):
        if splits:
            monkeypatch.setenv("ARC_EXPERT_PLAN", f"{columns}:{splits}:{ordered}")
        for turn in range(6):
            x, weights = normal(g, t, k), torch.rand(t, top, generator=g).cuda()
            ids = torch.rand(t, e, generator=g).topk(top, dim=1).indices.cuda()
            if turn == 1:
                ids[:] = -1  # nobody else chooses
            elif turn == 2:
                ids[:] = ids1.flip(1)  # the same experts: several passes of each
            elif turn == 3:
                ids[:, 0] = 2  # a popular one in front of the other two
            row = (0, 1, t - 1)[turn % 3]
            x[row], weights[row], ids[row] = x1[0], weights1[0], ids1[0]
            got = arc.moe(x, w_in, w_out, ids, weights)
            assert torch.equal(arc.moe(x, w_in, w_out, ids, weights), got)
            assert_within(got[row:row + 1], want, bound, (columns, turn))
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("t,kind,ordered", [(4, "bf16", 0), (4, "bf16", 1), (40, "bf16", 1), (4, "int4", 0), (40, "int4", 1)])
def test_experts_read_what_was_written_just_before(cuda_device, monkeypatch, t, kind, ordered):
    """Everything that a call reads is written by the launch in front of it, over other values that a call before has read: in a
    graph, where nothing but the order of launches stands between them."""
    monkeypatch.setenv("ARC_EXPERT_PLAN", f"8:2:{ordered}")
    g = torch.Generator().manual_seed(t)

    def values():
        ids = torch.rand(t, 9, generator=g).topk(2, dim=1).indices.cuda()
        w_in, w_out = _cancelling_experts(g, kind, 9, 512, 256, 264)
        flat = [*w_in, *w_out] if kind == "int4" else [w_in, w_out]
        return [normal(g, t, 512), ids, torch.rand(t, 2, generator=g).cuda(), *(v.clone() for v in flat)]

    def call(x, ids, weights, *w):
        w = (w[:2], w[2:]) if kind == "int4" else w
        return arc.moe(x, *w, ids, weights)

    sets = [values() for _ in range(4)]
    want = [call(*v) for v in sets]
    torch.cuda.synchronize()
    for last in range(len(sets[0])):  # whose copy comes last, directly in front of the call
        at = [v.clone() for v in sets[0]]
        order = [i for i in range(len(at)) if i != last] + [last]
        call(*at)
        graph = torch.cuda.CUDAGraph()
        got = []
        with torch.cuda.graph(graph):
            for v in sets * 3:
                for i in order:
                    at[i].copy_(v[i])
                got.append(call(*at))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[j % 4]) for j, y in enumerate(got)), last
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("m,plan", [(9, "16:2"), (150, "128:1"), (300, "pair:1"), (300, "pair:2")])
def test_adapters_read_what_was_written_just_before(cuda_device, monkeypatch, m, plan):
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    g = torch.Generator().manual_seed(m)
    n, k, r, count = 264, 520, 24, 5

    def values():
        return [normal(g, m, k), normal(g, n, k, scale=k ** -0.5), normal(g, count, r, k, scale=k ** -0.5),
                normal(g, count, n, r, scale=r ** -0.5), torch.randint(-1, count, (m,), generator=g).cuda(), normal(g, n),
                normal(g, m, n), torch.rand(count, generator=g).cuda()]

    def call(x, w, a, b, ids, bias, residual, scales):
        return arc.lora_linear(x, w, a, b, ids, bias, residual, scales=scales, activation="silu")

    sets = [values() for _ in range(4)]
    want = [call(*v) for v in sets]
    torch.cuda.synchronize()
    for last in range(len(sets[0])):
        at = [v.clone() for v in sets[0]]
        order = [i for i in range(len(at)) if i != last] + [last]
        call(*at)
        graph = torch.cuda.CUDAGraph()
        got = []
        with torch.cuda.graph(graph):
            for v in sets * 3:
                for i in order:
                    at[i].copy_(v[i])
                got.append(call(*at))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[j % 4]) for j, y in enumerate(got)), last
    assert arc.device_status(0) == 0


def _int4(g, e, n, k):
    packed = torch.randint(0, 256, (e, n, k // 2), generator=g, dtype=torch.uint8).cuda()
    return packed, ((0.5 + torch.rand(e, n, k // 128, generator=g)) * (0.2 * k ** -0.5)).to(torch.bfloat16).cuda()


def _int4_layer(g, t, top=2, e=6, k=256, i=128):
    x, w_in, w_out = normal(g, t, k), _int4(g, e, i, k), _int4(g, e, k, i)
    ids = torch.rand(t, e, generator=g).topk(top, dim=1).indices.cuda()
    return x, w_in, w_out, ids, torch.rand(t, top, generator=g).cuda()


def _within_int4(args, what):
    want, bound = moe_int4_linear(*args)
    assert_within(arc.moe(*args, activation=None), want, bound, what)
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("t", [3, 30])
@pytest.mark.parametrize("power", [-90, -80, -70, -64, -60, -57, -30, 0, 40, 55])
def test_int4_over_its_range(cuda_device, power, t):
    """Activations down to where products of codes leave fp32's range: what is lost there is 2^-80 a product, no more."""
    args = _int4_layer(torch.Generator().manual_seed(power + 200), t)
    args[0].mul_(2.0 ** power)
    _within_int4(args, power)


@pytest.mark.parametrize("t", [3, 30])
@pytest.mark.parametrize("power", [7, 14, 30, 60])
def test_int4_outliers_on_zero_codes(cuda_device, power, t):
    """A large activation whose codes are 0, and rows of zero codes: its 8 x cancels but for the rounding of the group's sum."""
    x, w_in, w_out, ids, weights = _int4_layer(torch.Generator().manual_seed(power), t)
    x[:, 5] = 1.4 * 2.0 ** power
    w_in[0][:, :, 2] &= 0x0F  # code 5 of every row: the high nibble of byte 2
    w_in[0][:, 7], w_out[0][:, 9] = 0, 0
    _within_int4((x, w_in, w_out, ids, weights), power)


def _adapter_layer(g, m, n, k, r, count, runs=0):
    x, w = normal(g, m, k), normal(g, n, k, scale=k ** -0.5)
    a, b = normal(g, count, r, k, scale=k ** -0.5), normal(g, count, n, r, scale=r ** -0.5)
    if runs:
        cuts = torch.randint(0, m + 1, (runs - 1,), generator=g).sort().values.tolist()
        owner = torch.randint(-1, count, (runs,), generator=g)
        ids = torch.repeat_interleave(owner, torch.tensor([q - p for p, q in zip([0] + cuts, cuts + [m])]))
    else:
        ids = torch.randint(-1, count, (m,), generator=g)
    return x, w, a, b, ids.cuda(), normal(g, n), normal(g, m, n), (0.25 + torch.rand(count, generator=g)).cuda()


def _within_adapters(args, act, what):
    want, bound = lora_reference(*args, act)
    got = arc.lora_linear(*args[:7], scales=args[7], activation=act)
    assert_within(got, want, bound, what)
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("plan", ["pair:1", "pair:2", "pair128:1", "pair128:2"])
@pytest.mark.parametrize("r", [33, 64, 65, 100, 128, 136, 192, 200, 256])
def test_ranks_of_several_blocks_by_pairs(cuda_device, monkeypatch, plan, r):
    """The adapters' part of the contraction as one to four blocks of 64 for each adapter, the last one whole or not, in row tiles
    of one adapter and of all five."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    g = torch.Generator().manual_seed(r)
    _within_adapters(_adapter_layer(g, 300, 264, 200, r, 5), "silu", "mixed")
    _within_adapters(_adapter_layer(g, 530, 520, 136, r, 5, runs=4), None, "prompts")


@pytest.mark.parametrize("plan", ["pair:1", "pair128:1"])
@pytest.mark.parametrize("r,count,runs", [(16, 12, 0), (72, 3, 0), (32, 9, 40), (256, 4, 9)])
def test_pairs_that_walk_over_tiles(cuda_device, monkeypatch, plan, r, count, runs):
    """Several tiles a pair, each with its own list of adapters."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    _within_adapters(_adapter_layer(torch.Generator().manual_seed(r), 2100, 5000, 72, r, count, runs), "gelu", plan)


@pytest.mark.parametrize("m,n,k", [(2048, 2048, 256), (1500, 1500, 512)])
def test_pairs_by_their_own_plan(cuda_device, m, n, k):
    assert "pair" in arc.kernel_name(_lib.OP_LINEAR, m, n, k)
    _within_adapters(_adapter_layer(torch.Generator().manual_seed(m), m, n, k, 128, 6, runs=7), "relu", (m, n, k))


@pytest.mark.parametrize("t,top,e,k,i,n", [(1, 1, 1, 1, 1, 1), (3, 2, 2, 1, 9, 2), (9, 1, 3, 65, 1, 7), (256, 1, 1, 8, 8, 1), (256, 16, 1024, 3, 2, 5)])
@pytest.mark.parametrize("gated", [True, False])
def test_smallest_experts(cuda_device, t, top, e, k, i, n, gated):
    g = torch.Generator().manual_seed(t)
    w_in, w_out = normal(g, e, 2 * i if gated else i, k), normal(g, e, n, i)
    ids = torch.rand(t, e, generator=g).topk(top, dim=1).indices.cuda()
    args = (normal(g, t, k), w_in, w_out, ids, torch.rand(t, top, generator=g).cuda())
    want, bound = moe_reference(*args, "gelu")
    assert_within(arc.moe(*args, activation="gelu"), want, bound, (t, k, i, n))
    assert arc.device_status(0) == 0


@pytest.mark.parametrize("m,n,k,r,count,runs", [(1, 1, 1, 1, 1, 0), (2, 3, 1, 1, 2, 0), (129, 1, 9, 2, 3, 2), (40000, 72, 64, 8, 1024, 0),
                                               (40000, 520, 64, 24, 50, 300)])
def test_smallest_and_longest_adapters(cuda_device, m, n, k, r, count, runs):
    _within_adapters(_adapter_layer(torch.Generator().manual_seed(m), m, n, k, r, count, runs), "silu", (m, n, k, r))


def test_serving_operators_beside_others_on_streams(cuda_device):
    """Kernels with TMEM, clusters and early launches of several operators at once, each with the bits of its call alone."""
    g = torch.Generator().manual_seed(3)
    small, large = _adapter_layer(g, 40, 520, 512, 24, 6), _adapter_layer(g, 2048, 2048, 256, 72, 6, runs=7)
    e_in, e_out = normal(g, 9, 512, 512, scale=512 ** -0.5), normal(g, 9, 512, 256, scale=256 ** -0.5)
    x, ids, weights = normal(g, 40, 512), torch.rand(40, 9, generator=g).topk(3, dim=1).indices.cuda(), torch.rand(40, 3).cuda()
    a, b = normal(g, 1024, 512), normal(g, 1024, 512)
    calls = [lambda: arc.lora_linear(*small[:7], scales=small[7]), lambda: arc.lora_linear(*large[:7], scales=large[7]),
             lambda: arc.moe(x, e_in, e_out, ids, weights), lambda: arc.matmul(a, b), lambda: arc.linear(a, b, activation="gelu")]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for turn in range(20):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                i = (turn + j) % len(calls)
                got.append((i, calls[i]()))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want[i]) for i, v in got) and arc.device_status(0) == 0
