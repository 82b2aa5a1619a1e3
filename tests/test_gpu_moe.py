"""Routing to experts and combining their rows against 64 bits.

Bounds, with u = 2^-24 (half a step of fp32).  A weight: exp is off by at most 2 u and its argument, a difference below 2^7 in size, by 2^7 u, which moves exp by
2^7 u of itself; sums of up to 16 (weights) or 1024 (softmax, added in 64 bits) terms, two quotients and a product add less than 24 u: 2^8 u = 2^-16
in all, and an absolute 2^-120 where fp32 ends.  A combined value: a term, a product and an addition, is off by (terms + 1) u of the magnitudes' sum; then
half a step of the result's type, which of fp16 is at least 2^-25 (subnormals)."""
import pytest
import torch

import moe_reference as ref
from nnfusion_amd import ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _check_route(gpu, logits, k, **kw):
    on = {n: v.to(gpu) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    got = ops.moe_route(logits.to(gpu), k, **on)
    want = ref.route(logits, k, **kw)
    for name, g, w in zip(("experts", "rows", "offsets", "positions"), got[1:], want[1:]):
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), w), name
    off = (got[0].cpu().double() - want[0]).abs()
    assert got[0].dtype == torch.float32 and bool((off <= 2.0 ** -16 * want[0].abs() + 2.0 ** -120).all()), off.max()
    return got


@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (1, 8, 2), (3, 60, 4), (64, 64, 6), (65, 64, 16), (33, 65, 8), (64, 128, 8), (17, 129, 3), (70, 256, 8), (5, 257, 8),
                                        (64, 512, 10), (130, 513, 16), (9, 1024, 16), (66, 1024, 1), (1000, 16, 2), (700, 100, 5)])
@pytest.mark.parametrize("type", [torch.float32, torch.float16, torch.bfloat16])
def test_softmax(gpu, tokens, n, k, type):
    logits = (2 * torch.randn((tokens, n), generator=_gen(tokens + n))).to(type)
    _check_route(gpu, logits, k, renormalize=tokens % 2 == 0, scale=1.0 if tokens % 3 else 2.5)


@pytest.mark.parametrize("tokens,n,k,groups,top_groups,group_top", [
    (1, 256, 8, 8, 4, 2), (70, 256, 8, 8, 4, 2), (65, 160, 6, 8, 3, 1), (64, 64, 4, 4, 1, 2), (5, 60, 3, 15, 2, 2), (9, 16, 1, 16, 1, 1), (67, 512, 8, 16, 5, 2), (3, 1024, 16, 2, 1, 2),
    (80, 384, 8, 1, 1, 1), (33, 72, 7, 9, 9, 1)])
@pytest.mark.parametrize("score,with_bias", [("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)])
def test_groups_and_bias(gpu, tokens, n, k, groups, top_groups, group_top, score, with_bias):
    gen = _gen(tokens * n)
    logits = 1.5 * torch.randn((tokens, n), generator=gen)
    bias = 0.1 * torch.randn((n,), generator=gen) if with_bias else None
    _check_route(gpu, logits, k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top, scale=2.5)


@pytest.mark.parametrize("tokens", [7, 100])
def test_ties_go_to_the_lowest_index(gpu, tokens):
    for n, k in ((8, 8), (128, 16), (600, 9)):
        _check_route(gpu, torch.zeros((tokens, n)), k)
        _check_route(gpu, torch.randint(-1, 2, (tokens, n), generator=_gen(n)).half(), k)
        # -0 and 0 are one number
        _check_route(gpu, torch.where(torch.rand((tokens, n), generator=_gen(n)) < 0.5, -0.0, 0.0), k)
        _check_route(gpu, torch.zeros((tokens, n)), min(k, n // 4), score="sigmoid", bias=torch.zeros(n), groups=4, top_groups=2, group_top=2)


def test_sums_closer_than_fp32_can_tell_are_compared_in_64_bits(gpu):
    """Scores saturated in fp32 (sigmoid of 18 .. 30: 1 - 1.5e-8 .. 1 - 1e-13), biases that differ by less than a rounding, and biases that make up for the scores'
    differences to the last bits."""
    gen = _gen(5)
    logits = 18 + 12 * torch.rand((40, 64), generator=gen)
    _check_route(gpu, logits, 8, score="sigmoid", bias=torch.zeros(64))
    _check_route(gpu, logits, 8, score="sigmoid", bias=1.0 + torch.zeros(64), groups=8, top_groups=3, group_top=2)
    _check_route(gpu, logits, 8, score="sigmoid", groups=8, top_groups=3, group_top=2)
    logits = torch.randn((1, 64), generator=gen).repeat(100, 1)
    level = (1.0 - torch.sigmoid(logits[0].double())).float()
    _check_route(gpu, logits, 8, score="sigmoid", bias=level)
    _check_route(gpu, logits, 8, bias=(0.5 - torch.softmax(logits[0].double(), 0)).float())
    _check_route(gpu, logits, 8, bias=1e6 * torch.ones(64))


@pytest.mark.parametrize("tokens", [3, 200, 5000])
def test_large_biases_that_cancel(gpu, tokens):
    """A group's two best sums are 1000 and -1000 and something: what decides is far below their rounding."""
    gen = _gen(tokens)
    n = 32
    logits = torch.randn((min(tokens, 200), n), generator=gen)
    bias = torch.tensor([1000.0, -1000.0] * (n // 2)) + 2.0 ** -12 * torch.randn((n,), generator=gen)
    for kw in (dict(groups=16, top_groups=5, group_top=2), dict(groups=16, top_groups=5, group_top=1), dict()):
        for score in ("softmax", "sigmoid"):
            want = ref.route(logits, 3, score=score, bias=bias, **kw)
            x = logits[torch.arange(tokens) % len(logits)]
            got = ops.moe_route(x.to(gpu), 3, score=score, bias=bias.to(gpu), **kw)
            assert torch.equal(got[1].cpu(), want[1][torch.arange(tokens) % len(logits)])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [12, 77])
def test_masked_experts(gpu, score, tokens):
    """-inf and NaN: last choice and weight 0, rows that leave nothing among them; +inf the largest number."""
    gen = _gen(tokens)
    n = 48
    logits = torch.randn((tokens, n), generator=gen)
    for value in (float("-inf"), float("nan"), torch.finfo(torch.float32).min):
        x = torch.where(torch.rand((tokens, n), generator=gen) < 0.9, torch.full_like(logits, value), logits)
        x[0] = value
        x[1, :3] = float("inf")
        x[2] = float("inf")
        x[3, 7] = -value
        bias = torch.randn((n,), generator=gen)
        bias[5], bias[6], bias[9] = float("-inf"), float("nan"), 1e30
        for kw in ({}, {"bias": bias}, {"groups": 6, "top_groups": 2, "group_top": 2}, {"groups": 6, "top_groups": 2, "group_top": 1, "bias": bias}, {"renormalize": False},
                   {"groups": 6, "top_groups": 3, "group_top": 2, "bias": bias}):
            _check_route(gpu, x, 6, score=score, **kw)


@pytest.mark.parametrize("total,live", [(5, 0), (5, 3), (64, 1), (64, 64), (65, 0), (300, 1), (300, 117), (300, 300), (300, 301), (300, -1), (4, 9)])
def test_tokens_that_are_not_there(gpu, total, live):
    logits = torch.randn((total, 40), generator=_gen(total))
    logits[max(0, live):] = float("nan")
    _check_route(gpu, logits, 3, tokens=torch.tensor([live], dtype=torch.int32))
    _check_route(gpu, logits, 3, score="sigmoid", bias=torch.zeros(40), tokens=torch.tensor(live, dtype=torch.int32))


def _sorted_order(experts, n):
    """rows, offsets, positions of a choice, by a stable sort"""
    flat = experts.flatten().long()
    order = torch.sort(flat, stable=True)[1]
    positions = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel()))
    offsets = torch.nn.functional.pad(torch.bincount(flat, minlength=n).cumsum(0), (1, 0))
    return (order // experts.shape[1]).int(), offsets.int(), positions.view_as(experts).int()


@pytest.mark.parametrize("tokens,n,k", [(4096, 8, 2), (4097, 256, 8), (20000, 60, 4), (70000, 1024, 16), (65, 2, 2), (5000, 1, 1)])
def test_the_order_of_many(gpu, tokens, n, k):
    logits = torch.randn((tokens, n), generator=_gen(n))
    logits[:, : max(1, n // 8)] += 2  # some are met much more often
    weights, experts, rows, offsets, positions = [t.cpu() for t in ops.moe_route(logits.to(gpu), k)]
    assert torch.equal(experts.long(), torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k])
    for got, want in zip((rows, offsets, positions), _sorted_order(experts, n)):
        assert torch.equal(got, want)
    assert bool((weights.double().sum(1) - 1).abs().max() < 2.0 ** -18)  # 16 of them, each rounded twice


@pytest.mark.parametrize("tokens", [9, 2048, 2049, 4500])
@pytest.mark.parametrize("n,k,groups,top_groups,group_top,score,with_bias", [(257, 8, 1, 1, 1, "softmax", False), (300, 16, 3, 2, 2, "softmax", True), (512, 10, 16, 4, 2, "sigmoid", True),
                                                                             (480, 5, 8, 3, 1, "softmax", False), (513, 7, 1, 1, 1, "sigmoid", True)])
def test_more_than_256_experts(gpu, tokens, n, k, groups, top_groups, group_top, score, with_bias):
    gen = _gen(tokens + n)
    x = 1.5 * torch.randn((tokens, n), generator=gen)
    x[::7, ::5] = float("-inf")
    bias = 0.05 * torch.randn((n,), generator=gen) if with_bias else None
    _check_route(gpu, x, k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top)


@pytest.mark.parametrize("tokens,n,k,groups,top_groups,group_top,score,type", [
    (8192, 256, 8, 8, 4, 2, "sigmoid", torch.float32), (8192, 128, 6, 16, 3, 2, "softmax", torch.float16), (6000, 512, 10, 16, 4, 1, "sigmoid", torch.bfloat16)])
def test_groups_of_many_tokens(gpu, tokens, n, k, groups, top_groups, group_top, score, type):
    """So many that some groups' sums and some experts' lie closer than fp32 can tell"""
    gen = _gen(n)
    logits = (1.5 * torch.randn((tokens, n), generator=gen)).to(type)
    bias = 0.05 * torch.randn((n,), generator=gen) if score == "sigmoid" else None
    _check_route(gpu, logits, k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top)


def test_skewed_to_one_expert(gpu):
    logits = torch.zeros((3000, 256))
    logits[:, 200] = 5
    _check_route(gpu, logits[:90], 2)
    _, experts, rows, offsets, _ = [t.cpu() for t in ops.moe_route(logits.to(gpu), 1)]
    assert bool((experts == 200).all()) and torch.equal(rows, torch.arange(3000).int()) and offsets[200] == 0 and offsets[201] == 3000


def test_results_go_where_the_caller_says_and_nowhere_else(gpu):
    tokens, n, k = 100, 24, 3
    logits = torch.randn((tokens + 1, n), generator=_gen(3)).to(gpu)[1:]  # (rows of 96 bytes: the base is not on 16 ..)
    odd = torch.randn((tokens * 25 + 1,), generator=_gen(4)).half().to(gpu)[1:].view(tokens, 25)  # (.. and here not on 4)
    for x in (logits, odd):
        n = x.shape[1]
        guard = 64
        buffers = [torch.full((size + 2 * guard,), -77, dtype=torch.int32, device=gpu) for size in (tokens * k, tokens * k, tokens * k, n + 1, tokens * k)]
        inner = [b[guard:-guard] for b in buffers]
        out = (inner[0].view(torch.float32).view(tokens, k), inner[1].view(tokens, k), inner[2], inner[3], inner[4].view(tokens, k))
        work = torch.empty(ops.moe_route_workspace_bytes(tokens, n, k), dtype=torch.uint8, device=gpu)
        got = ops.moe_route(x, k, out=out, workspace=work)
        for g, o, b, want in zip(got, out, buffers, ops.moe_route(x, k)):
            assert g is o and torch.equal(g, want)
            assert bool((b[:guard] == -77).all()) and bool((b[-guard:] == -77).all())


@pytest.mark.parametrize("tokens", [48, 500])
def test_captured_and_replayed(gpu, tokens):
    n, k = 96, 4
    logits, live = torch.zeros((tokens, n), device=gpu), torch.zeros((1,), dtype=torch.int32, device=gpu)
    x = torch.randn((tokens * k, 64), generator=_gen(8)).half().to(gpu)
    ops.moe_route(logits, k, tokens=live)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        routed = ops.moe_route(logits, k, score="sigmoid", tokens=live)
        y = ops.moe_combine(x, routed[0], routed[4])
    for seed, there in ((1, tokens), (2, 5), (3, 0), (4, tokens - 1)):
        logits.copy_(torch.randn((tokens, n), generator=_gen(seed)))
        live.fill_(there)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.moe_route(logits, k, score="sigmoid", tokens=live)
        for g, w in zip(routed, want):
            assert torch.equal(g, w)
        assert torch.equal(y, ops.moe_combine(x, want[0], want[4]))


def test_on_another_stream(gpu):
    logits = torch.randn((300, 128), generator=_gen(1)).to(gpu)
    want = ops.moe_route(logits, 8)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = ops.moe_route(logits, 8)
    stream.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_two_graphs_and_another_stream_at_once(gpu):
    """Each call with results and a workspace of its own, as torch's allocator gives it"""
    gens = [torch.randn((tokens, n), generator=_gen(20 + n)).to(gpu) for tokens, n in ((700, 64), (300, 128), (2000, 60))]
    want = [ops.moe_route(x, 6) for x in gens]
    graphs = []
    for x in gens[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.moe_route(x, 6)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for (graph, out), stream in zip(graphs, streams):
            for t in out:
                t.fill_(-5)
            stream.wait_stream(torch.cuda.current_stream())
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = ops.moe_route(gens[2], 6)
        torch.cuda.synchronize()
        for got, w in zip([g[1] for g in graphs] + [eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_a_workspace_that_two_calls_share_at_once_leads_nowhere_else(gpu):
    """What such calls give is not defined, but they write only where their results are."""
    tokens, n, k, guard = 3000, 200, 8, 4096
    sizes = [(tokens, k), (tokens, k), (tokens * k,), (n + 1,), (tokens, k)]
    workspace = torch.zeros(ops.moe_route_workspace_bytes(tokens, n, k), dtype=torch.uint8, device=gpu)
    calls = []
    for seed in (1, 2):
        buffers, out = [], []
        for i, size in enumerate(sizes):
            count = torch.Size(size).numel()
            b = torch.full((count + 2 * guard,), -77, dtype=torch.float32 if i == 0 else torch.int32, device=gpu)
            buffers.append(b)
            out.append(b[guard : guard + count].view(size))
        # (all pairs on a few experts here, on other ones there)
        logits = 4 * torch.randn((tokens, n), generator=_gen(seed)) + torch.where(torch.arange(n) // 16 == seed, 20.0, 0.0)
        calls.append((logits.to(gpu), tuple(out), buffers, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for logits, out, _, stream in calls:
            with torch.cuda.stream(stream):
                ops.moe_route(logits, k, out=out, workspace=workspace)
    torch.cuda.synchronize()
    for logits, out, buffers, _ in calls:
        for b in buffers:
            assert bool((b[:guard] == -77).all()) and bool((b[-guard:] == -77).all())
        for got, want in zip(ops.moe_route(logits, k, out=out, workspace=workspace), ops.moe_route(logits, k)):  # (one at a time they are right)
            assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [0, 5])
def test_nothing_to_do_is_refused(gpu, tokens):
    logits = torch.zeros((tokens, 8 if tokens == 0 else 0), device=gpu)
    with pytest.raises((RuntimeError, AssertionError)):
        ops.moe_route(logits, 2)
    with pytest.raises(RuntimeError):
        ops.moe_combine(torch.zeros((0, 64), dtype=torch.float16, device=gpu), torch.zeros((tokens, 2), device=gpu), torch.zeros((tokens, 2), dtype=torch.int32, device=gpu))


def _check_combine(gpu, x, weights, positions, residual=None, out=None):
    got = ops.moe_combine(x.to(gpu), weights.to(gpu), positions.to(gpu), None if residual is None else residual.to(gpu), out)
    want, size = ref.combine(x, weights, positions, residual)
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + (weights.shape[1] + 2) * 2.0 ** -24 * size * (1 + torch.finfo(x.dtype).eps) + 2.0 ** -25
    assert got.dtype == x.dtype
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (off - bound).max()
    return got


@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (1, 8, 4096), (3, 2, 7), (5, 3, 512), (2, 16, 520), (33, 6, 1030), (64, 9, 513), (7, 4, 4099), (500, 8, 2048), (1, 2, 20000)])
@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_combine(gpu, tokens, k, n, type):
    gen = _gen(tokens + k + n)
    rows = tokens * k
    x = torch.randn((rows, n), generator=gen).to(type)
    weights, positions = torch.rand((tokens, k), generator=gen), torch.randperm(rows, generator=gen).int().view(tokens, k)
    residual = torch.randn((tokens, n), generator=gen).to(type)
    _check_combine(gpu, x, weights, positions)
    _check_combine(gpu, x, weights, positions, residual)


@pytest.mark.parametrize("n", [64, 61])
def test_combine_takes_nothing_from_rows_that_do_not_count(gpu, n):
    gen = _gen(n)
    x = torch.randn((12, n), generator=gen).half()
    x[3], x[5] = float("nan"), float("inf")
    weights, positions = torch.rand((4, 3), generator=gen), torch.tensor([[0, 1, -1], [-1, -1, -1], [3, 5, 2], [12, 2147483647, -2147483648]], dtype=torch.int32)
    weights[2, 0] = weights[2, 1] = 0
    weights[0, 2] = float("nan")
    y = _check_combine(gpu, x, weights, positions)
    assert bool((y[1] == 0).all()) and bool((y[3] == 0).all())
    # the same row twice; an infinity that counts
    y = _check_combine(gpu, x.clamp(-9, 9).nan_to_num(), weights.nan_to_num(1.0), torch.full((4, 3), 7, dtype=torch.int32))
    y = ops.moe_combine(x.to(gpu), torch.ones((1, 2), device=gpu), torch.tensor([[0, 5]], dtype=torch.int32, device=gpu))
    assert bool(torch.isinf(y).all())


def test_combine_in_place_and_off_16_bytes(gpu):
    gen = _gen(2)
    x, residual = torch.randn((20, 64), generator=gen).half(), torch.randn((10, 64), generator=gen).half()
    weights, positions = torch.rand((10, 2), generator=gen), torch.randperm(20, generator=gen).int().view(10, 2)
    want = ops.moe_combine(x.to(gpu), weights.to(gpu), positions.to(gpu), residual.to(gpu))
    y = residual.to(gpu)
    assert ops.moe_combine(x.to(gpu), weights.to(gpu), positions.to(gpu), y, y) is y and torch.equal(y, want)
    off = torch.empty(20 * 64 + 1, dtype=torch.float16, device=gpu)[1:].view(20, 64)
    off.copy_(x)
    guarded = torch.full((10 * 64 + 3,), 7.0, dtype=torch.float16, device=gpu)
    out = guarded[1:-2].view(10, 64)
    assert torch.equal(ops.moe_combine(off, weights.to(gpu), positions.to(gpu), residual.to(gpu), out), want)
    assert guarded[0] == 7 and bool((guarded[-2:] == 7).all())


def test_combine_beyond_32_bit_offsets(gpu):
    rows, n = (1 << 31) // 4096 + 3, 4096
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device=gpu)
    x[-1], x[-2] = 3, 5
    positions = torch.tensor([[rows - 1, rows - 2]], dtype=torch.int32, device=gpu)
    y = ops.moe_combine(x, torch.tensor([[1.0, 2.0]], device=gpu), positions)
    assert bool((y == 13).all())
