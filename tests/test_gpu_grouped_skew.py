"""GPU: s2_grouped_linear where a router sends most rows to few groups."""
import pytest
import torch

from tests import operator_oracles as oracles

pytestmark = pytest.mark.gpu


def _operands(groups, rows, n, k):
    gen = torch.Generator(device="cuda").manual_seed(groups + rows)
    a = torch.randn(rows, k, device="cuda", generator=gen).bfloat16()
    w = torch.randn(groups, n, k, device="cuda", generator=gen).mul_(k**-0.5).bfloat16()
    return a, w


def _offsets(groups, rows, hot):
    """hot: {group: rows}; the others share what is left, some of them nothing."""
    left = rows - sum(hot.values()) - rows // 50  # the last rows belong to no group
    sizes = [hot.get(g, 0) for g in range(groups)]
    cold = [g for g in range(groups) if g not in hot]
    for i in range(left):
        sizes[cold[(i * 7) % len(cold)]] += 1
    off = [0]
    for s in sizes:
        off.append(off[-1] + s)
    return off


LAYOUTS = [(64, 512, {31: 512}), (64, 512, {0: 200, 63: 250}), (1024, 4000, {700: 3000}), (40, 300, {32: 250}),
           (33, 270, {32: 260}), (16, 250, {3: 129, 4: 65, 5: 1}), (100, 3200, {17: 1500, 18: 17, 99: 1200}), (1, 16, {})]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("form", [(136, 200, "gelu_tanh", "bf16"), (259, 1000, "none", "f32")], ids=lambda f: f[2])
def test_each_row_once(s2lib, gpu_ctx, layout, form):
    groups, rows, hot = layout
    n, k, act, out = form
    off = _offsets(groups, rows, hot) if groups > 1 else [0, rows]
    a, w = _operands(groups, rows, n, k)
    bias = torch.randn(groups, n, device="cuda")
    before = torch.randn(rows, n, device="cuda").to(torch.float32 if out == "f32" else torch.bfloat16)
    got = before.clone()
    s2lib.grouped_linear(gpu_ctx, a, w, torch.tensor(off, dtype=torch.int32, device="cuda"), bias,
                         act=oracles.ACTS.index(act), out=got)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.grouped_linear(a, w, off, bias, act, None, None, got.dtype, before))


def _time(ctx, call):
    """us of one call, replayed."""
    call()
    torch.cuda.synchronize()
    graph, home = torch.cuda.CUDAGraph(), ctx.stream
    with torch.cuda.graph(graph):
        ctx.set_stream(torch.cuda.current_stream())
        for _ in range(5):
            call()
    ctx.set_stream(home)
    times = []
    for _ in range(5):
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end) * 200)
    del graph
    return min(times)


@pytest.mark.parametrize("case", [(64, 512, 2048, 1024), (1024, 8192, 512, 512), (32, 256, 2560, 2560)], ids=str)
def test_one_hot_group_costs_no_more_than_all_groups(s2lib, gpu_ctx, case):
    """All rows in one group against the same rows spread over all groups, which reads every weight: one group's row
    tiles run side by side, so that it may take 1.8 times as long at most (it took 2.3 to 18 times as long where a group's
    tiles ran one after another; now 0.4 to 1.2)."""
    groups, rows, n, k = case
    a, w = _operands(groups, rows, n, k)
    out = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    half = groups // 2
    hot = torch.tensor([0] * (half + 1) + [rows] * (groups - half), dtype=torch.int32, device="cuda")
    even = torch.tensor([i * rows // groups for i in range(groups + 1)], dtype=torch.int32, device="cuda")
    one = _time(gpu_ctx, lambda: s2lib.grouped_linear(gpu_ctx, a, w, hot, out=out))
    all_ = _time(gpu_ctx, lambda: s2lib.grouped_linear(gpu_ctx, a, w, even, out=out))
    assert one < 1.8 * all_, (one, all_)
