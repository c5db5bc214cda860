"""GPU: the group norm's clusters are sized for two CTAs a SM; a kernel whose registers leave room for one only would run
them in two waves."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _time(s2lib, ctx, x, out, calls=12):
    s2lib.group_norm(ctx, x, 32, act=s2lib.S2_ACT_SILU, out=out)
    torch.cuda.synchronize()
    graph, home = torch.cuda.CUDAGraph(), ctx.stream
    with torch.cuda.graph(graph):
        ctx.set_stream(torch.cuda.current_stream())
        for _ in range(calls):
            s2lib.group_norm(ctx, x, 32, act=s2lib.S2_ACT_SILU, out=out)
    ctx.set_stream(home)
    times = []
    for _ in range(7):
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end) / calls * 1e3)
    del graph
    return min(times)


def test_long_slabs_run_in_one_wave(s2lib, gpu_ctx):
    """9,000 x 512 in 192 CTAs of 12 rows a thread: 11 us, 23.5 in two waves; x of half the rows, in 144 CTAs of 8 rows a
    thread, 8.9 either way.  In one wave twice the rows take less than twice the time."""
    whole, half = (torch.randn(1, rows, 512, device="cuda").bfloat16() for rows in (9000, 4500))
    long, short = (_time(s2lib, gpu_ctx, x, torch.empty_like(x)) for x in (whole, half))
    assert long < 1.8 * short, (long, short)
