"""As many prefixes as a call takes: what each request sees, and that finding it does not take a step a prefix."""
import pytest
import torch

from prefix_reference import check
from test_gpu_paged import BF16, FP16, _cuda
from test_gpu_prefix import _both, _ints, _query

pytestmark = pytest.mark.gpu


# rows of one KV head and head: one list of a prefix's rows, and a list of requests
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("prefixes", [63, 64, 65, 127, 128, 1000, 1024])
def test_every_request_sees_its_own_prefix(prefixes, rows):
    dev, batch = _cuda(), 300 if prefixes < 1000 else 1024
    gen = torch.Generator().manual_seed(prefixes)
    lengths = torch.randint(0, 40, (batch,), generator=gen).tolist()
    shared, own = _both(dev, [int(n) for n in torch.randint(0, 40, (prefixes,), generator=gen)], lengths, 1, 16, BF16 if rows == 1 else FP16, prefixes)
    q = _query(dev, batch, 1, rows, BF16 if rows == 1 else FP16, prefixes)
    most = 2 * batch // prefixes
    members = torch.randint(-1, most + 1, (prefixes,), generator=gen)
    members[-1] = 5
    counts = torch.randint(0, rows + 1, (batch,), generator=gen)
    check(q, own, shared, _ints(dev, *members.tolist()))
    check(q, own, shared, _ints(dev, *members.tolist()), _ints(dev, *counts.tolist()))
    check(q, own, shared, _ints(dev, *[0] * (prefixes - 1), batch))


def _time(dev, call, runs=7):
    call()
    times = []
    for _ in range(runs):
        events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        events[0].record()
        for _ in range(3):
            call()
        events[1].record()
        torch.cuda.synchronize(dev)
        times.append(events[0].elapsed_time(events[1]))
    return sorted(times)[runs // 2]


@pytest.mark.parametrize("rows", [1, 5, 64])
def test_a_prefix_each_takes_about_what_one_for_sixteen_does(rows):
    """1024 requests, 65536 slots of prefixes in all: 64 prefixes, and 1024.  One step a prefix for each 64 requests made that 9 to 50
    times as long."""
    import r2omni_amd as ro

    dev, times = _cuda(), []
    for prefixes in (64, 1024):
        shared, own = _both(dev, (65536 // prefixes,) * prefixes, (20 + rows,) * 1024, 2, 64, BF16, rows)
        q, members = _query(dev, 1024, 16, rows, BF16, rows), _ints(dev, *[1024 // prefixes] * prefixes)
        times.append(_time(dev, lambda: ro.paged_prefix_attention(q, own, shared, members=members)))
    assert times[1] < 4 * times[0], times


@pytest.mark.parametrize("rows", [1, 40])
def test_a_captured_call_follows_many_prefixes(rows):
    import r2omni_amd as ro

    dev, prefixes, batch = _cuda(), 130, 200
    gen = torch.Generator().manual_seed(rows)
    shared, own = _both(dev, (33,) * prefixes, (40,) * batch, 1, 16, BF16, rows)
    q, members = _query(dev, batch, 2, rows, BF16, rows), _ints(dev, *[1] * prefixes)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ro.paged_prefix_attention(q, own, shared, members=members)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = ro.paged_prefix_attention(q, own, shared, members=members)
    for _ in range(5):
        members.copy_(torch.randint(-1, 5, (prefixes,), generator=gen))
        shared.lengths.copy_(torch.randint(0, 34, (prefixes,), generator=gen))
        own.lengths.copy_(torch.randint(0, 41, (batch,), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        eager = check(q, own, shared, members)
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
