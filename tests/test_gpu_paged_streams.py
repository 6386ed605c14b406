"""GPU: a pool in 8 bits used on several streams, and what its host calls wait for."""

from __future__ import annotations

import pytest
import torch

from imba_chess_b200 import paged
from imba_chess_b200.kvpool import KVSequence
from tests.test_gpu_paged import DEV, _pool

pytestmark = pytest.mark.gpu

LONG = 400_000_000  # cycles of the device: some 0.2 s


def _step(pool, rows, seed):
    """A sequence of ``rows`` new tokens: (sequence, its append plan, keys and values, queries, its attention plan)."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda: torch.randn((rows, 2, 64), dtype=torch.bfloat16, device=DEV, generator=gen)  # noqa: E731
    seq = KVSequence(pool)
    slots = seq.reserve(rows)
    plan = paged.AppendPlan(pool, slots)
    sees = paged.AttentionPlan(pool, row_off=[0, rows], row_vis=list(range(1, rows + 1)), page_off=[0, len(seq.pages)],
                               pages=seq.pages, num_q_heads=2)
    return seq, plan, (rand(), rand()), rand(), sees


def test_pages_are_emptied_behind_their_last_readers():
    """A page that one stream still reads comes back to the pool and is handed
    out again: a step of another stream does not empty it under the reader."""
    pool = _pool(pages=4)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    b.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(b):
        seq, plan, kv, q, sees = _step(pool, 10, 1)
        paged.kv_append(pool, 0, plan, *kv)
        want = paged.paged_attention(pool, 0, sees, q)
    torch.cuda.synchronize()
    assert want.any()
    with torch.cuda.stream(b):
        torch.cuda._sleep(LONG)
        got = paged.paged_attention(pool, 0, sees, q)
    page = seq.pages[0]
    seq.release()
    again = KVSequence(pool)
    again.reserve(3)
    assert again.pages == [page]  # for stream b's next step
    with torch.cuda.stream(a):
        _, plan_a, kv_a, _, _ = _step(pool, 5, 2)
        paged.kv_append(pool, 0, plan_a, *kv_a)
    torch.cuda.synchronize()
    paged.check_status(pool)
    assert torch.equal(got, want)


def test_pages_are_emptied_before_other_streams_write():
    """One stream's step empties the pages of another's, which waits for it."""
    pool, alone = _pool(pages=4), _pool(pages=4)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
    _, plan_a, kv_a, _, _ = _step(pool, 5, 1)
    seq, plan_b, kv_b, _, _ = _step(pool, 20, 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(LONG)
        paged.kv_append(pool, 0, plan_a, *kv_a)
    with torch.cuda.stream(b):
        paged.kv_append(pool, 0, plan_b, *kv_b)
    torch.cuda.synchronize()
    paged.check_status(pool)
    slots = seq.slots(0, 20)
    paged.kv_append(alone, 0, paged.AppendPlan(alone, slots), *kv_b)
    for got, want in zip(paged.kv_read(pool, 0, slots), paged.kv_read(alone, 0, slots)):
        assert torch.equal(got, want) and got.any()


def test_graphs_on_their_own_stream():
    """A capture waits for no other stream; its replays are the caller's to order."""
    pool = _pool(pages=4)
    seq, plan, kv, q, sees = _step(pool, 10, 1)
    paged.kv_append(pool, 0, plan, *kv)
    want = paged.paged_attention(pool, 0, sees, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        paged.kv_append(pool, 0, plan, *kv)
        got = paged.paged_attention(pool, 0, sees, q)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    paged.check_status(pool)
    assert torch.equal(got, want)


def test_nothing_waits_for_the_device():
    """Pages handed out, plans from host lists, append, attention and reads
    are enqueued while the device is busy with something else."""
    pool = _pool(pages=8)
    _, plan, kv, q, sees = _step(pool, 10, 1)  # the first use: libraries and memory
    paged.kv_append(pool, 0, plan, *kv)
    paged.paged_attention(pool, 0, sees, q)
    slots = KVSequence(pool).reserve(10)
    paged.kv_read(pool, 0, slots)
    _, plan, kv, q, sees = _step(pool, 40, 2)
    paged.kv_append(pool, 0, plan, *kv)
    torch.cuda.synchronize()
    busy = torch.cuda.Event()
    torch.cuda._sleep(10 * LONG)
    busy.record()
    seq, plan, kv, q, sees = _step(pool, 20, 3)
    paged.kv_append(pool, 0, plan, *kv)
    got = paged.paged_attention(pool, 0, sees, q)
    read = paged.kv_read(pool, 0, seq.slots(0, 20))
    assert not busy.query()
    torch.cuda.synchronize()
    paged.check_status(pool)
    alone = _pool(pages=8)
    plan = paged.AppendPlan(alone, seq.slots(0, 20))
    paged.kv_append(alone, 0, plan, *kv)
    for mine, want in zip(read, paged.kv_read(alone, 0, seq.slots(0, 20))):
        assert torch.equal(mine, want)
    sees = paged.AttentionPlan(alone, row_off=[0, 20], row_vis=list(range(1, 21)), page_off=[0, 2], pages=seq.pages, num_q_heads=2)
    assert torch.equal(got, paged.paged_attention(alone, 0, sees, q))


def test_host_data_is_copied_when_it_is_given():
    """What a caller does with its arrays afterwards, pinned ones too, changes
    nothing; and a capture takes no host data."""
    pool = _pool(pages=8)
    slots = torch.arange(20, dtype=torch.int32).pin_memory()
    torch.cuda._sleep(LONG)
    plan = paged.AppendPlan(pool, slots)
    slots.fill_(3)
    torch.cuda.synchronize()
    assert plan.slots.tolist() == list(range(20))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            paged.AppendPlan(pool, [0, 1])
        with pytest.raises(RuntimeError, match="capture"):
            pool.begin_pages([0])
        keep = paged.AppendPlan(pool, plan.slots)
    graph.replay()
    torch.cuda.synchronize()
    paged.check_status(pool)
    del keep


@pytest.mark.parametrize("rows", [3, 100])
def test_calls_at_once(rows):
    """Two streams, and two graphs, with a plan each, over one pool at the same time."""
    n, streams = 3000, [torch.cuda.Stream() for _ in range(2)]
    pool = _pool(pages=200)
    seq = KVSequence(pool)
    slots = seq.reserve(n)
    gen = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(s, dtype=torch.bfloat16, device=DEV, generator=gen)  # noqa: E731
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), rand(n, 2, 64), rand(n, 2, 64))
    plan = lambda: paged.AttentionPlan(pool, row_off=[0, rows], row_vis=[n - i for i in range(rows)],  # noqa: E731
                                       page_off=[0, len(seq.pages)], pages=seq.pages, num_q_heads=4)
    plans, q = [plan(), plan()], [rand(rows, 4, 64) for _ in streams]
    want = [paged.paged_attention(pool, 0, plans[0], x) for x in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(25):
        for s, p, x, g in zip(streams, plans, q, got):
            with torch.cuda.stream(s):
                g.append(paged.paged_attention(pool, 0, p, x))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in streams], []
    for graph, p, x in zip(graphs, plans, q):
        with torch.cuda.graph(graph):
            outs.append([paged.paged_attention(pool, 0, p, x) for _ in range(5)])
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    paged.check_status(pool)
    for w, g, o in zip(want, got, outs):
        assert all(torch.equal(w, x) for x in g + o)


def test_a_new_pool_on_another_stream():
    """A pool that is still being cleared on the stream it was made on."""
    warm, ready = _pool(pages=4), torch.cuda.Stream()
    _, plan, kv, q, sees = _step(warm, 10, 1)
    paged.kv_append(warm, 0, plan, *kv)
    want = paged.kv_read(warm, 0, plan.slots)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(LONG)
        pool = _pool(pages=4)
    with torch.cuda.stream(ready):
        paged.kv_append(pool, 0, paged.AppendPlan(pool, plan.slots), *kv)
        got = paged.kv_read(pool, 0, plan.slots)
    torch.cuda.synchronize()
    paged.check_status(pool)
    late = paged.kv_read(pool, 0, plan.slots)
    for w, g, l in zip(want, got, late):
        assert torch.equal(w, g) and torch.equal(w, l)
