"""GPU: calls of the cache operators that the documentation allows, or refuses."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from imba_chess_b200 import _native, paged
from tests.test_gpu_paged import DEV, _check_stored, _f64, _fill, _pool, _rand

pytestmark = pytest.mark.gpu


def _reported(pool):
    with pytest.raises(_native.ImbaError) as e:
        paged.check_status(pool)
    assert e.value.code == _native.IMBA_ERR_RANGE
    paged.check_status(pool)


@pytest.mark.parametrize("far", [2**32 + 5, 2**31, -(2**32) + 5, -(2**40), 2**63 - 1])
def test_wide_integers_on_the_device(far):
    """int64 tensors on the device are taken by value: what is outside int32
    is outside the pool, and is skipped and reported."""
    rng = np.random.default_rng(1)
    pool = _pool(pages=4)
    k, v = (_rand(rng, (3, 2, 64), torch.float32) for _ in range(2))
    wide = lambda *x: torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
    paged.kv_append(pool, 0, paged.AppendPlan(pool, wide(5, 20, -1)), k, v)
    paged.check_status(pool)
    paged.kv_append(pool, 0, paged.AppendPlan(pool, wide(4, far, 21)), k, v)
    _reported(pool)
    kept = {5: (_f64(k[0]), _f64(v[0])), 20: (_f64(k[1]), _f64(v[1])), 4: (_f64(k[0]), _f64(v[0])), 21: (_f64(k[2]), _f64(v[2]))}
    _check_stored(pool, 0, kept)
    paged.kv_read(pool, 0, wide(5, far))
    _reported(pool)
    rows = dict(row_off=wide(0, 1), row_vis=wide(6), page_off=wide(0, 1), pages=wide(0), num_q_heads=2)
    q = _rand(rng, (1, 2, 64))
    want = paged.paged_attention(pool, 0, paged.AttentionPlan(pool, **rows), q)
    paged.check_status(pool)
    assert want.any()
    for name, bad in (("pages", wide(far)), ("row_vis", wide(far)), ("row_off", wide(0, far)), ("page_off", wide(0, far))):
        paged.paged_attention(pool, 0, paged.AttentionPlan(pool, **{**rows, name: bad}), q)
        _reported(pool)


def test_errors_of_a_graph_that_is_the_first_use():
    """A pool whose first operators are captured: what a replay reports stays
    until it is read, through further replays."""
    rng = np.random.default_rng(2)
    warm = _pool(pages=4)
    k, v = (_rand(rng, (2, 2, 64)) for _ in range(2))
    paged.kv_append(warm, 0, paged.AppendPlan(warm, [0, 1]), k, v)
    pool = _pool(pages=4)
    slots = torch.tensor([0, 9999], dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = paged.AppendPlan(pool, slots)
        paged.kv_append(pool, 0, plan, k, v)
    graph.replay()
    slots.copy_(torch.tensor([0, 1], dtype=torch.int32))
    graph.replay()
    _reported(pool)
    _check_stored(pool, 0, {i: (_f64(k[i]), _f64(v[i])) for i in (0, 1)})


@pytest.mark.parametrize("seqs", [65536, 65538])
def test_sequences_that_overlap(seqs):
    """Offsets that go back and forth over all rows, which ask for 2^32 tiles
    and more: reported, and every row is still some sequence's."""
    rng = np.random.default_rng(3)
    rows = 1 << 21
    pool = _pool(heads=1, dqk=32, dv=32, pages=2)
    _, pages, _ = _fill(pool, rng, [16])
    q = torch.randn((rows, 1, 32), dtype=torch.bfloat16, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    vis = torch.arange(rows, dtype=torch.int32, device=DEV) % 17
    plan = paged.AttentionPlan(pool, row_off=[0, rows], row_vis=vis, page_off=[0, 1], pages=pages[:1], num_q_heads=1)
    want = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    off = np.where(np.arange(seqs + 1) % 2 == 0, 0, rows)
    plan = paged.AttentionPlan(pool, row_off=off, row_vis=vis, page_off=np.arange(seqs + 1), pages=np.repeat(pages[:1], seqs),
                               num_q_heads=1)
    got = paged.paged_attention(pool, 0, plan, q, out=torch.zeros_like(q))
    _reported(pool)
    assert torch.equal(got, want)
