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


def test_outputs_that_share_memory():
    """Expanded outputs and other orders of the input's memory are refused;
    strided ones, and the queries themselves, are not."""
    rng = np.random.default_rng(4)
    pool = _pool()
    k, v, q = (_rand(rng, (4, h, 64)) for h in (2, 2, 4))
    plan = paged.AppendPlan(pool, [0, 1, 2, 3])
    base = torch.zeros(4 * 4 * 64, dtype=torch.bfloat16, device=DEV)
    bad = [base[:256].view(1, 4, 64).expand(4, 4, 64), base[:256].view(4, 1, 64).expand(4, 4, 64),
           base.as_strided((4, 4, 64), (256, 32, 1)), base.as_strided((4, 4, 64), (64, 64, 1))]
    for out in bad:
        with pytest.raises(ValueError, match="share memory"):
            paged.kv_append(pool, 0, plan, k, v, q=q, q_out=out)
    turned = q[:, :, :].as_strided((4, 4, 64), (64, 256, 1))
    with pytest.raises(ValueError, match="overlaps q"):
        paged.kv_append(pool, 0, plan, k, v, q=q, q_out=turned)
    once = q[:1].expand(4, 4, 64)
    with pytest.raises(ValueError, match="share memory"):
        paged.kv_append(pool, 0, plan, k, v, q=once, q_out=once)
    assert torch.equal(paged.kv_append(pool, 0, plan, k, v, q=once), once)  # (an input may be expanded)
    odd = torch.zeros((4, 64, 4), dtype=torch.bfloat16, device=DEV).transpose(1, 2)
    assert torch.equal(paged.kv_append(pool, 0, plan, k, v, q=q, q_out=odd), q)
    tight = torch.zeros(4 * 265, dtype=torch.bfloat16, device=DEV).as_strided((4, 4, 64), (265, 67, 1))
    assert torch.equal(paged.kv_append(pool, 0, plan, k, v, q=q, q_out=tight), q)
    first = q[:1].as_strided((1, 4, 64), (7, 64, 1))  # a row alone has any stride
    assert paged.kv_append(pool, 0, paged.AppendPlan(pool, [8]), k[:1], v[:1], q=q[:1], q_out=first) is first
    one = base[:256].view(1, 4, 64)[:, :1].expand(1, 1, 64)
    assert paged.kv_append(pool, 0, paged.AppendPlan(pool, [9]), k[:1], v[:1], q=q[:1, :1], q_out=one) is one
    for rows in (4, 90):  # both kernels
        n = rows
        sees = paged.AttentionPlan(pool, row_off=[0, n], row_vis=np.arange(n) % 5, page_off=[0, 1], pages=[0], num_q_heads=4)
        qq = _rand(rng, (n, 4, 64), torch.bfloat16, 0.3)
        for out in (qq[:1].expand(n, 4, 64), qq[:, :1].expand(n, 4, 64)):
            with pytest.raises(ValueError, match="share memory"):
                paged.paged_attention(pool, 0, sees, qq, out=out)
        want = paged.paged_attention(pool, 0, sees, qq)
        assert torch.equal(paged.paged_attention(pool, 0, sees, qq[:1].expand(n, 4, 64))[0], want[0])
        assert paged.paged_attention(pool, 0, sees, qq, out=qq) is qq and torch.equal(qq, want)
    paged.check_status(pool)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_in_place_of_split_lists(dtype):
    """The queries as the output, where several CTAs read a row."""
    rng = np.random.default_rng(5)
    pool = _pool(heads=1, pages=300)
    page_off, pages, _ = _fill(pool, rng, [4000, 600])
    for rows in (3, 20, 100):
        row_off = np.array([0, rows, rows + 2])
        plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=np.r_[np.full(rows, 4000), 600, 30], page_off=page_off,
                                   pages=pages, num_q_heads=2)
        q = _rand(rng, (rows + 2, 2, 64), dtype, 0.3)
        want = paged.paged_attention(pool, 0, plan, q)
        assert torch.equal(paged.paged_attention(pool, 0, plan, q, out=q), want)


def test_host_data_under_a_default_device():
    """Lists are host data whatever torch's default device is."""
    rng = np.random.default_rng(6)
    pool = _pool(pages=4)
    k, v, q = (_rand(rng, (3, h, 64)) for h in (2, 2, 2))
    torch.set_default_device("cuda")
    try:
        pool.alloc(2)
        plan = paged.AppendPlan(pool, [0, 1, 2])
        paged.kv_append(pool, 0, plan, k, v)
        sees = paged.AttentionPlan(pool, row_off=[0, 3], row_vis=[1, 2, 3], page_off=[0, 1], pages=[0], num_q_heads=2)
        got = paged.paged_attention(pool, 0, sees, q)
        paged.kv_read(pool, 0, [0, 1, 2])
        pool.begin_pages([3])
        with pytest.raises(ValueError, match="int32"):
            paged.AppendPlan(pool, [2**31])
    finally:
        torch.set_default_device(None)
    paged.check_status(pool)
    sees = paged.AttentionPlan(pool, row_off=[0, 3], row_vis=[1, 2, 3], page_off=[0, 1], pages=[0], num_q_heads=2)
    assert torch.equal(got, paged.paged_attention(pool, 0, sees, q)) and got.any()
