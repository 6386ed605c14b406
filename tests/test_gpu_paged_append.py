"""GPU: the append's 16-byte path on parts of heads of every size, its query
warps of several rows, and CTAs that go from page to page.  Tolerances as in
test_gpu_paged."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from imba_chess_b200 import paged
from tests.test_gpu_paged import DEV, E4M3, HALF, _check_stored, _f64, _pool, _rand, _turn

pytestmark = pytest.mark.gpu


def _check(pool, slots, k, v, q, got_q, pos, freq, layout, dtype, axis=None):
    want_k = _turn(_f64(k), pos, freq, layout, axis)
    if q is not None:
        want_q, size = _turn(_f64(q), pos, freq, layout, axis), np.abs(_f64(q)).max(-1, keepdims=True)
        assert (np.abs(_f64(got_q) - want_q) <= HALF[dtype] * np.abs(want_q) + 2.0**-20 * size).all()
    if pool.dtype == E4M3:
        vv = _f64(v)
        _check_stored(pool, 0, {int(s): (want_k[i], vv[i]) for i, s in enumerate(slots)}, eps=2.0**-20)
        return
    gk, gv = paged.kv_read(pool, 0, slots)
    paged.check_status(pool)
    size = np.abs(_f64(k)).max(-1, keepdims=True)
    assert (np.abs(_f64(gk) - want_k) <= HALF[pool.dtype] * np.abs(want_k) + 2.0**-20 * size).all()
    assert torch.equal(gv, v.to(pool.dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(64, 32), (64, 16), (32, 32), (32, 16), (96, 96), (96, 64), (96, 16), (128, 128), (128, 64), (128, 112)])
@pytest.mark.parametrize("pool_dtype", [E4M3, torch.bfloat16, torch.float32], ids=["e4m3", "bf16", "fp32"])
def test_rotation_of_parts_by_vectors(pool_dtype, d, rot, layout, dtype):
    """Contiguous rows, rotations that are multiples of 16 elements: whole
    pages, and single tokens, which take the other shape of work."""
    rng = np.random.default_rng(d + rot)
    heads, hq = 9, 11
    pool = _pool(pool_dtype, heads=heads, dqk=d, dv=d, pages=20)
    freq = [100 ** (-2 * p / rot) for p in range(rot // 2)]
    rotary = paged.Rotary(freq, device=DEV, layout=layout)
    order = rng.permutation(20)
    for slots in ((order[:5, None] * 16 + np.arange(16)).reshape(-1)[:77], order[6:17] * 16 + rng.integers(0, 16, 11)):
        n = len(slots)
        k, v, q = (_rand(rng, (n, h, d), dtype) for h in (heads, heads, hq))
        pos = np.r_[0, 3_000_000, rng.integers(0, 500, n - 2)]
        got = paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v, rotary=rotary, q=q,
                              positions=torch.tensor(pos, dtype=torch.int32, device=DEV))
        _check(pool, slots, k, v, q, got, pos, freq, layout, dtype)


@pytest.mark.parametrize("pool_dtype", [E4M3, torch.bfloat16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d,hq,rot", [(64, 4, 64), (64, 5, 58), (128, 8, 64), (32, 3, 32)])
def test_steps_of_many_pages(d, hq, rot, dtype, pool_dtype):
    """More pages than CTAs, with ends inside of a page and padding rows, and
    query warps of four rows; then a step that raises the scales of all pages
    and one of a token a page."""
    rng = np.random.default_rng(d + hq)
    heads, count = 2, 800
    pool = _pool(pool_dtype, heads=heads, dqk=d, dv=d, pages=count)
    freq = [1000 ** (-2 * p / rot) for p in range(rot // 2)]
    rotary = paged.Rotary(freq, device=DEV)
    pages = rng.permutation(count)
    first = [p * 16 + t for p, n in zip(pages, rng.integers(12, 16, count)) for t in range(n)]
    held = {}
    for slots, size in ((np.r_[first, -1, -1], 1.0), (pages * 16 + 15, 20.0), (pages * 16 + 3, 0.1)):
        slots = rng.permutation(slots)
        n = len(slots)
        assert n > 9472 or n == count  # from there on a warp takes four rows of queries, of 1,024 elements at most
        k, v, q = (_rand(rng, (n, h, d), dtype) for h in (heads, heads, hq))
        k, v = k * size, v * size
        pos = rng.integers(0, 100_000, n)
        got = paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v, rotary=rotary, q=q, q_out=torch.full_like(q, 7.0),
                              positions=torch.tensor(pos, dtype=torch.int32, device=DEV))
        live = slots >= 0
        assert (got[torch.tensor(~live, device=DEV)] == 7).all()
        lv = torch.tensor(np.flatnonzero(live), device=DEV)
        want_q, amax = _turn(_f64(q[lv]), pos[live], freq), np.abs(_f64(q[lv])).max(-1, keepdims=True)
        assert (np.abs(_f64(got[lv]) - want_q) <= HALF[dtype] * np.abs(want_q) + 2.0**-20 * amax).all()
        want_k, vv = _turn(_f64(k), pos, freq), _f64(v)
        if pool_dtype != E4M3:
            gk, gv = paged.kv_read(pool, 0, slots[live])
            size_k = np.abs(_f64(k[lv])).max(-1, keepdims=True)
            assert (np.abs(_f64(gk) - want_k[live]) <= HALF[pool_dtype] * np.abs(want_k[live]) + 2.0**-20 * size_k).all()
            assert torch.equal(gv, v[lv].to(pool_dtype))
        elif size >= 1:  # (the last step's tokens replace some, whose scales stay)
            held.update({int(s): (want_k[i], vv[i]) for i, s in enumerate(slots) if s >= 0})
            _check_stored(pool, 0, held, eps=2.0**-20)
        else:
            gk, gv = (_f64(t) for t in paged.kv_read(pool, 0, slots, torch.float32))
            step = np.exp2(_f64(pool.scales)[slots // 16, 0] - 127.0)  # [n, 2, heads]
            for g, want, part in ((gk, want_k, 0), (gv, vv, 1)):
                bound = np.maximum(np.abs(want) * 2.0**-4, step[:, part, :, None] * 2.0**-10) + 2.0**-20 * np.abs(want).max(-1, keepdims=True)
                assert (np.abs(g - want) <= bound).all()
    paged.check_status(pool)
