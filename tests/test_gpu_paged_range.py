"""GPU: attention over a pool in 8 bits at the ends of the range: masks and
scores of any size, values many powers of two apart.

Tolerances.  The keys that a row weighs here all have the same score to the
last bit (or scores a whole number apart), so weights are off by their own
rounding alone: f16, 2^-11 (fp32 queries: two parts, 2^-21), and the
exponential's 2^-20; the output by half a step of its type."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from imba_chess_b200 import paged
from tests.test_gpu_paged import DEV, HALF, _f64, _fill, _pool, _rand

pytestmark = pytest.mark.gpu

# (sequences' lengths, rows of each): a warp a unit, a CTA a unit, split lists,
# tiles of 24 rows, tiles of 128 rows, split tiles of 128 rows
SHAPES = {"warp": ([40] * 1300, [1] * 1300), "cta": ([100, 33, 7], [1, 5, 2]), "split": ([6000, 50], [1, 2]),
          "24": ([300, 64], [20, 20]), "128": ([200, 130], [90, 130]), "128 split": ([5000, 300], [100, 80])}


def _step(shape, dtype, seed, heads=1, q_heads=2, **kw):
    """A filled pool and a plan in which every row sees all its sequence's tokens, at position 0."""
    lens, nrow = SHAPES[shape]
    rng = np.random.default_rng(seed)
    pool = _pool(heads=heads, pages=sum(-(-n // 16) for n in lens) + 1)
    page_off, pages, slots = _fill(pool, rng, lens)
    row_off = np.r_[0, np.cumsum(nrow)]
    vis = np.repeat(lens, nrow)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=q_heads,
                               positions=np.zeros(len(vis), np.int32), **kw)
    off = np.r_[0, np.cumsum(lens)]
    return rng, pool, plan, [slots[off[g] : off[g + 1]] for g in range(len(lens))], nrow, vis


def _check(got, want, mean, dtype):
    """want: exact; mean: the weighted mean of |v|."""
    g = _f64(got)
    assert np.isfinite(g).all()
    own = 2.0**-11 if dtype == torch.bfloat16 else 2.0**-21
    off = np.abs(g - want)
    tol = HALF[dtype] * np.abs(want) + (own + 2.0**-20) * mean
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_bias_of_any_size(shape, dtype):
    """A row whose every key carries the same large bias weighs them alike,
    whatever its value; keys that carry less than that count for nothing."""
    rng, pool, plan, seqs, nrow, vis = _step(shape, dtype, 3)
    n = len(vis)
    q = torch.zeros((n, 2, 64), dtype=dtype, device=DEV)
    values = [paged.kv_read(pool, 0, s, torch.float32)[1] for s in seqs]
    mp = int(vis.max()) + 1
    half = (np.arange(2 * mp - 1) - (mp - 1)) % 3 == 0  # every third key, from the first on
    for size in (-1e5, -1e7, -1.1e9, 3.3e9, -1e20, 7e20, -1e30, -1.3e31, 1.1e36, -3.3e38, 3.3e38):
        table = np.full((2, 2 * mp - 1), size)
        table[1] = np.where(half, size, np.maximum(size - 0.25 * abs(size), np.finfo(np.float32).min) if abs(size) < 3e38 else -abs(size) * 0.9)
        if size == -3.3e38:
            table[1] = np.where(half, size, -np.inf)
        got = paged.paged_attention(pool, 0, plan, q, bias=torch.tensor(table, dtype=torch.float32, device=DEV))
        paged.check_status(pool)
        want, mean = np.zeros((n, 2, 64)), np.zeros((n, 2, 64))
        r = 0
        for v, k in zip(values, nrow):
            v = _f64(v[:, 0])
            want[r : r + k, 0], mean[r : r + k, 0] = v.mean(0), np.abs(v).mean(0)
            want[r : r + k, 1], mean[r : r + k, 1] = v[::3].mean(0), np.abs(v[::3]).mean(0)
            r += k
        _check(got, want, mean, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_far_bias_with_small_steps(shape, dtype):
    """Biases of some 10^7 that are whole numbers apart: weights before and
    behind each new maximum, of parts and of warps, fit together."""
    rng, pool, plan, seqs, nrow, vis = _step(shape, dtype, 5)
    n = len(vis)
    q = torch.zeros((n, 2, 64), dtype=dtype, device=DEV)
    values = [_f64(paged.kv_read(pool, 0, s, torch.float32)[1][:, 0]) for s in seqs]
    mp = int(vis.max()) + 1
    for base in (-10_000_003.0, 12_000_001.0):
        table = base + rng.integers(0, 4, (2, 2 * mp - 1)) + np.arange(2 * mp - 1) * 8 // mp
        got = paged.paged_attention(pool, 0, plan, q, bias=torch.tensor(table, dtype=torch.float32, device=DEV))
        want, mean = np.zeros((n, 2, 64)), np.zeros((n, 2, 64))
        r = 0
        for v, k in zip(values, nrow):
            for h in (0, 1):
                s = table[h, mp - 1 : mp - 1 + len(v)]
                w = np.exp(s - s.max())
                w /= w.sum()
                want[r : r + k, h], mean[r : r + k, h] = w @ v, w @ np.abs(v)
            r += k
        _check(got, want, mean, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", ["warp", "cta", "24", "128", "128 split"])
def test_scores_of_any_size(shape, dtype):
    """Scores from 1 to 2^100, of either sign: of keys 3 and 1 times a unit
    vector the ones that the row's sign prefers share the weight."""
    lens, nrow = SHAPES[shape]
    rng, pool, plan, seqs, nrow, vis = _step(shape, dtype, 7)
    pool.begin_pages(list(range(pool.num_pages)))
    slots = np.concatenate(seqs)
    three = np.concatenate([np.arange(len(s)) % 4 == 1 for s in seqs])
    k = torch.zeros((len(slots), 1, 64), device=DEV)
    k[:, 0, 5] = torch.tensor(np.where(three, 3.0, 1.0), dtype=torch.float32, device=DEV)
    v = _rand(rng, (len(slots), 1, 64), torch.bfloat16, 0.7).float()
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
    n = len(vis)
    size = np.exp2(rng.integers(8, 100, (n, 2))) * rng.integers(128, 256, (n, 2)) / 128 * np.where(np.arange(n) % 3 == 0, -1, 1)[:, None]
    q = torch.zeros((n, 2, 64), dtype=dtype, device=DEV)
    q[:, :, 5] = torch.tensor(size, dtype=torch.float32, device=DEV).to(dtype)
    got = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    want, mean = np.zeros((n, 2, 64)), np.zeros((n, 2, 64))
    r = 0
    for s, m in zip(seqs, nrow):
        vv = _f64(paged.kv_read(pool, 0, s, torch.float32)[1][:, 0])
        high = np.arange(len(s)) % 4 == 1
        for i in range(r, r + m):
            for h in (0, 1):
                w = vv[high if size[i, h] > 0 else ~high]
                want[i, h], mean[i, h] = w.mean(0), np.abs(w).mean(0)
        r += m
    _check(got, want, mean, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 20, 100])
def test_values_at_both_ends_of_the_range(rows, dtype):
    """A page of sixteen with values of 2^110, the others with 2^-96: the small
    ones' keys count in the row's sum all the same."""
    seqs, heads, pages = 80, 16, 32  # lists short and many: a unit sees sixteen pages of a list at least
    n = 16 * pages
    pool = _pool(heads=heads, pages=seqs * pages)
    ids = np.random.default_rng(rows).permutation(seqs * pages)
    slots = (ids[:, None] * 16 + np.arange(16)).reshape(-1)
    big = np.arange(n) // 16 % 16 == 4
    k, v = (torch.zeros((len(slots), heads, 64), device=DEV) for _ in range(2))
    k[:, :, 9] = torch.tensor(np.tile(big, seqs), dtype=torch.float32, device=DEV)[:, None]
    v[:] = torch.tensor(np.where(np.tile(big, seqs), 2.0**110, 2.0**-96), dtype=torch.float32, device=DEV)[:, None, None]
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
    q = torch.zeros((seqs * rows, heads, 64), dtype=dtype, device=DEV)
    q[:, :, 9] = 7.0
    plan = paged.AttentionPlan(pool, row_off=np.arange(seqs + 1) * rows, row_vis=np.full(seqs * rows, n),
                               page_off=np.arange(seqs + 1) * pages, pages=ids, num_q_heads=heads)
    got = paged.paged_attention(pool, 0, plan, q, scale=1.0)
    paged.check_status(pool)
    w = np.where(big, math.exp(7.0), 1.0)
    want = np.full((seqs * rows, heads, 64), 2.0**110 * w[big].sum() / w.sum())
    _check(got, want, want, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_values_of_the_largest_size(shape, dtype):
    """Values at the upper end of fp32 average to values of that size: no sum
    over keys, warps or parts runs over."""
    rng, pool, plan, seqs, nrow, vis = _step(shape, dtype, 11)
    pool.begin_pages(list(range(pool.num_pages)))
    slots = np.concatenate(seqs)
    k = torch.zeros((len(slots), 1, 64), device=DEV)
    v = torch.tensor(rng.choice([3e38, 2e38, 1.5e38], (len(slots), 1, 64)), dtype=torch.float32, device=DEV)
    v[..., 32:] *= -1
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
    q = torch.zeros((len(vis), 2, 64), dtype=dtype, device=DEV)
    got = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    means = np.stack([_f64(paged.kv_read(pool, 0, s, torch.float32)[1][:, 0]).mean(0) for s in seqs])
    want = np.repeat(means, nrow, axis=0)[:, None].repeat(2, 1)
    _check(got, want, np.abs(want), dtype)
