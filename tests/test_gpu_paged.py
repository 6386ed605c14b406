"""GPU: appending to paged pools and attention over a pool in 8 bits, against
plain implementations in 64 bits.

Tolerances.  A value in an 8-bit block of scale S is off by at most half a
step: 2^-4 of itself, or 2^-10 S where the code is subnormal; each growth of
the block's scale may round a subnormal code again, and the steps before the
last are at most half of it, so rounding adds up to less than 2^-9 S in all.
An fp32 rotation (two products, one sum, cosines and sines right to 2^-22) is
off by 2^-21 (|a| + |b|).  Attention: out is rounded to its type (half a step
relative to it), and a weight is off by its own rounding (f16: 2^-11, for fp32
queries two parts: 2^-21) plus twice what its score is off, which is counted
as d 2^-23 of the sum of |q k| |scale| (fp32 sums in any order; queries are
held to 2^-22).  Weights' errors reach an output as that share of sum w |v|.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from imba_chess_b200 import _native, paged
from imba_chess_b200.kvpool import KVPool, KVSequence

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def _pool(dtype=E4M3, layers=1, heads=2, dqk=64, dv=64, pages=32):
    return KVPool(num_layers=layers, num_heads=heads, attention_dim=dqk, linear_dim=dv, num_pages=pages, dtype=dtype,
                  device=DEV)


def _rand(rng, shape, dtype=torch.bfloat16, spread=2.0):
    x = rng.standard_normal(shape) * np.exp2(spread * rng.standard_normal(shape[1:]))
    return torch.tensor(x, dtype=torch.float32, device=DEV).to(dtype)


def _f64(t):
    return t.double().cpu().numpy()


def _turn(x, pos, freq, layout="half", axes=None):
    """The rotation in 64 bits."""
    half = len(freq)
    pos = np.asarray(pos, np.float64).reshape(len(x), -1)
    ang = pos[:, [0] * half if axes is None else axes] * np.asarray(freq)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = x.copy()
    i = (np.arange(half), np.arange(half) + half) if layout == "half" else (np.arange(half) * 2, np.arange(half) * 2 + 1)
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]] = a * c - b * s
    y[..., i[1]] = b * c + a * s
    return y


def _scale(amax):
    """2^e for the least e >= -100 with amax <= 448 2^e; 0 for an empty block."""
    e = np.ceil(np.log2(np.where(amax > 0, amax, 1) / 448.0))
    return np.where(amax > 0, np.exp2(np.maximum(e, -100)), 0.0)


def _block_scales(pool):
    return np.where(_f64(pool.scales) > 0, np.exp2(_f64(pool.scales) - 127.0), 0.0)  # [page, layer, 2, H]


def _check_stored(pool, layer, stored, eps=0.0):
    """``stored``: slot -> (k [H, d], v [H, d]) in 64 bits."""
    slots = sorted(stored)
    k, v = paged.kv_read(pool, layer, slots, torch.float32)
    paged.check_status(pool)
    scales = _block_scales(pool)
    for part, got in enumerate((k, v)):
        want = np.stack([stored[s][part] for s in slots])
        amax = np.zeros((pool.num_pages, pool.num_heads))
        np.maximum.at(amax, np.asarray(slots) // 16, np.abs(want).max(-1))
        used = sorted({s // 16 for s in slots})
        assert np.array_equal(scales[used, layer, part], _scale(amax)[used]), "scales"
        step = scales[np.asarray(slots) // 16, layer, part][..., None]
        bound = np.maximum(np.abs(want) * 2.0**-4, step * 2.0**-9) + eps * np.abs(want).max(-1, keepdims=True)
        off = np.abs(_f64(got) - want)
        assert (off <= bound).all(), float((off / np.maximum(bound, 1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dqk,dv", [(32, 32), (64, 64), (32, 64), (64, 32), (96, 96), (128, 128)])
def test_append_in_8_bits(dqk, dv, dtype):
    """Several calls into shuffled pages: whole pages, single tokens, odd and
    even halves of a pair, tokens that make the block's scale grow."""
    rng = np.random.default_rng(dqk + dv)
    pool = _pool(layers=2, heads=3, dqk=dqk, dv=dv, pages=24)
    stored = {}
    pages = rng.permutation(24)
    seq = [int(p) * 16 + t for p in pages for t in range(16)]
    for lo, hi, size in ((0, 37, 1.0), (37, 38, 300.0), (38, 43, 0.01), (43, 64, 1e-3), (64, 65, 1.0), (65, 200, 7.0)):
        order = rng.permutation(np.arange(lo, hi))
        slots = [seq[i] for i in order]
        k, v = _rand(rng, (hi - lo, 3, dqk), dtype) * size, _rand(rng, (hi - lo, 3, dv), dtype) * size
        paged.kv_append(pool, 1, paged.AppendPlan(pool, slots), k, v)
        for i, s in enumerate(slots):
            stored[s] = (_f64(k[i]), _f64(v[i]))
        _check_stored(pool, 1, stored)
    assert not pool.scales[:, 0].any()  # the other layer is untouched
    assert not pool.data.view(24, 2, -1)[:, 0].view(torch.uint8).any()


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 40, 30, 2])
@pytest.mark.parametrize("pool_dtype", [E4M3, torch.bfloat16, torch.float32], ids=["e4m3", "bf16", "fp32"])
def test_append_rotates(pool_dtype, rot, layout, axes):
    """Keys and queries turn to their positions, near and far, whole heads and
    parts of them, from strided inputs."""
    rng = np.random.default_rng(rot + axes)
    n, heads, hq, d = 45, 2, 5, 64
    dtype = torch.bfloat16 if pool_dtype == torch.bfloat16 else torch.float32
    pool = _pool(pool_dtype, heads=heads, pages=8)
    both = _rand(rng, (n, hq + 2 * heads, d), dtype)
    q, k, v = both[:, :hq], both[:, hq : hq + heads], both[:, hq + heads :]
    freq = [10000 ** (-2 * p / rot) for p in range(rot // 2)]
    axis = [p * axes // len(freq) for p in range(len(freq))] if axes > 1 else None
    cols = axes
    pos = rng.integers(0, 1 << 20, (n, cols)) if axes > 1 else np.r_[0, 1, 5_000_000, rng.integers(0, 300, n - 3)]
    rotary = paged.Rotary(freq, device=DEV, layout=layout, axes=axis)
    slots = rng.permutation(8 * 16)[:n]
    got_q = paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v, rotary=rotary, q=q,
                            positions=torch.tensor(pos, dtype=torch.int32, device=DEV).reshape(n, cols))
    want_q, want_k = _turn(_f64(q), pos, freq, layout, axis), _turn(_f64(k), pos, freq, layout, axis)
    size = np.abs(_f64(q)).max(-1, keepdims=True)
    assert (np.abs(_f64(got_q) - want_q) <= HALF[dtype] * np.abs(want_q) + 2.0**-20 * size).all()
    if pool_dtype == E4M3:
        _check_stored(pool, 0, {int(s): (want_k[i], _f64(v[i])) for i, s in enumerate(slots)}, eps=2.0**-20)
        return
    gk, gv = paged.kv_read(pool, 0, slots)
    size = np.abs(_f64(k)).max(-1, keepdims=True)
    assert (np.abs(_f64(gk) - want_k) <= HALF[dtype] * np.abs(want_k) + 2.0**-20 * size).all()
    assert torch.equal(gv, v)


def test_append_rotation_in_place_and_padding():
    """q_out may be q; padding rows (slot -1) leave the pool and their queries
    as they were."""
    rng = np.random.default_rng(3)
    pool = _pool()
    n = 9
    k, v, q = (_rand(rng, (n, h, 64)) for h in (2, 2, 4))
    slots = np.array([3, -1, 20, 21, -1, 40, 41, 42, -1])
    pos = torch.arange(100, 100 + n, dtype=torch.int32, device=DEV)
    rotary = paged.Rotary([0.1 * (i + 1) for i in range(32)], device=DEV)
    plan = paged.AppendPlan(pool, slots)
    apart = paged.kv_append(pool, 0, plan, k, v, rotary=rotary, positions=pos, q=q, q_out=torch.full_like(q, 7.0))
    before = q.clone()
    same = paged.kv_append(pool, 0, plan, k, v, rotary=rotary, positions=pos, q=q, q_out=q)
    paged.check_status(pool)
    assert same is q
    live = torch.tensor(slots >= 0, device=DEV)
    assert torch.equal(q[live], apart[live]) and torch.equal(q[~live], before[~live]) and (apart[~live] == 7).all()
    written = sorted({int(s) // 16 for s in slots if s >= 0})
    rest = [p for p in range(32) if p not in written]
    assert not pool.scales[rest].any() and pool.scales[written].all()
    turned = _turn(_f64(k), pos.cpu().numpy(), [0.1 * (i + 1) for i in range(32)])
    _check_stored(pool, 0, {int(s): (turned[i], _f64(v[i])) for i, s in enumerate(slots) if s >= 0}, eps=2.0**-20)


@pytest.mark.parametrize("pool_dtype", [E4M3, torch.float32], ids=["e4m3", "fp32"])
def test_append_same_slot_twice(pool_dtype):
    """Of rows with the same slot the last one is stored, every time."""
    rng = np.random.default_rng(5)
    for _ in range(20):
        pool = _pool(pool_dtype, pages=4)
        slots = rng.integers(0, 20, 64)
        k, v = _rand(rng, (64, 2, 64), torch.float32), _rand(rng, (64, 2, 64), torch.float32)
        paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
        stored = {int(s): (_f64(k[i]), _f64(v[i])) for i, s in enumerate(slots)}
        if pool_dtype == E4M3:
            _check_stored(pool, 0, stored)
        else:
            got = paged.kv_read(pool, 0, sorted(stored))
            for part in (0, 1):
                assert np.array_equal(_f64(got[part]), np.stack([stored[s][part] for s in sorted(stored)]))


def test_append_reports_what_it_skips():
    rng = np.random.default_rng(6)
    k, v = _rand(rng, (3, 2, 64), torch.float32), _rand(rng, (3, 2, 64), torch.float32)
    for bad in (-2, 32 * 16, 2**31 - 1):
        pool = _pool()
        paged.kv_append(pool, 0, paged.AppendPlan(pool, [1, bad, 2]), k, v)
        with pytest.raises(_native.ImbaError) as e:
            paged.check_status(pool)
        assert e.value.code == _native.IMBA_ERR_RANGE
        _check_stored(pool, 0, {1: (_f64(k[0]), _f64(v[0])), 2: (_f64(k[2]), _f64(v[2]))})  # and the status is clear
    for value in (math.inf, -math.inf, math.nan):
        pool = _pool()
        kk, vv = k.clone(), v.clone()
        kk[1, 0, 5] = value
        vv[2, 1, 63] = value
        paged.kv_append(pool, 0, paged.AppendPlan(pool, [0, 1, 2]), kk, vv)
        with pytest.raises(_native.ImbaError):
            paged.check_status(pool)
        kk[1, 0, 5] = vv[2, 1, 63] = 0.0  # stored as zero
        _check_stored(pool, 0, {i: (_f64(kk[i]), _f64(vv[i])) for i in range(3)})


def test_append_extreme_magnitudes():
    """Zeros, fp32's largest and smallest values, and a scale that grows from
    one end of the range to the other."""
    pool = _pool(heads=1, pages=6)
    big, tiny = 3.4e38, 1e-38
    k = torch.zeros((6, 1, 64), device=DEV)
    k[1] = big
    k[2] = tiny
    k[3] = -1e-3
    k[4, 0, 7] = 448.0
    k[5, 0, 7] = float(np.nextafter(np.float32(448.0), np.float32(500)))
    slots = [0, 16, 32, 48, 64, 80]
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, -k)
    stored = {s: (_f64(k[i]), -_f64(k[i])) for i, s in enumerate(slots)}
    _check_stored(pool, 0, stored)
    assert pool.scales[4, 0, 0, 0] == 127 and pool.scales[5, 0, 0, 0] == 128 and pool.scales[0, 0, 0, 0] == 0
    paged.kv_append(pool, 0, paged.AppendPlan(pool, [33, 49]), k[[1, 1]], k[[1, 1]])  # the tokens there vanish
    stored[33] = stored[49] = (_f64(k[1]), _f64(k[1]))
    _check_stored(pool, 0, stored)


def test_append_odd_head_sizes_in_full_precision():
    rng = np.random.default_rng(8)
    for dqk, dv, rot in ((8, 8, 8), (7, 5, 6), (1, 3, 0), (128, 40, 128)):
        pool = _pool(torch.float32, heads=3, dqk=dqk, dv=dv, pages=4)
        k, v = _rand(rng, (33, 3, dqk), torch.bfloat16), _rand(rng, (33, 3, dv), torch.bfloat16)
        slots = rng.permutation(64)[:33]
        freq = [0.7**i for i in range(rot // 2)]
        kw = {} if rot == 0 else {"rotary": paged.Rotary(freq, device=DEV, layout="interleaved"),
                                  "positions": torch.arange(33, dtype=torch.int32, device=DEV)}
        paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v, **kw)
        gk, gv = paged.kv_read(pool, 0, slots)
        want = _turn(_f64(k), np.arange(33), freq, "interleaved") if rot else _f64(k)
        assert np.allclose(_f64(gk), want, rtol=0, atol=2.0**-20 * np.abs(want).max())
        assert torch.equal(gv, v.float())


# ------------------------------------------------------------------------------------------------------------ attention
def _fill(pool, rng, lens, layer=0, size=1.0, dtype=torch.bfloat16):
    """Sequences of the given lengths in shuffled pages; (page_off, pages)."""
    need = [-(-n // 16) for n in lens]
    ids = rng.permutation(pool.num_pages)[: sum(need)]
    off = np.r_[0, np.cumsum(need)]
    slots = np.concatenate([ids[off[g] + np.arange(n) // 16] * 16 + np.arange(n) % 16 for g, n in enumerate(lens)] or [[]])
    n = len(slots)
    k = _rand(rng, (n, pool.num_heads, pool.attention_dim), dtype, 0.7) * size
    v = _rand(rng, (n, pool.num_heads, pool.linear_dim), dtype, 0.7) * size
    if n:
        paged.kv_append(pool, layer, paged.AppendPlan(pool, slots.astype(np.int64)), k, v)
    return off.astype(np.int32), ids.astype(np.int32), slots.astype(np.int64)


def _reference(pool, layer, q, scale, row_off, vis, page_off, pages, bias=None, pos=None, extra=None):
    """(exact output, bound) in 64 bits over what the pool holds."""
    n, hq, d = q.shape
    share = hq // pool.num_heads
    all_slots = np.concatenate([np.arange(16) + 16 * p for p in pages]) if len(pages) else np.zeros(0, np.int64)
    seq_slots = [all_slots[16 * page_off[g] : 16 * page_off[g + 1]] for g in range(len(row_off) - 1)]
    qd, half = _f64(q), HALF[q.dtype]
    out, tol = np.zeros((n, hq, pool.linear_dim)), np.zeros((n, hq, pool.linear_dim))
    own = 2.0**-11 if q.dtype == torch.bfloat16 else 2.0**-21
    cache = {}

    def read(slots):
        key = tuple(slots[:3]) + (len(slots),)
        if key not in cache:
            cache.clear()
            k, v = paged.kv_read(pool, layer, np.asarray(slots, np.int64), torch.float32)
            cache[key] = (_f64(k), _f64(v))
        return cache[key]

    for g in range(len(row_off) - 1):
        for r in range(row_off[g], row_off[g + 1]):
            m = int(vis[r])
            k, v = read(seq_slots[g]) if len(seq_slots[g]) else (np.zeros((0, pool.num_heads, d)), np.zeros((0, pool.num_heads, pool.linear_dim)))
            k, v, kpos = k[:m], v[:m], np.arange(m)
            if extra is not None:
                a, b = extra[0][r], extra[0][r + 1]
                ek, ev = paged.kv_read(pool, layer, np.asarray(extra[1][a:b], np.int64), torch.float32)
                k, v = np.concatenate([k, _f64(ek)]), np.concatenate([v, _f64(ev)])
                kpos = np.r_[kpos, extra[2][a:b]]
            if len(k) == 0:
                continue
            for h in range(hq):
                s = k[:, h // share] @ qd[r, h] * scale
                off = (np.abs(k[:, h // share]) @ np.abs(qd[r, h]) * abs(scale)).max() * d * 2.0**-23
                if bias is not None:
                    mp = (bias.shape[1] + 1) // 2
                    bb = bias[h, np.clip(kpos - pos[r] + mp - 1, 0, 2 * mp - 2)]
                    s = s + bb
                    off += np.abs(np.where(np.isfinite(bb), bb, 0)).max() * 2.0**-22
                if np.isneginf(s).all():
                    continue
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ v[:, h // share]
                tol[r, h] = half * np.abs(out[r, h]) + (own + 2 * off + 2.0**-20) * (w @ np.abs(v[:, h // share]))
    return out, tol


def _compare(got, ref):
    want, tol = ref
    off = np.abs(_f64(got) - want)
    assert np.isfinite(_f64(got)).all()
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads,share,dqk,dv", [(2, 1, 64, 64), (1, 3, 32, 32), (2, 8, 128, 128), (2, 2, 96, 96),
                                                (3, 1, 32, 64), (1, 20, 64, 32)])
def test_attention_ragged(heads, share, dqk, dv, dtype):
    """Rows of ragged sequences, from none to several pages, with and without
    a bias whose table ends inside the sequences; causal parts and whole ones."""
    rng = np.random.default_rng(heads * 1000 + dqk + dv)
    lens = [0, 1, 15, 16, 17, 31, 33, 64, 100, 257, 530]
    nrow = [2, 1, 3, 1, 2, 1, 4, 1, 40, 3, 17]
    pool = _pool(heads=heads, dqk=dqk, dv=dv, pages=90, layers=2)
    page_off, pages, _ = _fill(pool, rng, lens, layer=1)
    row_off = np.r_[0, np.cumsum(nrow)]
    vis = np.concatenate([[max(0, n - i) if n % 2 else n for i in range(r)] for n, r in zip(lens, nrow)])
    pos = vis + rng.integers(0, 4, len(vis))
    q = _rand(rng, (len(vis), heads * share, dqk), dtype, 0.3)
    bias = torch.tensor(rng.standard_normal((heads * share, 401)), dtype=torch.float32, device=DEV)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages,
                               num_q_heads=heads * share, positions=pos)
    for b, scale in ((None, None), (bias, 0.3)):
        got = paged.paged_attention(pool, 1, plan, q, bias=b, scale=scale)
        paged.check_status(pool)
        _compare(got, _reference(pool, 1, q, scale or dqk**-0.5, row_off, vis, page_off, pages,
                                 None if b is None else _f64(b), pos))
        assert torch.equal(got, paged.paged_attention(pool, 1, plan, q, bias=b, scale=scale))  # the same bits again


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,rows", [(5000, 1), (20011, 3), (3003, 40)])
def test_attention_long_sequence(n, rows, dtype):
    """A list that is split over many items, joined from their parts."""
    rng = np.random.default_rng(n)
    pool = _pool(heads=2, pages=n // 16 + 9)
    page_off, pages, _ = _fill(pool, rng, [n, 7])
    row_off, vis = np.array([0, rows, rows + 1]), np.r_[np.arange(n - rows + 1, n + 1), 7]
    q = _rand(rng, (rows + 1, 4, 64), dtype, 0.3) * 2
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=4)
    for _ in range(3):  # the plan's counters are left as they were found
        got = paged.paged_attention(pool, 0, plan, q)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages))


def test_attention_many_short_sequences():
    """Enough units that a warp takes one each."""
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 70, 700).tolist()
    lens[3] = 1500  # one of them is split all the same
    pool = _pool(heads=2, pages=sum(-(-n // 16) for n in lens) + 1)
    page_off, pages, _ = _fill(pool, rng, lens)
    row_off, vis = np.arange(701), np.asarray(lens)
    q = _rand(rng, (700, 2, 64), torch.bfloat16, 0.3)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=2)
    for _ in range(2):
        got = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dqk,dv", [(32, 32), (64, 64), (32, 64), (64, 32), (96, 96), (128, 128)])
def test_attention_tiles_of_24_rows(dqk, dv, dtype):
    """Some 20 rows a segment with its shared heads: one tile each, of a
    segment that sees nothing, of split and of short lists, with extra keys."""
    rng = np.random.default_rng(dqk + 2 * dv)
    lens, nrow, heads, share = [0, 30, 3000, 333, 17, 64], [5, 6, 5, 4, 5, 7], 2, 4
    pool = _pool(heads=heads, dqk=dqk, dv=dv, pages=250)
    page_off, pages, slots = _fill(pool, rng, lens + [50])
    row_off = np.r_[0, np.cumsum(nrow)]
    vis = np.concatenate([[max(0, n - r + 1 + i) if n % 2 else n for i in range(r)] for n, r in zip(lens, nrow)])
    per = rng.integers(0, 4, len(vis))
    off = np.r_[0, np.cumsum(per)]
    slot = rng.choice(slots[sum(lens):], off[-1])
    pos = vis + per
    kpos = np.concatenate([vis[r] + np.arange(per[r]) for r in range(len(vis))])
    q = _rand(rng, (len(vis), heads * share, dqk), dtype, 0.3)
    bias = torch.tensor(rng.standard_normal((heads * share, 201)), dtype=torch.float32, device=DEV)
    for more, extra in (({}, None), (dict(row_extra_off=off, extra_slot=slot, extra_pos=kpos), (off, slot, kpos))):
        plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off[:7], pages=pages,
                                   num_q_heads=heads * share, positions=pos, **more)
        for b in (None, bias):
            for _ in range(2):  # the plan's counters are left as they were found
                got = paged.paged_attention(pool, 0, plan, q, bias=b)
            paged.check_status(pool)
            _compare(got, _reference(pool, 0, q, dqk**-0.5, row_off, vis, page_off, pages,
                                     None if b is None else _f64(b), pos, extra))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_tiles_of_24_rows_a_warp_each(dtype):
    rng = np.random.default_rng(24)
    lens = rng.integers(0, 40, 600).tolist()
    lens[5] = 1200
    pool = _pool(heads=2, pages=sum(-(-n // 16) for n in lens) + 1)
    page_off, pages, _ = _fill(pool, rng, lens)
    row_off, vis = 5 * np.arange(601), np.repeat(lens, 5)
    q = _rand(rng, (3000, 8, 64), dtype, 0.3)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=8)
    for _ in range(2):
        got = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens", [[0, 5, 40], [300, 900, 16]])
def test_attention_extra_keys(lens, dtype):
    """Suffix chains and own tokens after the visible prefix, rows without
    any, rows with nothing but them."""
    rng = np.random.default_rng(13)
    nrow = [3, 30, 5]
    pool = _pool(heads=2, pages=120)
    page_off, pages, slots = _fill(pool, rng, lens + [100])
    chain = slots[sum(lens):]  # a fourth sequence holds the chains
    row_off = np.r_[0, np.cumsum(nrow)]
    vis = np.repeat(lens, nrow)
    per = rng.integers(0, 6, len(vis))
    per[0] = 0
    off = np.r_[0, np.cumsum(per)]
    slot = rng.choice(chain, off[-1])
    pos = vis + per
    kpos = np.concatenate([vis[r] + np.arange(per[r]) for r in range(len(vis))])
    q = _rand(rng, (len(vis), 4, 64), dtype, 0.3)
    bias = torch.tensor(rng.standard_normal((4, 101)), dtype=torch.float32, device=DEV)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off[:4], pages=pages, num_q_heads=4,
                               positions=pos, row_extra_off=off, extra_slot=slot, extra_pos=kpos)
    got = paged.paged_attention(pool, 0, plan, q, bias=bias)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages, _f64(bias), pos, (off, slot, kpos)))


def test_attention_masks_of_the_lowest_value():
    """A bias of -inf leaves a key out, the type's lowest value ranks it last:
    a row whose every key has it weighs them by nothing else."""
    rng = np.random.default_rng(17)
    pool = _pool(heads=1, pages=8)
    page_off, pages, _ = _fill(pool, rng, [40])
    vis, pos = np.array([40, 40, 40, 3]), np.array([40, 40, 40, 0])
    q = _rand(rng, (4, 2, 64), torch.float32, 0.3)
    mp = 41
    plan = paged.AttentionPlan(pool, row_off=[0, 4], row_vis=vis, page_off=page_off, pages=pages, num_q_heads=2, positions=pos)
    lowest = torch.finfo(torch.float32).min
    bias = torch.zeros((2, 2 * mp - 1), device=DEV)
    bias[0, ::2] = -math.inf
    bias[1, ::2] = lowest
    got = paged.paged_attention(pool, 0, plan, q, bias=bias)
    b = _f64(bias)
    b[1, ::2] = -1e30
    _compare(got, _reference(pool, 0, q, 0.125, [0, 4], vis, page_off, pages, b, pos))
    none = torch.stack([torch.full((2 * mp - 1,), -math.inf, device=DEV), torch.full((2 * mp - 1,), lowest, device=DEV)])
    got = paged.paged_attention(pool, 0, plan, q, bias=none)
    assert not got[:, 0].any()
    _, v = paged.kv_read(pool, 0, pages[0] * 16 + np.arange(3), torch.float32)
    assert np.allclose(_f64(got[3, 1]), _f64(v[:, 0]).mean(0), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_scales_far_apart(dtype):
    """Blocks whose scales differ by many powers of two, rising and falling,
    and queries of any size."""
    rng = np.random.default_rng(19)
    pool = _pool(heads=1, pages=20)
    sizes = [1.0, 1e-6, 1e6, 1e-12, 3e4, 1e-3, 1e9, 1.0]
    page_off, pages, slots = _fill(pool, rng, [16 * len(sizes)], dtype=torch.float32)
    pool.begin_pages(pages)
    k = _rand(rng, (128, 1, 64), torch.float32, 0.5) * 0.05
    v = _rand(rng, (128, 1, 64), torch.float32, 0.5) * torch.tensor(np.repeat(sizes, 16), dtype=torch.float32, device=DEV)[:, None, None]
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
    vis = np.array([128, 16, 32, 48, 64, 100, 128, 128])
    q = _rand(rng, (8, 1, 64), dtype, 0.3)
    q[6] *= 1e-20
    q[7] *= 1e4
    plan = paged.AttentionPlan(pool, row_off=[0, 8], row_vis=vis, page_off=page_off, pages=pages, num_q_heads=1)
    got = paged.paged_attention(pool, 0, plan, q)
    _compare(got, _reference(pool, 0, q, 0.125, [0, 8], vis, page_off, pages))


def test_attention_not_finite_queries_stay_in_their_rows():
    rng = np.random.default_rng(23)
    pool = _pool(heads=1, pages=8)
    page_off, pages, _ = _fill(pool, rng, [50])
    q = _rand(rng, (6, 2, 64), torch.bfloat16, 0.3)
    plan = paged.AttentionPlan(pool, row_off=[0, 6], row_vis=[50, 50, 0, 50, 50, 50], page_off=page_off, pages=pages, num_q_heads=2)
    good = paged.paged_attention(pool, 0, plan, q)
    q[1, 0, 3] = math.nan
    q[2] = math.nan  # sees nothing
    q[4, 1] = math.inf
    got = paged.paged_attention(pool, 0, plan, q)
    assert torch.isnan(got[1, 0]).all() and torch.isnan(got[4, 1]).all() and not got[2].any()
    for r, h in ((0, 0), (0, 1), (1, 1), (3, 0), (3, 1), (4, 0), (5, 0), (5, 1)):
        assert torch.equal(got[r, h], good[r, h])


@pytest.mark.parametrize("rows", [7, 100])
def test_attention_bias_at_extreme_positions(rows):
    """Positions at both ends of int32: every key is far before or behind,
    and the columns are the table's first and last."""
    rng = np.random.default_rng(rows)
    big = 2**31 - 1
    pool = _pool(heads=1, pages=20)
    page_off, pages, slots = _fill(pool, rng, [150, 20])
    row_off, vis = np.array([0, rows]), np.full(rows, 150)
    pos = rng.choice([-big - 1, -big, -(2**30), -1, 0, 75, 2**30, big - 100, big - 1, big], rows)
    pos[:4] = -big - 1, big, big - 4, 60
    q = _rand(rng, (rows, 1, 64), torch.bfloat16, 0.3)
    bias = torch.tensor(rng.standard_normal((1, 21)), dtype=torch.float32, device=DEV)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off[:2], pages=pages[:10], num_q_heads=1, positions=pos)
    got = paged.paged_attention(pool, 0, plan, q, bias=bias)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages, _f64(bias), pos))
    off, slot = 2 * np.arange(rows + 1), rng.choice(slots[150:], 2 * rows)
    kpos = np.where(np.repeat(pos, 2) > 0, np.repeat(pos, 2) - rng.integers(0, 9, 2 * rows), rng.choice([0, 3, big], 2 * rows))
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off[:2], pages=pages[:10], num_q_heads=1,
                               positions=pos, row_extra_off=off, extra_slot=slot, extra_pos=kpos)
    got = paged.paged_attention(pool, 0, plan, q, bias=bias)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages, _f64(bias), pos, (off, slot, kpos)))


@pytest.mark.parametrize("rows", [6, 20, 100])
def test_attention_bias_not_a_number(rows):
    """A NaN in the bias makes the rows NaN that see its key, and no others;
    behind what a row sees it does nothing."""
    rng = np.random.default_rng(rows)
    n = 150
    pool = _pool(heads=1, pages=20)
    page_off, pages, _ = _fill(pool, rng, [n])
    row_off, vis, pos = np.array([0, rows]), rng.integers(0, n + 1, rows), np.arange(rows)
    q = _rand(rng, (rows, 2, 64), torch.bfloat16, 0.3)
    table = rng.standard_normal((2, 2 * 256 - 1))
    odd = table.copy()
    column = 60 + 255
    odd[1, column] = math.nan
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=2, positions=pos)
    got = paged.paged_attention(pool, 0, plan, q, bias=torch.tensor(odd, dtype=torch.float32, device=DEV))
    paged.check_status(pool)
    sees = torch.tensor(vis > pos + 60, device=DEV)
    assert sees.any() and not sees.all()
    assert torch.isnan(got[sees, 1]).all()
    bias = torch.tensor(table, dtype=torch.float32, device=DEV)
    want, tol = _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages, _f64(bias), pos)
    hit = sees.cpu().numpy()
    assert np.isfinite(_f64(got)[:, 0]).all() and np.isfinite(_f64(got)[~hit]).all()
    off = np.abs(_f64(got) - want)
    assert (off[:, 0] <= tol[:, 0]).all() and (off[~hit] <= tol[~hit]).all()


def test_attention_strides_and_rows_left_alone():
    """Strided queries and outputs; rows behind the last sequence keep what
    they held."""
    rng = np.random.default_rng(29)
    pool = _pool(heads=2, pages=16)
    page_off, pages, _ = _fill(pool, rng, [100, 30])
    row_off, vis = np.array([0, 2, 5]), np.array([100, 7, 30, 29, 28, 5, 5])
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=4)
    for pad in (8, 3):  # aligned for vectors, and not
        wide = _rand(rng, (7, 4, 64 + pad), torch.bfloat16, 0.3)
        room = torch.full((7, 5, 64 + pad), 9.0, dtype=torch.bfloat16, device=DEV)
        q, out = wide[..., pad:], room[:, 1:, pad:]
        assert paged.paged_attention(pool, 0, plan, q, out=out) is out
        paged.check_status(pool)
        _compare(out[:5], _reference(pool, 0, q[:5], 0.125, row_off, vis, page_off, pages))
        assert torch.equal(out[:5], paged.paged_attention(pool, 0, plan, q.contiguous())[:5])
        assert (room[5:] == 9).all() and (room[:, 0] == 9).all() and (room[..., :pad] == 9).all()


def test_attention_reports_what_it_skips():
    rng = np.random.default_rng(31)
    pool = _pool(heads=1, pages=16)
    page_off, pages, _ = _fill(pool, rng, [100, 30])
    q = _rand(rng, (3, 1, 64), torch.float32, 0.3)
    row_off, vis = np.array([0, 2, 3]), np.array([100, 40, 30])

    def run(row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, **kw):
        plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=row_vis, page_off=page_off, pages=pages, num_q_heads=1, **kw)
        got = paged.paged_attention(pool, 0, plan, q)
        with pytest.raises(_native.ImbaError) as e:
            paged.check_status(pool)
        assert e.value.code == _native.IMBA_ERR_RANGE
        paged.check_status(pool)
        return got

    ref = _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages)
    for bad in (-1, 16, 2**31 - 1):
        wrong = pages.copy()
        wrong[0] = bad
        got = run(pages=wrong)
        assert np.isfinite(_f64(got)).all()
        _compare(got[2:], (ref[0][2:], ref[1][2:]))  # the other sequence is whole
    got = run(row_vis=np.array([100, 40, 33]))  # more than its pages hold: what they hold
    run(row_vis=np.array([100, 40, -1]))
    run(row_off=np.array([0, 2, 4]))
    run(row_off=np.array([2, 0, 3]))
    run(page_off=np.array([0, 7, 10]))
    run(row_extra_off=[0, 1, 1, 1], extra_slot=[16 * 16], extra_pos=[0])
    run(row_extra_off=[0, 5, 1, 1], extra_slot=[1], extra_pos=[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads,share,d", [(2, 1, 64), (1, 5, 64), (1, 2, 128)])
def test_attention_many_rows(heads, share, d, dtype):
    """Segments of many rows (tiles of 128 on the tensor cores, or of fewer
    rows by parts): causal parts and whole ones, some that see nothing, ends
    inside a page, a block and a tile, a bias that ends inside."""
    rng = np.random.default_rng(heads * 100 + share * 10 + d)
    lens = [0, 1, 16, 63, 64, 65, 130, 300]
    nrow = [70, 65, 64, 130, 80, 65, 130, 90]
    pool = _pool(heads=heads, dqk=d, dv=d, pages=60, layers=2)
    page_off, pages, _ = _fill(pool, rng, lens, layer=1)
    row_off = np.r_[0, np.cumsum(nrow)]
    vis = np.concatenate([[max(0, n - r + 1 + i) if n % 2 else n for i in range(r)] for n, r in zip(lens, nrow)])
    pos = vis + rng.integers(0, 4, len(vis))
    q = _rand(rng, (len(vis), heads * share, d), dtype, 0.3)
    bias = torch.tensor(rng.standard_normal((heads * share, 201)), dtype=torch.float32, device=DEV)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages,
                               num_q_heads=heads * share, positions=pos)
    for b, scale in ((None, None), (bias, -0.3)):
        got = paged.paged_attention(pool, 1, plan, q, bias=b, scale=scale)
        paged.check_status(pool)
        _compare(got, _reference(pool, 1, q, scale or d**-0.5, row_off, vis, page_off, pages,
                                 None if b is None else _f64(b), pos))
        assert torch.equal(got, paged.paged_attention(pool, 1, plan, q, bias=b, scale=scale))


@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_rows_split(d):
    """Few tiles over long lists: their parts are joined."""
    rng = np.random.default_rng(d)
    pool = _pool(heads=1, dqk=d, dv=d, pages=520)
    n, rows = [5001, 3000], [70, 65]
    page_off, pages, _ = _fill(pool, rng, n)
    row_off = np.array([0, 70, 135])
    vis = np.r_[5001 - 69 + np.arange(70), np.full(65, 3000)]
    q = _rand(rng, (135, 2, d), torch.bfloat16, 0.3)
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=2)
    for _ in range(3):
        got = paged.paged_attention(pool, 0, plan, q)
    paged.check_status(pool)
    _compare(got, _reference(pool, 0, q, d**-0.5, row_off, vis, page_off, pages))
    for x in (q.float(), q):  # the same plan for fp32 rows, and back
        got = paged.paged_attention(pool, 0, plan, x)
    _compare(got, _reference(pool, 0, q, d**-0.5, row_off, vis, page_off, pages))


def test_attention_many_rows_scales_far_apart():
    """V scales that differ within a block of 64 keys, by more than one
    reference holds: rows that see the small ones alone keep their precision."""
    rng = np.random.default_rng(43)
    pool = _pool(heads=1, pages=20)
    sizes = [1.0, 1e-6, 1e6, 1e-12, 3e4, 1e-3, 1e9, 1.0, 1e-9, 1e-9, 1e-9, 1e-9, 2.0, 1e-2]
    page_off, pages, slots = _fill(pool, rng, [16 * len(sizes)], dtype=torch.float32)
    pool.begin_pages(pages)
    n = len(slots)
    k = _rand(rng, (n, 1, 64), torch.float32, 0.5) * 0.05
    v = _rand(rng, (n, 1, 64), torch.float32, 0.5) * torch.tensor(np.repeat(sizes, 16), dtype=torch.float32, device=DEV)[:, None, None]
    paged.kv_append(pool, 0, paged.AppendPlan(pool, slots), k, v)
    vis = np.r_[np.arange(0, 130), np.full(20, n), np.arange(150, 200)]
    bias = np.zeros((1, 2 * n - 1))
    bias[0, : n - 1 - 30] = -60.0  # keys more than 30 back count for little: late rows see small V's
    bias = torch.tensor(bias, dtype=torch.float32, device=DEV)
    q = _rand(rng, (len(vis), 1, 64), torch.bfloat16, 0.3)
    row_off = np.array([0, len(vis)])
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=1, positions=vis)
    for b in (None, bias):
        got = paged.paged_attention(pool, 0, plan, q, bias=b)
        paged.check_status(pool)
        _compare(got, _reference(pool, 0, q, 0.125, row_off, vis, page_off, pages, None if b is None else _f64(b), vis))


def test_attention_many_rows_other_cases():
    """Not finite queries stay in their rows, strided rows, rows left alone
    and bad pages, on tiles of 128 rows."""
    rng = np.random.default_rng(47)
    pool = _pool(heads=1, pages=16)
    page_off, pages, _ = _fill(pool, rng, [100, 40])
    row_off, vis = np.array([0, 70, 140]), np.r_[np.full(70, 100), np.arange(70) % 41, [5, 5]]
    wide = _rand(rng, (142, 2, 67), torch.bfloat16, 0.3)
    room = torch.full((142, 3, 67), 9.0, dtype=torch.bfloat16, device=DEV)
    q, out = wide[..., 3:], room[:, 1:, 3:]
    plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=2)
    paged.paged_attention(pool, 0, plan, q, out=out)
    paged.check_status(pool)
    _compare(out[:140], _reference(pool, 0, q[:140], 0.125, row_off, vis, page_off, pages))
    good = paged.paged_attention(pool, 0, plan, q.contiguous())[:140]
    assert torch.equal(out[:140], good)
    assert (room[140:] == 9).all() and (room[:, 0] == 9).all() and (room[..., :3] == 9).all()
    odd = q.contiguous()
    odd[3, 1, 7], odd[5, 0, 0] = math.nan, math.inf
    got = paged.paged_attention(pool, 0, plan, odd)[:140]
    assert torch.isnan(got[3, 1]).all() and torch.isnan(got[5, 0]).all()
    got[3, 1], got[5, 0] = good[3, 1], good[5, 0]
    assert torch.equal(got, good)
    for bad in (-1, 16, 2**31 - 1):
        wrong = pages.copy()
        wrong[1] = bad
        plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=wrong, num_q_heads=2)
        got = paged.paged_attention(pool, 0, plan, q.contiguous())[:140]
        with pytest.raises(_native.ImbaError):
            paged.check_status(pool)
        assert torch.isfinite(got).all() and torch.equal(got[70:], good[70:])


def test_operators_together_under_a_graph():
    """Decode steps as a program runs them: a plan per step, append and
    attention for every layer, captured and replayed on another stream; the
    same bits as eager calls."""
    rng = np.random.default_rng(37)
    layers, heads, hq, d, start = 3, 2, 4, 64, [0, 15, 16, 130]
    pools = [_pool(layers=layers, heads=heads, pages=64) for _ in range(2)]
    rotary = paged.Rotary([100 ** (-i / 32) for i in range(32)], device=DEV)
    seqs = []
    for pool in pools:
        s = [KVSequence(pool) for _ in start]
        slots = KVSequence.reserve_many(s, start)
        r = np.random.default_rng(1)
        for l in range(layers):
            paged.kv_append(pool, l, paged.AppendPlan(pool, slots), _rand(r, (sum(start), heads, d)), _rand(r, (sum(start), heads, d)))
        seqs.append(s)
    n = len(start)
    q, k, v = (torch.empty((layers, n, h, d), dtype=torch.bfloat16, device=DEV) for h in (hq, heads, heads))
    pos = torch.empty(n, dtype=torch.int32, device=DEV)
    slot_buf, vis_buf = (torch.empty(n, dtype=torch.int32, device=DEV) for _ in range(2))
    for s in seqs[0]:
        s.reserve(20)  # pages ahead of time, so that the captured page lists stay as they are
    pools[0].begin_pages()
    page_off = np.r_[0, np.cumsum([len(s.pages) for s in seqs[0]])].astype(np.int32)
    pages = np.concatenate([s.pages for s in seqs[0]]).astype(np.int32)
    static = {"page_off": torch.tensor(page_off, device=DEV), "pages": torch.tensor(pages, device=DEV),
              "row_off": torch.arange(n + 1, dtype=torch.int32, device=DEV)}

    def step(pool, slots, vis, page_off, pages, row_off):
        rows = paged.AppendPlan(pool, slots)
        sees = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=page_off, pages=pages, num_q_heads=hq)
        outs = []
        for l in range(layers):
            turned = paged.kv_append(pool, l, rows, k[l], v[l], rotary=rotary, positions=pos, q=q[l])
            outs.append(paged.paged_attention(pool, l, sees, turned))
        return torch.stack(outs), (rows, sees)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    fill = lambda t: t.copy_(_rand(rng, tuple(t.shape)))  # noqa: E731
    slot_buf.fill_(-1)
    vis_buf.zero_()
    for t in (q, k, v):
        fill(t)
    pos.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        captured, keep = step(pools[0], slot_buf, vis_buf, **static)
    for i in range(18):
        for t in (q, k, v):
            fill(t)
        at = np.asarray(start) + i
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        slot_buf.copy_(torch.tensor([s.pages[a // 16] * 16 + a % 16 for s, a in zip(seqs[0], at)], dtype=torch.int32))
        vis_buf.copy_(torch.tensor(at + 1, dtype=torch.int32))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.current_stream().wait_stream(stream)
        mine = KVSequence.reserve_many(seqs[1], [1] * n)
        lists = [s.pages for s in seqs[1]]
        eager, _ = step(pools[1], mine, at + 1, np.r_[0, np.cumsum([len(p) for p in lists])], np.concatenate(lists),
                        np.arange(n + 1))
        assert torch.equal(captured, eager), i
    for pool in pools:
        paged.check_status(pool)
    ref = _reference(pools[1], 2, q[2][:1], 0.125, [0, 1], [start[0] + 18], [0, len(seqs[1][0].pages)], seqs[1][0].pages)
    turned = _turn(_f64(q[2][:1]), [start[0] + 17], [100 ** (-i / 32) for i in range(32)])
    ref = _reference(pools[1], 2, torch.tensor(turned, dtype=torch.bfloat16, device=DEV), 0.125, [0, 1], [start[0] + 18],
                     [0, len(seqs[1][0].pages)], seqs[1][0].pages)
    # the rotated query is rounded to bf16: an element on the border of two values may fall to the other one
    assert np.abs(_f64(eager[2][:1]) - ref[0]).max() <= 0.05 * np.abs(ref[0]).max()


def test_plans_on_another_stream_keep_their_memory():
    """A plan that is dropped while another stream still runs on it."""
    pool = _pool()
    rng = np.random.default_rng(53)
    k, v, q = (_rand(rng, (4, h, 64)) for h in (2, 2, 2))
    stream = torch.cuda.Stream()
    rows = paged.AppendPlan(pool, [0, 1, 2, 3])
    sees = paged.AttentionPlan(pool, row_off=[0, 4], row_vis=[1, 2, 3, 4], page_off=[0, 1], pages=[0], num_q_heads=2)
    held = [(len(p._plan), p._plan.data_ptr()) for p in (rows, sees)]
    paged.kv_append(pool, 0, rows, k, v)
    want = paged.paged_attention(pool, 0, sees, q)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)
        paged.kv_append(pool, 0, rows, k, v)
        got = paged.paged_attention(pool, 0, sees, q)
    del rows, sees
    fresh = [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for n, _ in held for _ in range(4)]
    assert not {t.data_ptr() for t in fresh} & {at for _, at in held}
    torch.cuda.synchronize()
    paged.check_status(pool)
    assert torch.equal(got, want)


def test_pool_past_32_bits():
    """Pages whose bytes lie past 2^32, in the last layer."""
    rng = np.random.default_rng(59)
    pool = _pool(layers=16, heads=8, pages=17000)  # 4.5 GB
    assert pool.page_bytes * 16900 > 2**32
    ids = np.array([16999, 3, 16990, 16500, 16998])
    slots = (ids[:, None] * 16 + np.arange(16)).reshape(-1)[:75]
    k, v = (_rand(rng, (75, 8, 64)) for _ in range(2))
    paged.kv_append(pool, 15, paged.AppendPlan(pool, slots), k, v)
    paged.check_status(pool)
    got = paged.kv_read(pool, 15, slots, torch.float32)
    for mine, want in zip(got, (k, v)):  # half a step of e4m3, at least that of the block's smallest codes
        assert (np.abs(_f64(mine) - _f64(want)) <= np.maximum(2.0**-4 * np.abs(_f64(want)), 2.0**-10 * 2 * np.abs(_f64(want)).max() / 448)).all()
    for rows in (1, 90):
        q = _rand(rng, (rows, 8, 64), torch.bfloat16, 0.3)
        row_off, vis = np.array([0, rows]), np.full(rows, 75)
        plan = paged.AttentionPlan(pool, row_off=row_off, row_vis=vis, page_off=[0, 5], pages=ids, num_q_heads=8)
        out = paged.paged_attention(pool, 15, plan, q)
        paged.check_status(pool)
        _compare(out, _reference(pool, 15, q, 0.125, row_off, vis, [0, 5], ids))
    low = paged.kv_read(pool, 15, np.arange(48, 64), torch.float32)  # page 3 holds its own tokens
    assert torch.equal(low[0], got[0][16:32])
    assert not paged.kv_read(pool, 14, slots, torch.float32)[0].any()


def test_refusals():
    pool, full = _pool(), _pool(torch.bfloat16)
    rng = np.random.default_rng(41)
    k, v, q = (_rand(rng, (4, h, 64)) for h in (2, 2, 4))
    plan = paged.AppendPlan(pool, [0, 1, 2, 3])
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    rotary = paged.Rotary([1.0, 0.5], device=DEV)
    bad = [
        dict(k=k[:3]), dict(v=v[:, :1]), dict(k=k.half(), v=v.half()), dict(v=v.float()), dict(k=k.cpu()),
        dict(q=q[:, :, :32]), dict(q=q.float()), dict(q_out=q), dict(q=q, q_out=q[:3]), dict(rotary=rotary),
        dict(rotary=rotary, positions=pos.long()), dict(rotary=rotary, positions=pos[:3]),
        dict(rotary=rotary, positions=pos[:, None].expand(4, 9)), dict(rotary=paged.Rotary([1.0, 0.5], device=DEV, axes=[0, 1]), positions=pos),
        dict(rotary=paged.Rotary([1.0] * 33, device=DEV), positions=pos),
        dict(rotary=paged.Rotary([1.0], device="cpu"), positions=pos), dict(plan=paged.AppendPlan(full, [0, 1, 2, 3])),
    ]
    for kw in bad:
        args = {"plan": plan, "k": k, "v": v, **kw}
        with pytest.raises(ValueError):
            paged.kv_append(pool, 0, args.pop("plan"), args.pop("k"), args.pop("v"), **args)
    with pytest.raises(_native.ImbaError):
        paged.kv_append(pool, 1, plan, k, v)
    for slots in ([[0]], [0.5], [2**31]):
        with pytest.raises(ValueError):
            paged.AppendPlan(pool, slots)
    rows = dict(row_off=[0, 4], row_vis=[1, 1, 1, 1], page_off=[0, 1], pages=[0], num_q_heads=4)
    with pytest.raises(ValueError, match="8 bits"):
        paged.AttentionPlan(full, **rows)
    for kw in (dict(num_q_heads=3), dict(num_q_heads=0), dict(row_off=[0]), dict(row_off=[]), dict(positions=[0]),
               dict(extra_slot=[0]), dict(extra_slot=[0], extra_pos=[0, 1], row_extra_off=[0] * 5),
               dict(extra_slot=[0], extra_pos=[0], row_extra_off=[0])):
        with pytest.raises(ValueError):
            paged.AttentionPlan(pool, **{**rows, **kw})
    sees = paged.AttentionPlan(pool, **rows)
    bias = torch.zeros((4, 9), device=DEV)
    for args, kw in (((q[:3],), {}), ((q.half(),), {}), ((q.transpose(1, 2).contiguous().transpose(1, 2),), {}),
                     ((q,), dict(out=q.float())), ((q,), dict(bias=bias)), ((q,), dict(bias=bias[:, :8]))):
        with pytest.raises(ValueError):
            paged.paged_attention(pool, 0, sees, *args, **kw)
    with pytest.raises(ValueError):
        paged.paged_attention(_pool(), 0, sees, q)
    with pytest.raises(_native.ImbaError):
        paged.paged_attention(pool, 7, sees, q)
    with pytest.raises(ValueError):
        paged.kv_read(full, 0, [0], torch.float32)
    torch.cuda.synchronize()
    paged.check_status(pool)


def test_empty_calls():
    pool = _pool()
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=DEV)
    q = paged.kv_append(pool, 0, paged.AppendPlan(pool, []), none, none, q=none)
    assert q.shape == none.shape
    k, v = paged.kv_read(pool, 0, [])
    assert k.shape == v.shape == none.shape
    plan = paged.AttentionPlan(pool, row_off=[0], row_vis=[], page_off=[0], pages=[], num_q_heads=2)
    assert paged.paged_attention(pool, 0, plan, none).shape == none.shape
    plan = paged.AttentionPlan(pool, row_off=[0, 1, 1, 2], row_vis=[0, 0], page_off=[0, 0, 0, 0], pages=[], num_q_heads=2)
    out = paged.paged_attention(pool, 0, plan, torch.ones((2, 2, 64), device=DEV))
    assert not out.any()
    paged.check_status(pool)
