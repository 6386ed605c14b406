"""What is measured of the cache operators: the calls a serving program makes per layer, beside their plain forms.

* ``append``: new tokens' keys and values into a paged cache, keys and queries rotated to their positions on the way
  (``imba_chess_b200.paged.kv_append``).  A cache in 8 bits keeps e4m3 values and, for each page of 16 tokens, head, and K or
  V, one power-of-two scale 2^e (the byte e + 127, 0: an empty block).  e is the smallest for which the block's largest
  magnitude is at most 448 * 2^e, never below -100, and never smaller than it was; when it grows, the block's
  earlier values are rounded to the new scale.
* ``attend``: attention over such a cache in 8 bits (``imba_chess_b200.paged.paged_attention``):
  row r sees the first ``vis[r]`` tokens of its sequence, with an optional relative-position bias; a row that sees nothing gets zeros.

A page's layout is [K: heads x 16 x d_qk | V: heads x 16 x d_v], and in 8 bits V's tokens lie in pairs, heads x 8 x d_v x 2.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
E4M3_MAX = 448.0
MIN_EXP = -100
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp32": 4, "e4m3": 1}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one game's next move: the smallest call a server makes, all latency
        _append("append one token", seqs=1, new=(1, 1), old=(137, 137), heads=8, q_heads=8, dqk=64, dv=64),
        # 1,024 games, one token each, d512 / 8 heads: pages that are begun, part-filled and full
        _append("append game step", seqs=1024, new=(1, 1), old=(1, 300), heads=8, q_heads=8, dqk=64, dv=64),
        # the prefill of 1,024 game prefixes of ragged length
        _append("append game prefixes", seqs=1024, new=(1, 300), old=(0, 0), heads=8, q_heads=8, dqk=64, dv=64),
        # four long documents continued far from their start, shared key / value heads
        _append("append long documents", seqs=4, new=(9000, 16384), old=(5, 40), heads=8, q_heads=32, dqk=128, dv=128,
                first=200_000),
        # boards as (ply, rank, file) tokens: three rotation axes, pairs side by side, part of the head rotated, a cache in full
        # precision, keys and values as slices of one projection
        _append("append board squares", seqs=31, new=(64, 64), old=(0, 100), heads=4, q_heads=4, dqk=96, dv=96, dtype="fp32",
                pool="fp32", layout="interleaved", rot=72, axes=3, fused=True),
        # one game's next move
        _attend("attend one game", seqs=1, rows=(1, 1), old=(137, 137), heads=8, q_heads=8, dqk=64, dv=64, bias=True),
        # 1,024 games, one token each
        _attend("attend game step", seqs=1024, rows=(1, 1), old=(1, 300), heads=8, q_heads=8, dqk=64, dv=64, bias=True),
        # a search wave: 256 parents with every legal move as a sibling row
        _attend("attend sibling wave", seqs=256, rows=(20, 40), old=(20, 200), heads=8, q_heads=8, dqk=64, dv=64, bias=True),
        # ragged long sequences, one new token each, shared key / value heads
        _attend("attend long sequences", seqs=32, rows=(1, 1), old=(4000, 32768), heads=8, q_heads=32, dqk=128, dv=128),
        # one far sequence, a few drafted tokens at once
        _attend("attend one far sequence", seqs=1, rows=(5, 5), old=(131_000, 131_000), heads=8, q_heads=32, dqk=128, dv=128,
                causal=True),
        # the next part of four prompts over what the cache holds of them
        _attend("attend prompt part", seqs=4, rows=(512, 512), old=(2000, 8000), heads=16, q_heads=16, dqk=64, dv=64, causal=True),
        # the exact-precision model's queries over a short ragged cache
        _attend("attend in fp32", seqs=96, rows=(1, 7), old=(0, 2500), heads=4, q_heads=4, dqk=64, dv=64, dtype="fp32", causal=True),
    ]


def _append(name, *, seqs, new, old, heads, q_heads, dqk, dv, dtype="bf16", pool="e4m3", layout="half", rot=None, axes=1, first=0,
            fused=False, lens=1):
    c = {"op": "append", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "old_lo": old[0], "old_hi": old[1], "heads": heads,
         "q_heads": q_heads, "dqk": dqk, "dv": dv, "dtype": dtype, "pool": pool, "layout": layout, "rot": dqk if rot is None else rot,
         "axes": axes, "first": first, "fused": fused, "lens": lens}
    return {"name": name, **c} if name else c


def _attend(name, *, seqs, rows, old, heads, q_heads, dqk, dv, dtype="bf16", bias=False, causal=False, lens=1):
    c = {"op": "attend", "seqs": seqs, "new_lo": rows[0], "new_hi": rows[1], "old_lo": old[0], "old_hi": old[1], "heads": heads,
         "q_heads": q_heads, "dqk": dqk, "dv": dv, "dtype": dtype, "bias": bias, "causal": causal, "lens": lens}
    return {"name": name, **c} if name else c


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    heads = rng.choice([1, 2, 3, 4, 8, 16])
    dqk, dv = rng.choice([(64, 64), (64, 64), (128, 128), (128, 128), (32, 32), (96, 96), (32, 64), (64, 32)])
    c = {"seqs": _log(rng, 1, 1024), "heads": heads, "q_heads": heads * rng.choice([1, 1, 2, 3, 4, 8]), "dqk": dqk, "dv": dv,
         "lens": rng.randrange(1 << 30)}
    if rng.random() < 0.5:
        lo, hi, old = rng.random(), _log(rng, 1, 16384), rng.choice([0, _log(rng, 1, 300)])
        c.update(dtype=rng.choice(["bf16", "bf16", "fp32"]), pool=rng.choice(["e4m3", "e4m3", "e4m3", "bf16", "fp32"]),
                 layout=rng.choice(["half", "half", "interleaved"]), axes=rng.choice([1, 1, 1, 2, 3]),
                 rot=2 * rng.randint(1, dqk // 2) if rng.random() < 0.4 else dqk, first=rng.choice([0, _log(rng, 1, 1_000_000)]),
                 fused=rng.random() < 0.3 and dqk == dv, old=(rng.randint(0, old), old))
        while work(case := _append(None, new=(max(1, int(lo * hi)), hi), **c))["bytes"] > 8e8 and hi > 1:
            hi = -(-hi // 2)  # no larger than the largest listed case
        return case
    rows_lo, rows, old_lo, old = rng.random(), rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 512)]), rng.random(), _log(rng, 1, 131_000)
    c.update(dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]), bias=rng.random() < 0.4, causal=rng.random() < 0.5)
    while True:
        case = _attend(None, rows=(max(1, int(rows_lo * rows)), rows), old=(int(old_lo * old), old), **c)
        w = work(case)
        if (w["bytes"] <= 8e8 and w["flops"] <= 3e10) or rows * old <= 1:
            return case
        rows, old = (-(-rows // 2), old) if rows > 64 or old <= 1 else (rows, -(-old // 2))


def _lengths(case):
    """(tokens held before, new tokens or rows) of each sequence: of the case alone."""
    r = random.Random(case["lens"])
    lo, hi = case["old_lo"], case["old_hi"]
    spread = _log if lo >= 1 and hi > 10 * lo else (lambda g, a, b: g.randint(a, b))
    olds = [spread(r, lo, hi) for _ in range(case["seqs"])]
    lo, hi = case["new_lo"], case["new_hi"]
    spread = _log if hi > 10 * lo else (lambda g, a, b: g.randint(a, b))
    news = [spread(r, lo, hi) for _ in range(case["seqs"])]
    return olds, news


def _held(case, olds, news):
    """Tokens that each sequence's pages hold during the call: a causal row is itself one of them."""
    add = case["op"] == "append" or case["causal"]
    return [o + n if add else o for o, n in zip(olds, news)]


def work(case):
    olds, news = _lengths(case)
    held, n = _held(case, olds, news), sum(news)
    h, hq, dqk, dv, e = case["heads"], case["q_heads"], case["dqk"], case["dv"], BYTES[case["dtype"]]
    if case["op"] == "append":
        pe = BYTES[case["pool"]]
        byte = n * h * (dqk + dv) * (e + pe) + 2 * n * hq * dqk * e + n * 4 * (1 + case["axes"])
        return {"bytes": byte, "flops": 3 * n * (h + hq) * case["rot"] + 2 * n * h * (dqk + dv)}
    pages = sum(-(-t // PAGE) for t in held)
    byte = sum(held) * h * (dqk + dv) + pages * (2 * h + 4) + n * hq * (dqk + dv) * e + n * 4
    seen = sum(m * o + m * (m + 1) // 2 if case["causal"] else m * o for o, m in zip(olds, news))
    return {"bytes": byte, "flops": 2 * seen * hq * (dqk + dv)}


# --------------------------------------------------------------------------------------------------------------- inputs
def _values(gen, n, heads, dim, dtype):
    """Keys or values as projections give them: normal, channels of unequal size, now and then a large one."""
    x = torch.randn((n, heads, dim), generator=gen, device="cuda", dtype=torch.float32)
    size = torch.exp2(torch.randn((heads, dim), generator=gen, device="cuda"))
    token = torch.exp2(0.5 * torch.randn((n, 1, 1), generator=gen, device="cuda"))
    return (x * size * token).to(dtype)


def _inputs(case, seed):
    """The call's inputs and what the cache held before it (rows of tokens, not yet in any cache)."""
    olds, news = _lengths(case)
    held = _held(case, olds, news)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h, hq, dqk, dv, dt = case["heads"], case["q_heads"], case["dqk"], case["dv"], DTYPES[case["dtype"]]
    pages = [-(-t // PAGE) for t in held]
    s = {"case": case, "olds": olds, "news": news, "held": held, "num_pages": max(1, sum(pages))}
    ids = torch.randperm(s["num_pages"], generator=gen, device="cuda")  # pages in no order, as a pool hands them out
    first = torch.tensor([0] + pages, device="cuda").cumsum(0)
    s["pages"], s["page_off"] = ids[: sum(pages)].int(), first.int()

    def slots(starts, counts):
        n = torch.tensor(counts, device="cuda")
        seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), n)
        t = torch.arange(int(sum(counts)), device="cuda") - (n.cumsum(0) - n)[seq] + torch.tensor(starts, device="cuda")[seq]
        return ids[(first[seq] + t // PAGE).clamp(max=s["num_pages"] - 1)] * PAGE + t % PAGE, seq, t

    n = sum(news)
    if case["op"] == "append":
        s["old_slots"], _, _ = slots([0] * len(olds), olds)
        s["old_k"] = _values(gen, sum(olds), h, dqk, dt)
        s["old_v"] = _values(gen, sum(olds), h, dv, dt)
        s["slots"], _, t = slots(olds, news)
        s["slots"] = s["slots"].int()
        if case["fused"]:
            both = _values(gen, n, hq + 2 * h, dqk, dt)
            s["q"], s["k"], s["v"] = both[:, :hq], both[:, hq : hq + h], both[:, hq + h :]
        else:
            s["q"], s["k"], s["v"] = _values(gen, n, hq, dqk, dt), _values(gen, n, h, dqk, dt), _values(gen, n, h, dv, dt)
        pos = (t + case["first"]).int()
        if case["axes"] > 1:  # the token's ply, then where it stands on the board
            pos = torch.stack([pos // 64, pos % 64 // 8, pos % 8][: case["axes"]], 1).contiguous()
        s["positions"] = pos
        half = case["rot"] // 2
        s["inv_freq"] = [10000.0 ** (-p / half) for p in range(half)]
        s["axis"] = [p * case["axes"] // half for p in range(half)]
        return s
    s["old_slots"], _, _ = slots([0] * len(held), held)
    s["old_k"], s["old_v"] = _values(gen, sum(held), h, dqk, torch.bfloat16), _values(gen, sum(held), h, dv, torch.bfloat16)
    row_seq = torch.repeat_interleave(torch.arange(len(news), device="cuda"), torch.tensor(news, device="cuda"))
    s["row_off"] = torch.tensor([0] + news, device="cuda").cumsum(0).int()
    row = torch.arange(n, device="cuda") - s["row_off"].long()[row_seq]
    old = torch.tensor(olds, device="cuda")[row_seq]
    s["vis"] = (old + row + 1 if case["causal"] else old).int()
    s["row_pos"] = (s["vis"] - 1 if case["causal"] else old).int()
    s["q"] = (torch.randn((n, hq, dqk), generator=gen, device="cuda") * 0.7).to(dt)
    s["max_pos"] = max(2, max(held) // 2 + 3)  # some distances lie beyond the table's ends
    s["bias"] = 0.5 * torch.randn((hq, 2 * s["max_pos"] - 1), generator=gen, device="cuda") if case["bias"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    h, dqk, dv = case["heads"], case["dqk"], case["dv"]
    pool = case.get("pool", "e4m3")
    k, v, old_slots = s.pop("old_k"), s.pop("old_v"), s.pop("old_slots")
    if own:
        from imba_chess_b200 import paged
        from imba_chess_b200.kvpool import KVPool

        dev = torch.device("cuda", torch.cuda.current_device())
        s["pool"] = KVPool(num_layers=1, num_heads=h, attention_dim=dqk, linear_dim=dv, num_pages=s["num_pages"],
                           dtype=DTYPES[pool], device=dev)
        if k.shape[0]:
            paged.kv_append(s["pool"], 0, paged.AppendPlan(s["pool"], old_slots.int()), k, v)
        if case["op"] == "append":
            s["rotary"] = paged.Rotary(s["inv_freq"], layout=case["layout"], axes=s["axis"] if case["axes"] > 1 else None, device=dev)
            s["plan"] = paged.AppendPlan(s["pool"], s["slots"])
            s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=dev)
        else:
            s["plan"] = paged.AttentionPlan(s["pool"], row_off=s["row_off"], row_vis=s["vis"], page_off=s["page_off"],
                                            pages=s["pages"], num_q_heads=case["q_heads"],
                                            positions=s["row_pos"] if case["bias"] else None)
        return s
    s["data"] = torch.zeros((s["num_pages"], h * PAGE * (dqk + dv)), dtype=DTYPES[pool], device="cuda")
    s["scales"] = torch.zeros((s["num_pages"], 2, h), dtype=torch.uint8, device="cuda") if pool == "e4m3" else None
    if k.shape[0]:
        _store(s, old_slots, k.float(), v.float())
    return s


# ----------------------------------------------------------------------------------------------------------------- runs
def run(s):
    if s["case"]["op"] == "append":
        return _append_own(s) if own else _append_plain(s)
    return _attend_own(s) if own else _attend_plain(s)


def _append_own(s):
    from imba_chess_b200 import paged

    q = paged.kv_append(s["pool"], 0, s["plan"], s["k"], s["v"], rotary=s["rotary"], positions=s["positions"], q=s["q"],
                        q_out=s["q_out"])
    out = {"pages": s["pool"].data, "q": q}
    return out if s["pool"].scales is None else {**out, "scales": s["pool"].scales[:, 0].view(torch.float8_e8m0fnu)}


def _attend_own(s):
    from imba_chess_b200 import paged

    return paged.paged_attention(s["pool"], 0, s["plan"], s["q"], bias=s["bias"])


def _blocks(s):
    """The pages' K as [page, head, 16, d_qk] and V as [page, head, pair, 2, d_v] in 8 bits or [page, head, 16, d_v]: views."""
    c, n = s["case"], s["num_pages"]
    cut = c["heads"] * PAGE * c["dqk"]
    k = s["data"][:, :cut].view(n, c["heads"], PAGE, c["dqk"])
    if s["scales"] is None:
        return k, s["data"][:, cut:].view(n, c["heads"], PAGE, c["dv"])
    return k, s["data"][:, cut:].view(n, c["heads"], PAGE // 2, c["dv"], 2).transpose(3, 4)


def _store(s, slots, k, v):
    """Float rows into the pages."""
    kb, vb = _blocks(s)
    slots = slots.long()
    page, at = slots // PAGE, slots % PAGE
    if s["scales"] is None:
        kb[page, :, at] = k.to(kb.dtype)
        vb[page, :, at] = v.to(vb.dtype)
        return
    for part, (block, x) in enumerate(((kb, k), (vb, v))):
        most = torch.zeros(s["num_pages"], x.shape[1], device=x.device)
        most.scatter_reduce_(0, page[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        frac, exp = torch.frexp(most)
        byte = (exp - 9 + (frac > E4M3_MAX / 512)).clamp(min=MIN_EXP) + 127
        before = s["scales"][:, part].int()
        byte = torch.maximum(before, torch.where(most > 0, byte, 0))
        s["scales"][:, part] = byte.to(torch.uint8)
        lead = (slice(None), slice(None)) + (None,) * (block.dim() - 2)
        block.copy_(torch.ldexp(block.float(), (before - byte)[lead]).to(block.dtype))
        codes = torch.ldexp(x, (127 - byte)[page][:, :, None]).to(block.dtype).view(torch.uint8)
        if part == 0:
            block.view(torch.uint8)[page, :, at] = codes
        else:
            block.view(torch.uint8)[page, :, at // 2, at % 2] = codes


def _rotate(x, s):
    c = s["case"]
    pos = s["positions"].double().reshape(x.shape[0], -1)
    axis = torch.tensor(s["axis"], device=x.device)
    angle = pos[:, axis] * torch.tensor(s["inv_freq"], dtype=torch.float64, device=x.device)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x, out = x.float(), x.float().clone()
    rot = c["rot"]
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if c["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def _append_plain(s):
    _store(s, s["slots"], _rotate(s["k"], s), s["v"].float())
    out = {"pages": s["data"], "q": _rotate(s["q"], s).to(s["q"].dtype)}
    return out if s["scales"] is None else {**out, "scales": s["scales"].view(torch.float8_e8m0fnu)}


def _attend_plain(s):
    c = s["case"]
    h, dqk, dv = c["heads"], c["dqk"], c["dv"]
    share = c["q_heads"] // h
    n, seqs, rows = s["q"].shape[0], c["seqs"], max(s["news"])
    longest = max(1, -(-max(s["held"]) // PAGE))
    kb, vb = _blocks(s)
    # every sequence's pages side by side, padded to the longest
    lo = s["page_off"].long()
    at = (lo[:-1, None] + torch.arange(longest, device="cuda")).clamp(max=s["pages"].numel() - 1)
    table = s["pages"].long()[at] if s["pages"].numel() else torch.zeros_like(at)
    scale = torch.exp2(s["scales"].float() - 127)[table]
    k = kb.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[:, :, 0, :, None, None]
    v = vb.contiguous().view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[:, :, 1, :, None, None, None]
    k = k.transpose(1, 2).reshape(seqs, h, longest * PAGE, dqk)
    v = v.transpose(1, 2).reshape(seqs, h, longest * PAGE, dv)
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), s["row_off"].diff().long(), output_size=n)
    row = torch.arange(n, device="cuda") - s["row_off"].long()[seq]
    q = torch.zeros((seqs, rows, h, share, dqk), device="cuda")
    q[seq, row] = s["q"].float().view(n, h, share, dqk)
    vis = torch.zeros((seqs, rows), dtype=torch.long, device="cuda")
    vis[seq, row] = s["vis"].long()
    scores = q.permute(0, 2, 3, 1, 4).reshape(seqs, h, share * rows, dqk) @ k.transpose(2, 3) / math.sqrt(dqk)
    scores = scores.view(seqs, h, share, rows, longest * PAGE)
    key = torch.arange(longest * PAGE, device="cuda")
    if s["bias"] is not None:
        pos = torch.zeros((seqs, rows), dtype=torch.long, device="cuda")
        pos[seq, row] = s["row_pos"].long()
        far = (key - pos[..., None] + s["max_pos"] - 1).clamp(0, 2 * s["max_pos"] - 2)
        scores = scores + s["bias"][:, far].view(h, share, seqs, rows, -1).permute(2, 0, 1, 3, 4)
    scores = scores.masked_fill((key >= vis[..., None])[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    out = (p.view(seqs, h, share * rows, -1) @ v).view(seqs, h, share, rows, dv) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 3, 1, 2, 4)[seq, row].reshape(n, c["q_heads"], dv).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------------------- exact
def _to_e4m3(x):
    """Round to the nearest e4m3 value, ties to an even last digit; |x| is at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(x / step) * step


def _fit(most):
    """The exponent for a block whose largest magnitude is `most`."""
    e = torch.ceil(torch.log2(most.clamp(min=1e-300) / E4M3_MAX))
    e = torch.where(E4M3_MAX * torch.exp2(e - 1) >= most, e - 1, e)
    e = torch.where(E4M3_MAX * torch.exp2(e) < most, e + 1, e)
    return e.clamp(min=MIN_EXP)


def _exact_blocks(num_pages, calls, paired):
    """The pages' codes and scale bytes after the calls [(slots, rows in 64 bits)], one after the other."""
    heads, dim = calls[0][1].shape[1:]
    codes = torch.zeros((num_pages * PAGE, heads, dim), dtype=torch.float64, device="cuda")
    exp = torch.full((num_pages, heads), -127.0, dtype=torch.float64, device="cuda")
    for slots, x in calls:
        if not x.shape[0]:
            continue
        most = torch.zeros((num_pages, heads), dtype=torch.float64, device="cuda")
        most.index_reduce_(0, slots // PAGE, x.abs().amax(2), "amax")
        new = torch.where(most > 0, torch.maximum(exp, _fit(most)), exp)
        shrink = torch.repeat_interleave(torch.exp2(exp - new), PAGE, 0)
        codes = _to_e4m3(codes * shrink[..., None])
        codes[slots] = _to_e4m3(x / torch.exp2(new)[slots // PAGE][..., None])
        exp = new
    blocks = codes.view(num_pages, PAGE, heads, dim).transpose(1, 2)
    if paired:
        flat = blocks.reshape(num_pages, heads, PAGE // 2, 2, dim).transpose(3, 4).reshape(num_pages, -1)
    else:
        flat = blocks.reshape(num_pages, -1)
    return blocks, flat, exp


def _exact_turn(x, s):
    """The rotation as a product of complex numbers."""
    rot = s["case"]["rot"]
    pos = s["positions"].to(torch.float64).reshape(x.shape[0], -1)
    angle = torch.stack([pos[:, a] * f for a, f in zip(s["axis"], s["inv_freq"])], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    x = x.double()
    part = x[..., :rot]
    if s["case"]["layout"] == "half":
        z = torch.complex(part[..., : rot // 2], part[..., rot // 2 :]) * turn
        part = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(part.reshape(*part.shape[:2], -1, 2).contiguous()) * turn
        part = torch.view_as_real(z).flatten(-2)
    return torch.cat([part, x[..., rot:]], -1)


def exact(case, seed):
    s = _inputs(case, seed)
    n = s["num_pages"]
    if case["op"] == "append":
        new = (_exact_turn(s["k"], s), s["v"].double())
        old, slots = (s["old_k"].double(), s["old_v"].double()), s["slots"].long()
        if case["pool"] == "e4m3":
            parts = [_exact_blocks(n, [(s["old_slots"], old[i]), (slots, new[i])], i == 1) for i in (0, 1)]
            scales = torch.exp2(torch.stack([p[2] for p in parts], 1))
            return {"pages": torch.cat([p[1] for p in parts], 1), "q": _exact_turn(s["q"], s), "scales": scales}
        flat = []
        for i in (0, 1):
            rows = torch.zeros((n * PAGE, *new[i].shape[1:]), dtype=torch.float64, device="cuda")
            rows[s["old_slots"]], rows[slots] = old[i], new[i]
            flat.append(rows.view(n, PAGE, *new[i].shape[1:]).transpose(1, 2).reshape(n, -1))
        return {"pages": torch.cat(flat, 1), "q": _exact_turn(s["q"], s)}
    out = torch.zeros((s["q"].shape[0], case["q_heads"], case["dv"]), dtype=torch.float64, device="cuda")
    share = case["q_heads"] // case["heads"]
    r = t = 0
    for held, rows in zip(s["held"], s["news"]):  # one sequence after the other, on pages of its own
        if held:
            pages = -(-held // PAGE)
            slots = torch.arange(held, device="cuda")
            kv = []
            for x in (s["old_k"], s["old_v"]):
                b, _, e = _exact_blocks(pages, [(slots, x[t : t + held].double())], False)
                x = (b * torch.exp2(e)[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :held]
                kv.append(x.repeat_interleave(share, 0))
            q = s["q"][r : r + rows].double().transpose(0, 1)
            w = torch.einsum("hrd,hkd->hrk", q, kv[0]) / case["dqk"] ** 0.5
            ahead = slots[None, :] - s["row_pos"][r : r + rows, None]
            if s["bias"] is not None:
                w = w + s["bias"].double()[:, (ahead + s["max_pos"] - 1).clamp(0, 2 * s["max_pos"] - 2)]
            w = torch.where(slots[None, None, :] < s["vis"][None, r : r + rows, None], w, -math.inf)
            out[r : r + rows] = torch.einsum("hrk,hkd->rhd", torch.softmax(w, -1), kv[1])
        r, t = r + rows, t + held
    return out
