"""Operators on a paged KV pool: appending rotated keys and values, and
attention over a pool held in 8 bits.

A serving program makes the plans once per step and calls the operators for
every layer::

    pool = KVPool(..., dtype=torch.float8_e4m3fn)
    rotary = Rotary([10000 ** (-i / 32) for i in range(32)], device=pool.device)
    rows = AppendPlan(pool, slots)                     # where the step's tokens go
    sees = AttentionPlan(pool, row_off=..., row_vis=..., page_off=..., pages=..., num_q_heads=32)
    for layer in range(pool.num_layers):
        q = kv_append(pool, layer, rows, k, v, rotary=rotary, positions=positions, q=q)
        out = paged_attention(pool, layer, sees, q)

They stand beside ``B200HSTUChessModel.kv_scatter`` / ``kv_gather`` (rows of a
model's own pool, as they are); a model with ``kv_dtype=torch.float8_e4m3fn``
runs its steps on them.  Everything is enqueued on the current stream of the
pool's device and nothing but ``check_status`` waits for the device (host lists
and arrays are copied through pinned memory): what only the device can see
(a slot or a page outside the pool, a row that is not finite) is skipped,
written to ``pool``'s status word and raised by ``check_status(pool)``.

A plan keeps the tensors it was made from and its scratch: calls on one plan
must not overlap (two streams, two captured graphs), and int32 tensors that were
on the device already are used as they are, so leave them as they were when the
plan was made.  A call on another stream than the plan's waits for nothing by
itself, as with any tensor, and marks the plan's memory as used there; a captured
graph needs its plans kept alive.  A pool in 8 bits orders its streams where it
empties pages (``kvpool``).
"""

from __future__ import annotations

import ctypes
import math
import struct
from fractions import Fraction

import torch

from . import _native
from .kvpool import PAGE, KVPool, to_device

_PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16}
_POOL_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _native.DTYPE_E4M3}
_MAX_AXES = 8
_FNS: dict = {}
# imba_append_desc and imba_attend_args as one struct.pack each: these calls run once per layer
_APPEND = struct.Struct("@4i5P12q4i3PP")
_ATTEND = struct.Struct("@2i2P4qfiP")
assert _APPEND.size == ctypes.sizeof(_native.AppendDesc) and _ATTEND.size == ctypes.sizeof(_native.AttendArgs)


def _cache(pool: KVPool):
    """The pool's geometry for the library, and its status word."""
    got = getattr(pool, "_cache", None)
    if got is None:
        if pool.device.type != "cuda" or pool.dtype not in _POOL_DTYPES:
            raise ValueError(f"the cache operators take a CUDA pool in fp32, bf16 or e4m3, got {pool.dtype} on {pool.device}")
        if max(pool.attention_dim, pool.linear_dim) > 128:
            raise ValueError("the cache operators take head dimensions up to 128")
        desc = _native.CacheDesc(pool.num_layers, pool.num_heads, pool.attention_dim, pool.linear_dim,
                                 _POOL_DTYPES[pool.dtype])
        got = pool._cache = (ctypes.byref(desc), ctypes.byref(pool.desc), pool.status, desc)
    return got


def check_status(pool: KVPool) -> None:
    """Raise ``ImbaError`` if an operator on this pool reported one (waits for
    the current stream)."""
    status = _cache(pool)[2]
    code = int(status.item())
    if code != _native.IMBA_OK:
        status.zero_()
        raise _native.ImbaError(code, "device-side check")


# the current stream's handle, without a Stream object where torch has the short way
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(pool: KVPool, what: str, *args, plan=None) -> None:
    """One library call on the current stream of the pool's device."""
    index = pool.data.get_device()
    fn = _FNS.get(what) or _FNS.setdefault(what, getattr(_native.load(), what))
    stream = _raw_stream(index)
    if pool.scales is not None and stream not in pool._ordered:
        pool.join_stream()
    if plan is not None and stream != plan._stream:
        _used_on(plan, index)
    if torch.cuda.current_device() == index:
        code = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            code = fn(*args, stream)
    if code:
        _native.check(code, what)


def _used_on(plan, index: int) -> None:
    """The plan's memory is not handed out again before the current stream,
    which is not the one that it was made on, has passed this call."""
    with torch.cuda.device(index):
        if not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream()
            for t in plan._memory:
                t.record_stream(stream)


def _ints(x, pool: KVPool, what: str, shape: tuple[int, ...] | None = None) -> torch.Tensor:
    """A contiguous int32 tensor on the pool's device.  Wider integers that are
    on the device already are clamped, not wrapped: what was outside int32 is
    then outside every pool and is reported there."""
    t = x if isinstance(x, torch.Tensor) else torch.as_tensor(x, device="cpu")
    if t.numel() and (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool):
        raise ValueError(f"{what} must be integers")
    if t.dtype != torch.int32 and not t.is_cuda and t.numel() and (int(t.max()) > 2**31 - 1 or int(t.min()) < -(2**31)):
        raise ValueError(f"{what} has values outside int32")
    if t.is_cuda and t.device != pool.data.device:
        raise ValueError(f"{what} is on {t.device}, the pool on {pool.data.device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{what} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_cuda:
        return to_device(t.to(torch.int32).contiguous(), pool.data.device)
    if t.dtype == torch.int64:
        t = t.clamp(-(2**31), 2**31 - 1)
    elif t.dtype in (torch.uint32, torch.uint64):
        raise ValueError(f"{what} on the device must be int32 or int64, got {t.dtype}")
    return t.to(torch.int32).contiguous()


def _rows(t: torch.Tensor, pool: KVPool, what: str, shape: tuple[int, ...], dtype) -> None:
    if t.dtype != dtype or t.shape != shape or t.get_device() != pool.data.get_device():
        raise ValueError(f"{what} must be {dtype} {shape} on {pool.data.device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _apart(t: torch.Tensor, what: str) -> None:
    """An output whose elements share no memory (an expanded tensor's do)."""
    if t.is_contiguous():
        return
    need = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride < need:
                raise ValueError(f"{what} has elements that share memory: shape {tuple(t.shape)}, strides {t.stride()}")
            need += stride * (size - 1)


class Rotary:
    """Rotary positions: pair ``p`` of a head turns by ``positions[axis[p]] *
    inv_freq[p]`` radians.  ``inv_freq`` has one value per pair, in the order
    of the pairs; ``layout`` "half" pairs element p with p + len(inv_freq),
    "interleaved" 2 p with 2 p + 1; the head's other elements pass through.
    ``axes`` gives each pair's position axis (time, height, width, ...) when
    tokens have several positions.  Angles are kept as 64-bit fractions of a
    turn, so they stay right at any position."""

    def __init__(self, inv_freq, *, device, layout: str = "half", axes=None) -> None:
        freq = [float(f) for f in inv_freq]
        if layout not in ("half", "interleaved"):
            raise ValueError(f"unknown rotary layout {layout!r}")
        if not 1 <= len(freq) <= 64 or not all(math.isfinite(f) for f in freq):
            raise ValueError("inv_freq must hold 1 to 64 finite values")
        self.num_axes = 1
        self.axis: torch.Tensor | None = None
        device = torch.device(device)
        if axes is not None:
            axes = [int(a) for a in axes]
            if len(axes) != len(freq) or min(axes) < 0 or max(axes) >= _MAX_AXES:
                raise ValueError(f"axes must give each pair an axis in [0, {_MAX_AXES})")
            self.num_axes = max(axes) + 1
            self.axis = torch.tensor(axes, dtype=torch.int32, device=device)
        turns = [round(Fraction(f) / (2 * _PI) * 2**64) % 2**64 for f in freq]
        self.turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64, device=device)
        self.rot_dim = 2 * len(freq)
        self.layout = layout


class AppendPlan:
    """A step's rows by the pages they go to: row r's token is stored in slot
    ``slots[r]`` (page * 16 + offset; -1: a padding row).  Of rows with the
    same slot the last one is stored.  ``status`` (int32 ``[1]``) is the word
    that errors go to, the pool's by default."""

    def __init__(self, pool: KVPool, slots, *, status: torch.Tensor | None = None) -> None:
        _, desc, pool_status, _ = _cache(pool)
        if status is None:
            status = pool_status
        else:
            _rows(status, pool, "status", (1,), torch.int32)
        self._status = status
        self.pool = pool
        self.slots = _ints(slots, pool, "slots")
        if self.slots.dim() != 1:
            raise ValueError("slots must be one-dimensional")
        self.num_rows = int(self.slots.shape[0])
        need = int(_native.load().imba_append_plan_bytes(self.num_rows))
        if need == 0:
            raise ValueError(f"too many rows for one step: {self.num_rows}")
        self._plan = torch.empty(need, dtype=torch.uint8, device=pool.data.device)
        self._desc = ctypes.create_string_buffer(_APPEND.size)
        self._refs = (ctypes.cast(self._desc, ctypes.POINTER(_native.AppendDesc)), self._plan.data_ptr(), need,
                      self.slots.data_ptr(), status.data_ptr())
        self._memory = (self._plan, self.slots, status)
        self._stream = _raw_stream(self._plan.get_device())
        _call(pool, "imba_append_plan", desc, self.num_rows, self.slots.data_ptr(), self._plan.data_ptr(), need,
              status.data_ptr())


def kv_append(pool: KVPool, layer: int, plan: AppendPlan, k: torch.Tensor, v: torch.Tensor, *,
              rotary: Rotary | None = None, positions: torch.Tensor | None = None, q: torch.Tensor | None = None,
              q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store a step's keys ``[n, H, d_qk]`` and values ``[n, H, d_v]`` (fp32
    or bf16, any strides) in one layer of the pool, the keys rotated to
    ``positions`` (int32 ``[n]``, or ``[n, axes]``) when ``rotary`` is given.
    ``q`` ``[n, q_heads, d_qk]`` is rotated along and returned, in ``q_out`` or
    a new tensor.  ``q_out`` may be ``q``, and shares no memory with what else
    the call reads.  Rows without a slot are left as they were: in a new tensor
    they hold nothing defined."""
    cache, desc, _, _ = _cache(pool)
    if plan.pool is not pool:
        raise ValueError("the plan was made for another pool")
    n, dqk = plan.num_rows, pool.attention_dim
    dtype = k.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"keys and values must be fp32 or bf16, got {dtype}")
    _rows(k, pool, "k", (n, pool.num_heads, dqk), dtype)
    _rows(v, pool, "v", (n, pool.num_heads, pool.linear_dim), dtype)
    q_heads, q_ptrs, q_strides = 0, (0, 0), (0, 0, 0, 0, 0, 0)
    if q is not None:
        if q.dim() != 3 or dqk % 2:
            raise ValueError("q must be [n, q_heads, d_qk] with an even d_qk")
        _rows(q, pool, "q", (n, q.shape[1], dqk), dtype)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=q.device)
        else:
            _rows(q_out, pool, "q_out", q.shape, dtype)
            _apart(q_out, "q_out")
            if q_out.data_ptr() == q.data_ptr() and any(
                    a != b for a, b, size in zip(q.stride(), q_out.stride(), q.shape) if size > 1):
                raise ValueError("q_out overlaps q in another order")
        if q.numel():
            q_heads, q_ptrs, q_strides = q.shape[1], (q.data_ptr(), q_out.data_ptr()), (*q.stride(), *q_out.stride())
    elif q_out is not None:
        raise ValueError("q_out without q")
    turns = (0, 0, 0, 0, 0, 0, 0)
    if rotary is not None:
        if rotary.rot_dim > dqk:
            raise ValueError(f"the rotation takes {rotary.rot_dim} elements, a head has {dqk}")
        if rotary.turns.device != pool.data.device:
            raise ValueError("rotary is on another device than the pool")
        if positions is None:
            raise ValueError("a rotation needs positions")
        one = positions.dim() == 1
        axes = 1 if one else int(positions.shape[-1])
        if not rotary.num_axes <= axes <= _MAX_AXES:
            raise ValueError(f"the rotation takes {rotary.num_axes} positions a row, got {axes}")
        _rows(positions, pool, "positions", (n,) if one else (n, axes), torch.int32)
        positions = positions.contiguous()
        turns = (rotary.rot_dim, rotary.layout == "interleaved", axes, 0, rotary.turns.data_ptr(),
                 0 if rotary.axis is None else rotary.axis.data_ptr(), positions.data_ptr())
    if pool._fresh:
        pool.begin_pages()
    ref, ptr, size, slots, status = plan._refs
    _APPEND.pack_into(plan._desc, 0, n, layer, _DTYPES[dtype], q_heads, slots, k.data_ptr(), v.data_ptr(), *q_ptrs,
                      *k.stride(), *v.stride(), *q_strides, *turns, status)
    _call(pool, "imba_kv_append", cache, desc, ref, ptr, size, plan=plan)
    return q_out


def kv_read(pool: KVPool, layer: int, slots, dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The tokens in ``slots`` as dense ``[n, H, d_qk]`` and ``[n, H, d_v]``,
    in the pool's type; from a pool in 8 bits in bf16, which holds every stored
    value, or fp32.  Rows of slots outside the pool hold nothing defined."""
    cache, desc, status, _ = _cache(pool)
    dtype = dtype or (torch.bfloat16 if pool.dtype == torch.float8_e4m3fn else pool.dtype)
    if dtype not in _DTYPES or (pool.dtype != torch.float8_e4m3fn and dtype != pool.dtype):
        raise ValueError(f"a {pool.dtype} pool is not read as {dtype}")
    slots = _ints(slots, pool, "slots").reshape(-1)
    n = int(slots.shape[0])
    k = torch.empty((n, pool.num_heads, pool.attention_dim), dtype=dtype, device=pool.data.device)
    v = torch.empty((n, pool.num_heads, pool.linear_dim), dtype=dtype, device=pool.data.device)
    _call(pool, "imba_kv_read", cache, desc, int(layer), n, slots.data_ptr(), _DTYPES[dtype], k.data_ptr(),
          v.data_ptr(), status.data_ptr())
    return k, v


class AttentionPlan:
    """What a step's rows see of a pool in 8 bits.

    Rows ``row_off[g] .. row_off[g + 1]`` are of sequence ``g``, whose tokens
    lie in ``pages[page_off[g] .. page_off[g + 1]]``; row ``r`` sees the first
    ``row_vis[r]`` of them (a causal row its own token too: position + 1) and
    then its extra keys, if given: slots ``extra_slot[row_extra_off[r] ..
    row_extra_off[r + 1]]`` (a suffix chain, the row's own token).
    ``positions`` (and ``extra_pos``) are for a relative-position bias.  All
    are int32; on the device they are used as they are."""

    def __init__(self, pool: KVPool, *, row_off, row_vis, page_off, pages, num_q_heads: int, positions=None,
                 row_extra_off=None, extra_slot=None, extra_pos=None) -> None:
        cache, desc, status, _ = _cache(pool)
        if pool.dtype != torch.float8_e4m3fn:
            raise ValueError(f"attention runs over a pool in 8 bits, got {pool.dtype}")
        if num_q_heads <= 0 or num_q_heads % pool.num_heads:
            raise ValueError(f"num_q_heads must be a multiple of the pool's {pool.num_heads} heads")
        self.pool, self.num_q_heads = pool, int(num_q_heads)
        row_vis = _ints(row_vis, pool, "row_vis").reshape(-1)
        self.num_rows = int(row_vis.shape[0])
        row_off, page_off, pages = (_ints(x, pool, n).reshape(-1) for x, n in (
            (row_off, "row_off"), (page_off, "page_off"), (pages, "pages")))
        if row_off.shape[0] < 1 or row_off.shape != page_off.shape:
            raise ValueError("row_off and page_off must hold one more entry than there are sequences")
        seqs = int(row_off.shape[0]) - 1
        keep = {"seg_row_off": row_off, "row_vis": row_vis, "group_page_off": page_off, "group_pages": pages}
        if positions is not None:
            keep["positions"] = _ints(positions, pool, "positions", (self.num_rows,))
        extra = 0
        if extra_slot is not None:
            if row_extra_off is None or extra_pos is None:
                raise ValueError("extra_slot needs row_extra_off and extra_pos")
            keep["extra_slot"] = _ints(extra_slot, pool, "extra_slot").reshape(-1)
            extra = int(keep["extra_slot"].shape[0])
            keep["extra_pos"] = _ints(extra_pos, pool, "extra_pos", (extra,))
            keep["row_extra_off"] = _ints(row_extra_off, pool, "row_extra_off", (self.num_rows + 1,))
        self._keep = keep
        d = self._desc = _native.AttendDesc(self.num_rows, seqs, seqs, int(pages.shape[0]), extra, self.num_q_heads)
        for name, t in keep.items():
            setattr(d, name, t.data_ptr())
        d.status = status.data_ptr()
        need = int(_native.load().imba_attend_plan_bytes(cache, ctypes.byref(d)))
        if need == 0:
            raise ValueError("too many rows, pages or extra keys for one step")
        self._plan = torch.empty(need, dtype=torch.uint8, device=pool.data.device)
        self._args = ctypes.create_string_buffer(_ATTEND.size)
        self._refs = (ctypes.byref(d), ctypes.cast(self._args, ctypes.POINTER(_native.AttendArgs)),
                      self._plan.data_ptr(), need)
        self._memory = (self._plan, status, *keep.values())
        self._stream = _raw_stream(self._plan.get_device())
        _call(pool, "imba_attend_plan", cache, desc, ctypes.byref(d), self._plan.data_ptr(), need)


def paged_attention(pool: KVPool, layer: int, plan: AttentionPlan, q: torch.Tensor, *, scale: float | None = None,
                    bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q . k + bias) v of each row over what its plan says it
    sees: ``q`` ``[n, q_heads, d_qk]`` (fp32 or bf16; the last dimension
    contiguous) to ``out`` ``[n, q_heads, d_v]`` of the same type.  ``scale``
    is 1 / sqrt(d_qk) by default; ``bias`` is fp32 ``[q_heads, 2 max_pos -
    1]``, its column the key's position less the row's, clamped, plus max_pos
    - 1.  A row that sees nothing gets zeros; a row of no sequence is left as
    it was, and holds nothing defined in a new tensor.  ``out`` may be ``q``."""
    cache, desc, _, _ = _cache(pool)
    if plan.pool is not pool:
        raise ValueError("the plan was made for another pool")
    n, heads, dtype = plan.num_rows, plan.num_q_heads, q.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"queries must be fp32 or bf16, got {dtype}")
    _rows(q, pool, "q", (n, heads, pool.attention_dim), dtype)
    if out is None:
        out = torch.empty((n, heads, pool.linear_dim), dtype=dtype, device=q.device)
    else:
        _rows(out, pool, "out", (n, heads, pool.linear_dim), dtype)
        _apart(out, "out")
    if q.stride(2) != 1 or out.stride(2) != 1:
        raise ValueError("the last dimension of q and out must be contiguous")
    column, max_pos = 0, 0
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] % 2 == 0 or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [q_heads, 2 max_pos - 1]")
        _rows(bias, pool, "bias", (heads, bias.shape[1]), torch.float32)
        if not plan._desc.positions:
            raise ValueError("a bias needs the plan's positions")
        column, max_pos = bias.data_ptr(), (bias.shape[1] + 1) // 2
    rows, args, ptr, size = plan._refs
    (q0, q1, _), (o0, o1, _) = q.stride(), out.stride()
    _ATTEND.pack_into(plan._args, 0, layer, _DTYPES[dtype], q.data_ptr(), out.data_ptr(), q0, q1, o0, o1,
                      pool.attention_dim**-0.5 if scale is None else scale, max_pos, column)
    _call(pool, "imba_attend", cache, desc, rows, args, ptr, size, plan=plan)
    return out
