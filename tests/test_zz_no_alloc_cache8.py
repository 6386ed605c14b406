"""GPU: the allocation-free step on a handle whose KV pool is in 8 bits: the
scratch holds the plans of the append and of the attention too, for waves of
the documented size."""

from __future__ import annotations

import ctypes

import pytest
import torch

from imba_chess_b200 import _native, synth
from imba_chess_b200.kvpool import KVSequence
from imba_chess_b200.model import B200HSTUChessModel
from imba_chess_b200.plan import DeviceStep, piece_ids_from_tokens, side_ids_from_tokens
from imba_chess_b200.steps import WaveGroup, root_plan, wave_plan

pytestmark = pytest.mark.gpu

ROWS = 50  # at d512 / 8 layers / 8 heads


def _run(model, plan, pool, how):
    dev, lib = model.device, _native.load()
    ds = DeviceStep(plan, dev)
    R, NL = plan.num_rows, int(plan.legal_ids.shape[0])
    out = {"logits": torch.full((R, model.dims.vocab), float("nan"), device=dev),
           "value_logits": torch.full((R, 3), float("nan"), device=dev),
           "legal_logits": torch.full((NL,), float("nan"), device=dev)}
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    for k, t in out.items():
        setattr(ds.desc, k, t.data_ptr())
    ds.desc.status = status.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    pool.begin_pages()
    args = (model._handle, ctypes.byref(ds.desc), ctypes.byref(pool.desc))
    if how == "noalloc":
        assert lib.imba_step_noalloc(*args, stream) == _native.IMBA_OK
    else:
        ws = model.workspace(R)
        assert lib.imba_step(*args, ws.data_ptr(), ws.numel(), stream) == _native.IMBA_OK
    torch.cuda.synchronize()
    assert int(status.item()) == _native.IMBA_OK
    return out


@pytest.mark.parametrize("siblings", [(1, 1), (4, 6), (15, 16)])
def test_noalloc_step_on_a_pool_in_8_bits(siblings):
    """Waves of some rows a parent (tiles of 8, 16 and 24 rows), and their
    children's, with suffix chains: bit for bit what imba_step gives."""
    dims = synth.D512
    model = B200HSTUChessModel(synth.make_state_dict(dims, 21, profile="reference"), dtype=torch.bfloat16, device="cuda:0",
                               kv_dtype=torch.float8_e4m3fn)
    lib = _native.load()
    assert int(lib.imba_step_workspace_bytes(model._handle, ROWS)) <= _native.NOALLOC_SCRATCH_BYTES
    pool = model.new_pool(256)
    wave = synth.grouped_wave(dims, n_parents=3, plies=(5, 40), siblings=siblings, seed=7)
    seqs = [KVSequence(pool) for _ in wave.prefix_lens]
    model.run(DeviceStep(root_plan(seqs, wave.prefix_tokens)[0], model.device), pool)
    arenas = [KVSequence(pool) for _ in seqs]
    counts = [int((wave.group_index == g).sum()) for g in range(3)]
    chains = [[[]] * c for c in counts]
    n = sum(counts)
    assert n <= ROWS
    legal = list(wave.legal_ids)
    for _ in range(2):
        plan, rows = wave_plan([WaveGroup(seqs[g], wave.prefix_lens[g], arenas[g], chains[g]) for g in range(3)],
                               piece_ids_from_tokens(wave.row_tokens), side_ids_from_tokens(wave.row_tokens), legal)
        want = _run(model, plan, pool, "workspace")
        got = _run(model, plan, pool, "noalloc")
        for k in want:
            assert torch.isfinite(got[k]).all() and torch.equal(got[k], want[k]), k
        chains = [[[r] for r in rows[g]] for g in range(3)]
