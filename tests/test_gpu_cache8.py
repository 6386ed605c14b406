"""GPU: a model whose KV pool is in 8 bits (``kv_dtype=torch.float8_e4m3fn``).

The steps are checked against the fp32 oracle run on the keys and values that
the pool holds (read back after the step and put in the place of the oracle's
own), to the bounds of the model's type; what the pool holds is checked
against the oracle's own keys and values to e4m3's rounding."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from imba_chess_b200 import _native, paged, synth
from imba_chess_b200.kvpool import KVSequence
from imba_chess_b200.model import B200HSTUChessModel
from imba_chess_b200.plan import DeviceStep, piece_ids_from_tokens, side_ids_from_tokens
from imba_chess_b200.server import ActorInferenceServer
from imba_chess_b200.steps import WaveGroup, root_plan, wave_plan
from oracle.hstu_np import OracleModel
from tests import golden_io
from tests.test_gpu_server import _replay

pytestmark = pytest.mark.gpu

ATOL = {torch.float32: 1e-4, torch.bfloat16: 3e-2}  # of logits: the bounds of the model's type
E4M3 = torch.float8_e4m3fn


class _Stored(OracleModel):
    """The oracle with each layer's new keys and values taken from a pool."""

    stored: list | None = None

    def uvqk(self, layer, x):
        u, v, q, k = super().uvqk(layer, x)
        if self.stored is not None:
            self.own.append((k, v))
            k, v = self.stored[layer]
        return u, v, q, k


def _model(dims, dtype, seed=9):
    sd = synth.make_state_dict(dims, seed, profile="reference")
    return B200HSTUChessModel(sd, dtype=dtype, device="cuda:0", kv_dtype=E4M3), _Stored(sd, dims)


def _read(model, pool, slots):
    """Per layer ([n, H, d_qk], [n, H, d_v]) of what the pool holds."""
    s = np.asarray(slots, np.int64)
    return [tuple(t.cpu().numpy() for t in paged.kv_read(pool, l, s, torch.float32))
            for l in range(model.dims.num_layers)]


def _run(model, pool, plan):
    R = plan.num_rows
    out = {"logits": torch.empty((R, model.dims.vocab), device=model.device),
           "value_logits": torch.empty((R, 3), device=model.device)}
    model.run(DeviceStep(plan, model.device), pool, **out)
    torch.cuda.synchronize()
    model.check_status()
    return {k: v.cpu().numpy() for k, v in out.items()}


def _close(got, ref, dtype):
    for k in ("logits", "value_logits"):
        assert np.isfinite(got[k]).all()
        assert np.abs(got[k] - ref[k]).max() <= ATOL[dtype], k


def _rounded(own, stored, dtype):
    """Stored rows are the oracle's to half a step of e4m3 (2^-4; 2^-10 of the
    scale for subnormal codes, and once more when the scale grew: the scale is
    at most 2^-8 of the block's largest magnitude, which is at most the
    layer's), past what the model's type leaves of them."""
    off_by = {torch.float32: 2.0**-16, torch.bfloat16: 2.0**-6}[dtype]
    for (k, v), (sk, sv) in zip(own, stored):
        for a, b in ((k, sk), (v, sv)):
            most = np.abs(a).max()
            assert (np.abs(a - b) <= np.abs(a) * 2.0**-4 + most * (2.0**-17 + off_by)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dims", [synth.SMALL, synth.D256], ids=["d128", "d256"])
def test_steps_match_oracle(dims, dtype):
    """A prefill of several documents, a wave of siblings and a wave with
    suffix chains, positions past max_pos among them (d128)."""
    model, oracle = _model(dims, dtype)
    pool = model.new_pool(256)
    rng = np.random.default_rng(1)
    lens = [1, 16, 33, 60]
    tokens = [synth.random_tokens(rng, n, dims) for n in lens]
    seqs = [KVSequence(pool) for _ in lens]
    plan, _ = root_plan(seqs, tokens)
    got = _run(model, pool, plan)
    prefix = [_read(model, pool, s.slots(0, n)) for s, n in zip(seqs, lens)]
    L = dims.num_layers
    oracle.stored, oracle.own = [tuple(np.concatenate([p[l][i] for p in prefix]) for i in (0, 1)) for l in range(L)], []
    ref = oracle.forward(synth.concat_tokens(tokens), np.r_[0, np.cumsum(lens)])
    _close(got, ref, dtype)
    _rounded(oracle.own, oracle.stored, dtype)

    most = max(lens)
    padded = []
    for l in range(L):
        kv = []
        for i in (0, 1):
            x = np.zeros((len(lens), dims.num_heads, most, dims.attention_dim), np.float32)
            for g, n in enumerate(lens):
                x[g, :, :n] = prefix[g][l][i].transpose(1, 0, 2)
            kv.append(x)
        padded.append(tuple(kv))
    counts = [7, 0, 20, 33]
    arenas = [KVSequence(pool) for _ in lens]
    chains = [[[]] * c for c in counts]
    for wave in range(2):
        n = sum(counts)
        tok = synth.random_tokens(rng, n, dims)
        plan, rows = wave_plan([WaveGroup(seqs[g], lens[g], arenas[g], chains[g]) for g in range(len(lens))],
                               piece_ids_from_tokens(tok), side_ids_from_tokens(tok), [[0]] * n)
        got = _run(model, pool, plan)
        group = np.repeat(np.arange(len(lens)), counts)
        own = np.concatenate([arenas[g].slots_of(rows[g]) for g in range(len(lens))])
        oracle.stored, oracle.own = _read(model, pool, own), []
        kw = {}
        if wave:
            parents = np.concatenate([arenas[g].slots_of([c[0] for c in chains[g]]) for g in range(len(lens))])
            kw = {"suffix_kv": [(k[:, :, None], v[:, :, None]) for k, v in _read(model, pool, parents)],
                  "suffix_positions": np.asarray(lens)[group][:, None], "suffix_mask": np.ones((n, 1), bool)}
        ref = oracle.forward_decode_grouped(new_token_batch=tok, positions=np.asarray(lens)[group] + wave, group_index=group,
                                            prefix_kv_grouped=padded, prefix_lens_list=lens, **kw)
        _close(got, ref, dtype)
        _rounded(oracle.own, oracle.stored, dtype)
        chains = [[[r] for r in rows[g]] for g in range(len(lens))]


def test_model_api():
    """forward(return_kv) and forward_decode_grouped on dense tensors: what
    they return as KV is what the pool held, and calls start afresh."""
    dims = synth.SMALL
    model, oracle = _model(dims, torch.float32)
    rng = np.random.default_rng(2)
    lens = [20, 7]
    tok = synth.random_tokens(rng, sum(lens), dims)
    batch = {**{k: torch.from_numpy(v) for k, v in tok.items()}, "seq_offsets": torch.tensor([0, 20, 27])}
    out = model.forward(batch, return_loss=False, return_kv=True)
    L = dims.num_layers
    oracle.stored, oracle.own = [tuple(x.transpose(0, 1).cpu().numpy() for x in kv) for kv in out["kv_caches"]], []
    ref = oracle.forward(tok, [0, 20, 27])
    _close({k: out[k].cpu().numpy() for k in ("logits", "value_logits")}, ref, torch.float32)
    prefix = []
    for k, v in out["kv_caches"]:
        pk, pv = torch.zeros((2, *k.shape), device=k.device), torch.zeros((2, *v.shape), device=v.device)
        for g, (a, b) in enumerate(((0, 20), (20, 27))):
            pk[g, :, : b - a], pv[g, :, : b - a] = k[:, a:b], v[:, a:b]
        prefix.append((pk, pv))
    new = synth.random_tokens(rng, 5, dims)
    group = np.array([0, 1, 1, 0, 1])
    suffix = [(torch.randn((5, dims.num_heads, 2, 64), device="cuda"), torch.randn((5, dims.num_heads, 2, 64), device="cuda"))
              for _ in range(L)]
    mask = np.array([[0, 0], [1, 0], [1, 1], [0, 1], [1, 1]], bool)
    call = dict(new_token_batch={k: torch.from_numpy(v) for k, v in new.items()}, positions=torch.tensor([22, 9, 9, 22, 9]),
                group_index=torch.from_numpy(group), prefix_kv_grouped=prefix, prefix_lens=torch.tensor(lens),
                prefix_lens_list=lens, suffix_kv=suffix, suffix_positions=torch.tensor([[20, 21], [7, 8], [7, 8], [20, 21], [7, 8]]),
                suffix_mask=torch.from_numpy(mask))
    got = model.forward_decode_grouped(**call)
    # the prefix holds stored values already, alone in their blocks: they come back as they were
    stored = []
    region = -(-20 // 16) * 16 + 16  # the scratch pool: both prefixes' pages, then each row's suffix and own token
    at, where = region, np.zeros((5, 2), int)
    for r in range(5):
        for j in range(2):
            if mask[r, j]:
                where[r, j] = at
                at += 1
        at += 1
    for l in range(L):
        stored.append(tuple(t.cpu().numpy() for t in paged.kv_read(model._scratch, l, where.reshape(-1), torch.float32)))
    oracle.stored, oracle.own = [tuple(x[:, :, 0].cpu().numpy() for x in kv) for kv in got["kv"]], []
    ref = oracle.forward_decode_grouped(
        new_token_batch=new, positions=call["positions"].numpy(), group_index=group,
        prefix_kv_grouped=[(k.cpu().numpy(), v.cpu().numpy()) for k, v in prefix], prefix_lens_list=lens,
        suffix_kv=[tuple(x.reshape(5, 2, *x.shape[1:]).transpose(0, 2, 1, 3) for x in kv) for kv in stored],
        suffix_positions=call["suffix_positions"].numpy(), suffix_mask=mask)
    _close({k: got[k].cpu().numpy() for k in ("logits", "value_logits")}, ref, torch.float32)
    again = model.forward_decode_grouped(**call)
    for k in ("logits", "value_logits"):
        assert torch.equal(got[k], again[k])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_server_session_on_recycled_pages(dtype):
    """The reference's scripted session, twice on one server: the same
    answers, arena rows and chains, so that pages that come back to the pool
    start afresh."""
    doc = golden_io.load_session()
    dims = synth.ModelDims(**{**doc["model"]["dims"], "model_dim": 128, "attention_dim": 64, "linear_dim": 64, "num_heads": 2})
    sd = synth.make_state_dict(dims, 3, profile="reference")
    model = B200HSTUChessModel(sd, dtype=dtype, device="cuda:0", kv_dtype=E4M3)
    server = ActorInferenceServer(model=model, device="cuda:0", dtype=dtype, kv_pool_pages=64, kv_dtype=E4M3)
    first = _replay(doc, server, check=False)
    chains = {f"{w},{t}": {str(n): c for n, c in ts.node_chains.items()} for (w, t), ts in server._turns.items()}
    assert chains == doc["node_chains"]
    for key in list(server._turns):
        server.release_turn(*key)
    for w in list(server._games):
        server.release_game(w)
    assert server.pool.free_pages == 64 and server.pool.scales.any()
    server.pool.data.view(torch.uint8).fill_(0x55)  # what the last sessions left must not matter
    second = _replay(doc, server, check=False)
    assert first == second


def test_refusals():
    sd = synth.make_state_dict(synth.SMALL, 1)
    with pytest.raises(ValueError, match="kv_dtype"):
        B200HSTUChessModel(sd, dtype=torch.bfloat16, device="cuda:0", kv_dtype=torch.float32)
    with pytest.raises(_native.ImbaError):  # head dims of 8
        B200HSTUChessModel(synth.make_state_dict(synth.TINY, 1), dtype=torch.float32, device="cuda:0", kv_dtype=E4M3)
    model8 = B200HSTUChessModel(sd, dtype=torch.bfloat16, device="cuda:0", kv_dtype=E4M3)
    model16 = B200HSTUChessModel(sd, dtype=torch.bfloat16, device="cuda:0")
    with pytest.raises(ValueError, match="kv_dtype|KV"):
        ActorInferenceServer(model=model16, device="cuda:0", dtype=torch.bfloat16, kv_pool_pages=64, kv_dtype=E4M3)
    rng = np.random.default_rng(0)
    for model, other in ((model8, model16), (model16, model8)):
        pool = other.new_pool(8)
        plan, _ = root_plan([KVSequence(pool)], [synth.random_tokens(rng, 3, synth.SMALL)])
        with pytest.raises(ValueError, match="pool"):
            model.run(DeviceStep(plan, model.device), pool)
        with pytest.raises(ValueError, match="pool"):
            model.kv_gather(pool, 0, torch.zeros(1, dtype=torch.int32, device="cuda"))
    # the C entry points that write dense rows as they are do not write codes
    pool = model8.new_pool(8)
    t = torch.zeros(4096, device="cuda")
    strides = (ctypes.c_int64 * 4)(1, 1, 1, 1)
    lib = _native.load()
    p = t.data_ptr()
    args = (model8._handle, ctypes.byref(pool.desc), 0, 1, p)
    assert lib.imba_kv_scatter(*args, p, p, None, None) == _native.IMBA_ERR_UNSUPPORTED
    assert lib.imba_kv_scatter_indexed(*args, p, p, p, p, strides, strides, None, None) == _native.IMBA_ERR_UNSUPPORTED
    k = torch.randn((2, 2, 64), device="cuda").bfloat16()
    slots = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    model8.kv_scatter(pool, 1, slots, k, k)  # the model's own does
    gk, gv = model8.kv_gather(pool, 1, slots)
    assert torch.equal(gk, gv) and (gk.float() - k.float()).abs().max() <= k.float().abs().max() * 2.0**-4
    with pytest.raises(_native.ImbaError):
        model8.kv_scatter(pool, 1, slots + 1000, k, k)
        model8.check_status()
