"""CPU: pools made and used under torch's modes."""

from __future__ import annotations

import torch

from imba_chess_b200.kvpool import KVPool, KVSequence


def test_pool_made_in_inference_mode():
    """Its pages are emptied outside of that mode too."""
    with torch.inference_mode():
        pool = KVPool(num_layers=1, num_heads=2, attention_dim=64, linear_dim=64, num_pages=4, dtype=torch.float8_e4m3fn,
                      device=torch.device("cpu"))
        pool.scales.fill_(130)
    seq = KVSequence(pool)
    seq.reserve(20)
    pool.begin_pages()
    assert (pool.scales[seq.pages] == 0).all() and (pool.scales == 130).sum() == 2 * 4
    pool.status.zero_()
    with torch.inference_mode():
        pool.begin_pages([0, 1, 2, 3])
    assert not pool.scales.any()
