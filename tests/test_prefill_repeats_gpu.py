"""The packed prefill of long ragged prompts gives the same K and V rows every time,
and the oracle's; where it does not, the message says which rows, heads and dims
differ, by how much, and what the device status word holds."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LENS = [2900, 517, 3333]
REPEATS = 40


def _where(what, got, want):
    """Differing entries of [heads, rows, dims] as text."""
    from bitnet_tt import _lib

    bad = (got != want) & ~(got.isnan() & want.isnan())
    heads, rows, dims = (torch.nonzero(bad.any(-1).any(-1)).flatten().tolist(),
                         torch.nonzero(bad.any(-1).any(0)).flatten().tolist(),
                         torch.nonzero(bad.any(0).any(0)).flatten().tolist())
    most = float((got.float() - want.float()).abs().nan_to_num(nan=float("inf")).max())
    return (f"{what}: {int(bad.sum())} values differ by up to {most:.4g}; heads {heads}; {len(rows)} rows "
            f"{rows[:4]} .. {rows[-4:]} (tiles of 256: {sorted({r // 256 for r in rows})[:12]}); {len(dims)} dims "
            f"{dims[:8]}; device status {_lib.last_device_status()}")


def test_packed_prefill_rows_repeat_and_are_the_oracles(cuda):
    from bitnet_tt.config import BitNetConfig
    from bitnet_tt.inference import Batch32Generator
    from bitnet_tt.model import create_model
    from bitnet_tt.utils.weights import load_weights_to_model, synthetic_state_dict
    from oracle.model import OracleBitNet

    cfg = BitNetConfig(hidden_size=2560, num_layers=2, num_attention_heads=20, num_key_value_heads=5,
                       intermediate_size=6912, vocab_size=1000, max_position_embeddings=4096)
    lazy = synthetic_state_dict(cfg, 11)
    sd = {k: lazy[k].numpy() for k in lazy}
    model = create_model(cfg, cuda)
    load_weights_to_model(model, sd)
    prompts = [np.random.default_rng(n).integers(0, cfg.vocab_size, size=n) for n in LENS]
    gen = Batch32Generator(model, batch_size=len(LENS), max_seq_len=max(LENS) + 64)
    gen.prefill(prompts)
    torch.cuda.synchronize()
    first = [(c.key_cache.clone(), c.value_cache.clone()) for c in gen.state.caches]
    oracle = OracleBitNet(cfg, sd, max_len=4096)
    for b, p in enumerate(prompts):
        cache = oracle.new_cache(1, len(p))[0]
        oracle.layer_prefill(0, oracle.embed[torch.from_numpy(p)], 1, len(p), cache)
        for name, mine, ref in (("K", first[0][0], cache[0]), ("V", first[0][1], cache[1])):
            got, want = mine[b, :, :len(p)].float().cpu(), ref[0, :, :len(p)]
            assert torch.equal(got, want), _where(f"oracle, sequence {b} {name}", got, want)
    for r in range(REPEATS):
        for c in gen.state.caches:
            c.key_cache.fill_(float("nan")), c.value_cache.fill_(float("nan"))
        gen.prefill(prompts)
        torch.cuda.synchronize()
        for i, (c, want) in enumerate(zip(gen.state.caches, first)):
            for b, n in enumerate(LENS):
                for name, mine, ref in (("K", c.key_cache, want[0]), ("V", c.value_cache, want[1])):
                    got = mine[b, :, :n]
                    assert torch.equal(got, ref[b, :, :n]), _where(f"repeat {r}, layer {i}, sequence {b} {name}", got,
                                                                   ref[b, :, :n])
