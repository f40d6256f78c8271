"""A block's C structs hold the addresses of its tensors."""
import gc
import weakref

import mlx_rs_b200.synth as S
from mlx_rs_b200.block import SparseMoeBlock


def test_replaced_weights_of_a_moe_block_stay_alive():
    cfg = S.MoeConfig(256, 8, 2, 128, 64, S.SCORING_SOFTMAX_BIAS, True, True)
    blk = SparseMoeBlock(S.to_device(S.host_block(cfg, 3), "cpu"))
    w = blk.weights
    at = {name: getattr(w, name).w for name in ("router", "gate", "up", "down", "shared_gate", "shared_expert_gate")}
    refs = [weakref.ref(t) for t in at.values()] + [weakref.ref(w.expert_bias), weakref.ref(w.up.biases)]
    del at
    other = S.to_device(S.host_block(cfg, 4), "cpu")
    for name in ("router", "gate", "up", "down", "shared_gate", "shared_expert_gate", "expert_bias"):
        setattr(w, name, getattr(other, name))
    gc.collect()
    assert all(r() is not None for r in refs)
