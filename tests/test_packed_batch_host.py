"""CPU: what PackedBatch refuses before it reaches the device."""
import importlib

import numpy as np
import pytest


class NoDevice:
    """Takes the weights; anything else would be a call to the device."""

    def write_weight_tensor(self, name, value):
        pass


@pytest.fixture()
def batch(mpc):
    pb = importlib.import_module(mpc.__name__ + ".packed_batch")
    cfg = pb.PackedBatchConfig(hidden=128, heads=2, kv_heads=1, ffn=160, vocab=300, slot=24)
    return pb.PackedBatch(NoDevice(), cfg, pb.make_weights(cfg))


@pytest.mark.parametrize("lengths", [[], [0], [3, 0, 2]])
def test_prompts_without_tokens_are_refused(batch, lengths):
    with pytest.raises(ValueError, match="at least one token"):
        batch.prefill([np.arange(n) for n in lengths])
    assert batch.lengths == []
