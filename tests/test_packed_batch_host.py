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


def test_a_step_is_captured_between_prefill_and_the_first_step(batch):
    with pytest.raises(RuntimeError, match="after prefill"):
        batch.capture()
    batch.lengths = [3, 5]
    with pytest.raises(RuntimeError, match="needs capture"):
        batch.step([1, 2])
    batch.steps = 2  # the recorded run would write over the first step's keys
    with pytest.raises(RuntimeError, match="before the first step"):
        batch.capture()


def test_continuations_need_an_alternative(mpc):
    pb = importlib.import_module(mpc.__name__ + ".packed_batch")
    cfg = pb.PackedBatchConfig(hidden=128, heads=2, kv_heads=1, ffn=160, vocab=300, slot=24, top=0)
    batch = pb.PackedBatch(NoDevice(), cfg, pb.make_weights(cfg))
    batch.lengths = [2]
    with pytest.raises(ValueError, match="top is 0"):
        batch.generate(np.zeros((2, 2), np.float32), 1)
