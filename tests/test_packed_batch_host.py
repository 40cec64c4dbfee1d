"""CPU: what PackedBatch, and the tables of packed sequences, refuse before they reach the device."""
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


def test_counts_of_a_table(mpc):
    counts = importlib.import_module(mpc.__name__ + ".kernels")._counts
    assert list(counts(range(3))) == [0, 1, 2] and list(counts([])) == [] and counts(None) is None
    assert list(counts(np.array([4, 5]), counts(iter([1, 2])))) == [4, 5]  # as many as an iterator gave
    for bad in ([-1], [2 ** 64], [2 ** 64 + 5]):
        with pytest.raises(ValueError, match="64 bits"):
            counts(bad)
    with pytest.raises(ValueError, match="for 2 sequences"):
        counts([1], counts([1, 1]))
