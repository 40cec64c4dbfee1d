"""GPU: a batch of prompts and its next tokens through the packed operators together, against the same layer
in 64 bits.

The keys and values that the reference attends to in a step are those of the device's own stores (a rounding
error of 1e-6 in a key may move it to the next of its 16 values, which is checked apart: the stores hold exactly
the quantised rows of the device).  Tolerance of a log probability: the chain's products and norms are f32 with
matmuls as three tf32 products and attention within 2e-5 of its own size; logits here are of order one with some
512 and 1376 terms summed, so errors of 1e-4 bound them with room: 1e-4 absolute."""
import math

import numpy as np
import pytest
import torch

from test_batch_ops_gpu import attention64, logprobs64, quantise64, rope64

pytestmark = pytest.mark.gpu
TOL = 1e-4


def layer64(w, cfg, ids, positions, attend):
    """The layer's scores in f64; ``attend(q, k, v)`` is the attention."""
    t = {n: torch.from_numpy(v).cuda().double() for n, v in w.items()}
    ids, positions = torch.from_numpy(ids).cuda().long(), torch.from_numpy(positions).cuda()

    def norm(x, g):
        return x / (x.square().mean(-1, keepdim=True) + cfg.eps).sqrt() * g

    def rope(x, heads):
        return rope64(x, positions, list(cfg.sections), heads, cfg.head_dim, "half_split", "cyclic", "shared", False)

    x = t["table"][ids]
    h = norm(x, t["attn_norm"])
    q, k, v = rope(h @ t["wq"], cfg.heads), rope(h @ t["wk"], cfg.kv_heads), h @ t["wv"]
    x = x + attend(q, k, v) @ t["wo"]
    h = norm(x, t["mlp_norm"])
    x = x + (torch.nn.functional.silu(h @ t["wg"]) * (h @ t["wu"])) @ t["wd"]
    return norm(x, t["final_norm"]) @ t["head"]


@pytest.mark.parametrize("lengths", [[37, 1, 128, 70], [5]])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_prompts_and_steps(mpc, executor, kernels, lengths, head_dim):
    import importlib
    pb = importlib.import_module(mpc.__name__ + ".packed_batch")
    cfg = pb.PackedBatchConfig(hidden=256, heads=4, kv_heads=2, head_dim=head_dim, ffn=352, vocab=1000, slot=200,
                               sections=(head_dim // 2 - 20, 10, 10), top=3)
    rng = np.random.default_rng(5)
    w = pb.make_weights(cfg, 1)
    prompts = [rng.integers(0, cfg.vocab, n) for n in lengths]
    # an image of 6 x 6 patches inside the first prompt where it fits: one instant, rows and columns apart
    at = [np.repeat(np.arange(n, dtype=np.float32)[:, None], 3, 1) for n in lengths]
    if lengths[0] >= 37:
        at[0][:36] = np.stack([np.zeros(36), np.arange(36) // 6, np.arange(36) % 6], 1)
    at = np.concatenate(at)
    batch = pb.PackedBatch(executor, cfg, w)
    scores = batch.prefill(prompts, at)

    ids = np.concatenate(prompts)
    logits = layer64(w, cfg, ids, at, lambda q, k, v: attention64(q, k, v, cfg.heads, cfg.kv_heads, lengths, lengths))
    targets = np.concatenate([np.append(p[1:], -1) for p in prompts])
    want = logprobs64(logits, torch.from_numpy(targets).cuda().float(), cfg.top, 1.0).cpu().numpy()
    last = np.cumsum(lengths) - 1
    assert np.isnan(scores[last, 0]).all()
    assert np.nanmax(np.abs(scores[:, :2 + cfg.top] - want[:, :2 + cfg.top])) <= TOL

    def stored(name, rows):
        whole = torch.from_numpy(executor.read_tensor(name)).cuda().double()
        return torch.cat([whole[i * cfg.slot:i * cfg.slot + n] for i, n in enumerate(rows)])

    for name, source in (("key_store", "p.kr"), ("value_store", "p.v")):
        assert torch.equal(stored(name, lengths), quantise64(torch.from_numpy(executor.read_tensor(source)).cuda()))

    batch.capture()
    starts = [i * cfg.slot for i in range(len(lengths))]
    tokens = scores[last, 2 + cfg.top].astype(int)
    for i in range(4):
        got = batch.step(tokens).copy()
        n = [m + i + 1 for m in lengths]
        k, v = (torch.from_numpy(executor.read_tensor(s)).cuda() for s in ("key_store", "value_store"))
        where = np.repeat(np.array([m - 1 for m in n], np.float32)[:, None], 3, 1)
        logits = layer64(w, cfg, tokens, where,
                         lambda q, _k, _v: attention64(q, k, v, cfg.heads, cfg.kv_heads, [1] * len(n), n, starts))
        want = logprobs64(logits, torch.full((len(n),), -1.0, device="cuda"), cfg.top, 1.0).cpu().numpy()
        assert np.abs(got[:, 1:2 + cfg.top] - want[:, 1:2 + cfg.top]).max() <= TOL, i
        for name, source in (("key_store", "s.kr"), ("value_store", "s.v")):  # the step's rows are in the stores
            rows = torch.from_numpy(executor.read_tensor(name)).cuda().double()[[s + m - 1 for s, m in zip(starts, n)]]
            assert torch.equal(rows, quantise64(torch.from_numpy(executor.read_tensor(source)).cuda()))
        tokens = got[:, 2 + cfg.top].astype(int)
    assert batch.steps == 4


def test_generate_and_a_full_slot(mpc, executor):
    import importlib
    pb = importlib.import_module(mpc.__name__ + ".packed_batch")
    cfg = pb.PackedBatchConfig(hidden=128, heads=2, kv_heads=1, ffn=160, vocab=300, slot=24)
    batch = pb.PackedBatch(executor, cfg, pb.make_weights(cfg))
    scores = batch.prefill([np.arange(20), np.arange(7)])
    batch.capture()
    tokens = batch.generate(scores, 4)
    assert [len(t) for t in tokens] == [4, 4] and all(0 <= i < 300 for t in tokens for i in t)
    with pytest.raises(mpc.CudaError) as e:
        batch.step([1, 2])
    assert e.value.code == "CaptureUnsupported" and batch.steps == 4
    with pytest.raises(ValueError):
        batch.prefill([np.arange(24)])
