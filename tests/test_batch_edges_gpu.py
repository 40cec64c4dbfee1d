"""GPU: the operators for batches of packed sequences where a server takes them far from their usual sizes:
captured steps over slots much longer than the sequences in them, extreme logits and temperatures, streams that
change, tables whose sequences meet.  Against plain implementations in 64 bits; tolerances of the neighbouring
tests unless a test derives its own."""
import math

import numpy as np
import pytest
import torch

from test_batch_ops_gpu import ATTENTION_TOL, DT, attention64, quantise64, randn, rel, to_torch

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------- captured steps over long slots
@pytest.mark.parametrize("dim,kv", [(64, 1), (128, 8)])
@pytest.mark.parametrize("ages", [[10], [1000], [10, 1, 1000, 30]])
def test_captured_decode_of_young_sequences_in_long_slots(kernels, executor, mpc, ages, dim, kv):
    """A slot of 32768 rows of a 4-bit store holds a few keys when the step is captured and is nearly full at its
    end.  A split product afterwards, which counts its CTAs' arrivals on the same words, is right as well."""
    heads, slot, n = 4 * kv if kv == 1 else kv, 32768, len(ages)
    inv = mpc.KernelInvocation
    starts = [i * slot for i in range(n)]
    k, v = randn((slot * n, kv * dim), "f32", 201), randn((slot * n, kv * dim), "f32", 202)
    for name, t in (("ks", k), ("vs", v)):
        store = kernels.kv_store_q4(slot * n, kv, dim)
        kernels.kv_write(store, kernels.wrap_tensor(t), 0)  # (the steps write the same rows again)
        executor.adopt(name, store)
    executor.adopt("seqs", kernels.sequences([1] * n, ages, starts))
    offsets = [0, 1, 300, 5000, slot - max(ages)]
    q = randn((len(offsets), n, heads * dim), "f32", 203)
    for name, w in (("q", heads), ("kn", kv), ("vn", kv)):
        executor.write_zeroed_tensor(name, (n, w * dim))
    nodes = [inv("kv-write-packed", ["ks", "kn", "seqs"], "ks"), inv("kv-write-packed", ["vs", "vn", "seqs"], "vs"),
             inv("attention-packed", ["q", "ks", "vs", "seqs"], "out",
                 {"head_count": heads, "head_dimension": dim, "kv_head_count": kv, "causal": True})]
    for node in nodes:
        executor.run(node)
    executor.begin_step_capture(["key_count"])
    for node in nodes:
        executor.run(node)
    executor.end_step_capture()
    assert executor.step_max_offset() == offsets[-1]
    k64, v64 = quantise64(k), quantise64(v)
    out = np.empty((n, heads * dim), np.float32)
    for i, offset in enumerate(offsets):
        rows = [s + m - 1 + offset for s, m in zip(starts, ages)]
        executor.replay_step_io({"q": q[i].cpu().numpy(), "kn": k[rows].cpu().numpy(), "vn": v[rows].cpu().numpy()}, {"out": out}, offset=offset)
        want = attention64(q[i], k64, v64, heads, kv, [1] * n, [m + offset for m in ages], starts)
        assert rel(torch.from_numpy(out).cuda(), want) <= ATTENTION_TOL["f32"], offset
        if i == 0:  # what the recorded run left in row 0 of each sequence is overwritten by now
            whole = torch.from_numpy(executor.read_tensor("ks")).cuda().double()
            assert torch.equal(whole, k64)
    for rows, inner, columns in ((1, 40000, 36), (3, 9001, 132), (16, 20011, 64)):
        a, b = randn((rows, inner), "f32", 204), randn((inner, columns), "f32", 205)
        got = to_torch(kernels, kernels.matmul(kernels.wrap_tensor(a), kernels.wrap_tensor(b)))
        assert rel(got, a.double() @ b.double()) <= 1e-5
