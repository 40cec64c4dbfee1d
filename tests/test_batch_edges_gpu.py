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


# ---------------------------------------------------------------------------- log probabilities
def check_logprobs(kernels, x, tokens, top, temperature):
    """Against 64 bits, each value by itself.  A difference of logits over the temperature carries three roundings of
    f32 (2^-22 of its size, below 1e-6), the log-sum some 1e-6: 1e-5 + 1e-6 |value|.  The entropy and the top
    columns, columns included, apart from the chosen token.  Log probabilities are not positive, entropies not negative."""
    got = to_torch(kernels, kernels.token_logprobs(kernels.wrap_tensor(x), kernels.wrap_tensor(tokens), top=top, temperature=temperature)).double()
    z = x.double() / temperature
    logp = torch.log_softmax(z, 1)
    entropy = -torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(1)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    want = torch.cat([logp.gather(1, tokens.long()[:, None]), entropy[:, None], logp.gather(1, order)], 1)
    assert torch.equal(got[:, 2 + top:], order.double())
    a = got[:, :2 + top]
    assert torch.equal(torch.isnan(a), torch.isnan(want))
    low = want < -3e38  # beyond f32
    assert (a[low] < -3e38).all()
    fine = torch.isfinite(want) & ~low
    assert torch.equal(torch.isfinite(a) & ~low, fine)
    worst = ((a - want).abs() - 1e-5 - 1e-6 * want.abs())[fine].max()
    assert worst <= 0, worst
    assert (a[:, 0][fine[:, 0]] <= 0).all() and (a[:, 1][fine[:, 1]] >= 0).all()


@pytest.mark.parametrize("rows,vocab", [(6, 32000), (200, 32000), (6, 131072), (200, 1001)])
@pytest.mark.parametrize("case", ["mask 5000", "low 100", "even", "near", "at", "steep"])
def test_token_logprobs_at_the_low_end_of_f16(kernels, case, rows, vocab):
    """Logits down to the type's lowest value count for what they are, whatever the maximum and the temperature."""
    g = torch.Generator(device="cuda").manual_seed(211)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g).float()
    temperature = 1.0
    if case == "mask 5000":
        x = torch.full((rows, vocab), -65504.0, device="cuda")
        x[:, 7] = 0.0
        temperature = 5000.0
    elif case == "low 100":
        x = torch.randn((rows, vocab), device="cuda", generator=g) * 300 - 33500
        temperature = 100.0
    elif case == "even":
        x = torch.full((rows, vocab), -32800.0, device="cuda")
        x[:, 5] = -32752.0
    elif case == "near":
        x = torch.full((rows, vocab), -65504.0, device="cuda")
        x[:, vocab // 2] = -65472.0
        x[1::2, :3] = -math.inf
        temperature = 10.0
    elif case == "at":
        x = torch.full((rows, vocab), -32800.0, device="cuda")
        x[:, 9] = -32768.0
        temperature = 8.0
    else:
        x = torch.randn((rows, vocab), device="cuda", generator=g) * 4
        x[:, ::3] = -65504.0
        temperature = 300.0
    x = x.half()
    torch.cuda.synchronize()
    check_logprobs(kernels, x, tokens, 3, temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(5, 32000), (300, 5000), (3, 200)])
@pytest.mark.parametrize("most,temperature", [(30.1, 0.01), (5000.7, 0.1), (5000.7, 0.01), (-5000.7, 0.01), (30.1, 1e-6), (3.0, 1e-30),
                                              (-40000.0, 1.0), (3.0, 1e4), (1e9, 1.0), (-1e9, 0.5), (3e38, 1.0), (3e38, 1e30), (-3e38, 1e30)])
def test_token_logprobs_of_large_logits_and_far_temperatures(kernels, dtype, rows, vocab, most, temperature):
    """One column above the others by far, two close ones, and a spread about the maximum, where the quotient of
    logit and temperature is far from zero: the log-sum keeps its digits."""
    limit = float(torch.finfo(DT[dtype]).max)
    most = max(-limit, min(limit, most))
    x = randn((rows, vocab), "f32", 212)
    x[0] -= x[0].abs().max() + 1
    x[0, 77] = 0.0                      # (a probability of one at low temperatures)
    x[1] = -abs(x[1])
    x[1, [3, vocab - 2]] = 0.0          # two alike
    unit = min(max(temperature, 1e-30), 1e37)
    x = (most + x.double() * 2 * unit).clamp(-limit, limit).float().to(DT[dtype])
    tokens = torch.randint(0, vocab, (rows,), device="cuda").float()
    tokens[0], tokens[1] = 77, 3
    torch.cuda.synchronize()
    check_logprobs(kernels, x, tokens, 5, temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -3.3e15, -1e30, -1.7e38])
@pytest.mark.parametrize("rows", [4, 200])
def test_token_logprobs_beside_large_negative_masks(kernels, dtype, mask, rows):
    """Whole stretches of a row hold a mask's value, as large as callers choose them."""
    vocab = 40000
    x = randn((rows, vocab), dtype, 213, 3.0)
    x[:, : vocab - 500] = mask
    x[1::2] = x[1::2].flip(1)
    tokens = torch.randint(0, vocab, (rows,), device="cuda").float()
    tokens[0] = vocab - 3
    torch.cuda.synchronize()
    check_logprobs(kernels, x, tokens, 7, 1.0)
    x[:] = mask  # and nothing else
    torch.cuda.synchronize()
    check_logprobs(kernels, x, tokens, 7, 1.0)


def test_token_logprobs_by_the_value(kernels):
    """The cases of ordinary logits, each value held to its own size rather than to the largest of the tensor."""
    for i, (dtype, rows, vocab, top, temperature) in enumerate([("f32", 8, 32000, 5, 1.0), ("bf16", 300, 999, 64, 1.0), ("f16", 5, 50001, 20, 1.3),
                                                                ("f16", 160, 1024, 1, 1.0), ("f32", 3, 5, 5, 0.7), ("bf16", 2, 131073, 32, 1.0)]):
        x = randn((rows, vocab), dtype, 214 + i, 3.0)
        x[::3, : vocab // 2] = -math.inf
        x[1::3, ::2] = torch.finfo(DT[dtype]).min
        tokens = torch.randint(0, vocab, (rows,), device="cuda").float()
        torch.cuda.synchronize()
        check_logprobs(kernels, x, tokens, top, temperature)


def test_token_logprobs_refuses_temperatures_without_a_reciprocal(kernels, mpc):
    x = kernels.zeros((2, 8))
    for t in (1e-39, 1e-45):
        with pytest.raises(mpc.CudaError) as e:
            kernels.token_logprobs(x, temperature=t)
        assert e.value.code == "ShapeUnsupported"


# ---------------------------------------------------------------------------- streams
def test_stream_changed_while_work_is_under_way(kernels, mpc, executor):
    """Calls in turn on two streams, each with work of its own in front: they share workspaces (the split keys of f32
    prompts, parts of keys, arrival counters), and do not overlap."""
    heads, kv, dim = 8, 2, 128
    busy = randn((2048, 2048), "f32", 221)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    prompts, many = [700, 300, 41], [20000]
    calls = []
    for i in range(8):
        n, m = (prompts, prompts) if i % 4 < 2 else ([1], many)
        q = randn((sum(n), heads * dim), "f32" if i % 4 < 2 else "bf16", 222 + 3 * i)
        dtype = "f32" if i % 4 < 2 else "bf16"
        k, v = randn((sum(m), kv * dim), dtype, 223 + 3 * i), randn((sum(m), kv * dim), dtype, 224 + 3 * i)
        calls.append((q, k, v, kernels.sequences(n, m), torch.empty_like(q), attention64(q, k, v, heads, kv, n, m), dtype))
    torch.cuda.synchronize()
    try:
        for i, (q, k, v, seqs, out, _, _) in enumerate(calls):
            side = streams[i % 2]
            with torch.cuda.stream(side):
                for _ in range(3 * (i % 2)):
                    busy @ busy
            kernels.set_stream(side.cuda_stream)
            kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim, kv_head_count=kv, out=kernels.wrap_tensor(out))
        executor.write_zeroed_tensor("x", (4, 64))
        executor.begin_step_capture()
        with pytest.raises(mpc.CudaError) as e:
            kernels.set_stream(None)
        assert e.value.code == "CaptureUnsupported"
        executor.abort_step_capture()
    finally:
        kernels.set_stream(None)
    torch.cuda.synchronize()
    for *_, out, want, dtype in calls:
        assert rel(out, want) <= ATTENTION_TOL[dtype]


@pytest.mark.parametrize("side", [False, True])
def test_wrapped_tensors_that_torch_is_still_filling(kernels, mpc, side):
    """torch's stream and the device's own are apart: a call waits for the work that was under way on torch's
    current stream when the tensor was wrapped."""
    busy, x = randn((4096, 4096), "f32", 231), randn((300, 512), "f32", 232)
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(20):
            busy @ busy
        late.copy_(x)
        buf = kernels.wrap_tensor(late)
    got = kernels.download(kernels.add(buf, buf))
    assert np.array_equal(got, 2 * x.cpu().numpy())
    torch.cuda.synchronize()
    with pytest.raises(mpc.CudaError):
        kernels.wrap_tensor(x.cpu())
    kernels.set_stream(1)  # torch's default stream by its other name
    try:
        with torch.cuda.stream(torch.cuda.default_stream()):
            y = x + 1
            got = kernels.download(kernels.add(kernels.wrap_tensor(y), kernels.wrap_tensor(y)))
        assert np.array_equal(got, (2 * (x + 1)).cpu().numpy())
    finally:
        kernels.set_stream(None)


# ---------------------------------------------------------------------------- tables whose sequences meet
def test_sequences_that_would_write_the_same_rows_are_refused(kernels, mpc):
    """Two sequences may read the same rows; rows written by both would be of neither."""
    rows = randn((4, 64), "f32", 241)
    buf = kernels.wrap_tensor(rows)
    for store in (kernels.kv_store_q4(100, 1, 64), kernels.zeros((100, 64))):
        for queries, keys, starts in (([2, 2], [10, 10], [0, 0]), ([2, 2], [10, 11], [0, 0]), ([3, 1], [50, 8], [0, 40]), ([1, 3], [8, 9], [41, 40])):
            with pytest.raises(mpc.CudaError) as e:
                kernels.kv_write_packed(store, buf, kernels.sequences(queries, keys, starts))
            assert e.value.code == "ShapeUnsupported"
        for queries, keys, starts in (([2, 2], [10, 12], [0, 0]), ([4, 0], [10, 10], [0, 0]), ([1, 3], [8, 8], [43, 40]), ([0, 4, 0], [0, 4, 0], [0, 0, 0])):
            kernels.kv_write_packed(store, buf, kernels.sequences(queries, keys, starts))
    # attention over shared rows stays as it was
    q, k, v = randn((4, 64), "f32", 242), randn((20, 64), "f32", 243), randn((20, 64), "f32", 244)
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), kernels.sequences([2, 2], [20, 20], [0, 0]), 1, 64))
    assert rel(got, attention64(q, k, v, 1, 1, [2, 2], [20, 20], [0, 0])) <= ATTENTION_TOL["f32"]


@pytest.mark.parametrize("queries,keys,starts,write,read", [
    ([1, 1], [10, 10], [0, 40], 30, 30),           # up to the second one's first row
    ([1, 1], [10, 12], [0, 0], 0, 88),             # the first one's next row is the second one's
    ([1, 0], [10, 50], [0, 5], 0, 45),             # ... also where that one does not write
    ([1, 0], [50, 10], [0, 0], 50, 50),            # a sequence that only reads a part of the rows
    ([1, 0, 1], [10, 0, 20], [0, 10, 60], 20, 20),  # an empty place in the batch
    ([0, 1], [10, 10], [0, 10], 80, 80),           # a finished sequence in front of the one that grows
])
def test_how_far_a_captured_step_may_advance(kernels, executor, mpc, queries, keys, starts, write, read):
    inv = mpc.KernelInvocation
    n = sum(queries)
    executor.adopt("store", kernels.kv_store_q4(100, 1, 64))
    executor.adopt("seqs", kernels.sequences(queries, keys, starts))
    executor.write_tensor("x", np.ones((n, 64), np.float32))
    for node, most in ((inv("kv-write-packed", ["store", "x", "seqs"], "store"), write),
                       (inv("attention-packed", ["x", "store", "store", "seqs"], "out", {"head_count": 1, "head_dimension": 64, "causal": True}), read)):
        executor.run(node)
        executor.begin_step_capture(["key_count"])
        executor.run(node)
        executor.end_step_capture()
        assert executor.step_max_offset() == min(most, 100 - max(s + k for s, k in zip(starts, keys))), node


def test_a_captured_read_back_follows_its_sequences(kernels, executor, mpc):
    """kv-read-packed reads what kv-write-packed has just written, at every offset of a step."""
    inv = mpc.KernelInvocation
    ages, starts, total = [3, 60, 1], [0, 100, 200], 300
    t = randn((total, 128), "f32", 245)
    store = kernels.kv_store_q4(total, 2, 64)
    kernels.kv_write(store, kernels.wrap_tensor(t), 0)
    executor.adopt("store", store)
    executor.adopt("seqs", kernels.sequences([1, 2, 1], ages, starts))
    executor.write_zeroed_tensor("x", (4, 128))
    nodes = [inv("kv-write-packed", ["store", "x", "seqs"], "store"), inv("kv-read-packed", ["store", "seqs"], "back")]
    for node in nodes:
        executor.run(node)
    executor.begin_step_capture(["key_count"])
    for node in nodes:
        executor.run(node)
    executor.end_step_capture()
    assert executor.step_max_offset() == 40
    x, back = np.empty((4, 128), np.float32), np.empty((4, 128), np.float32)
    for offset in (0, 1, 7, 40):
        x[:] = randn((4, 128), "f32", 246 + offset).cpu().numpy()
        executor.replay_step_io({"x": x}, {"back": back}, offset=offset)
        want = quantise64(torch.from_numpy(x).cuda())
        assert torch.equal(torch.from_numpy(back).cuda().double(), want), offset
        whole = torch.from_numpy(executor.read_tensor("store")).cuda().double()
        assert torch.equal(whole[[s + m - n + i + offset for s, m, n in zip(starts, ages, [1, 2, 1]) for i in range(n)]], want)


# ---------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (4, 2, 64), (3, 3, 80), (2, 1, 200), (2, 2, 300)])
@pytest.mark.parametrize("queries,keys", [([1], [45]), ([1, 1], [3, 2001]), ([2], [1003]), ([5, 40], [5, 77]), ([1], [4999]), ([130], [130]), ([128], [128]), ([64], [256])])
def test_infinite_values_that_a_query_sees(kernels, dtype, heads, kv, dim, queries, keys):
    """An infinity in the last value row of a sequence is infinite for those who see it, and nothing to the others."""
    q = randn((sum(queries), heads * dim), dtype, 251)
    k, v = randn((sum(keys), kv * dim), dtype, 252), randn((sum(keys), kv * dim), dtype, 253)
    v[-1, :2] = 0
    finite = v.clone()
    v[-1, 0], v[-1, 1] = math.inf, -math.inf
    torch.cuda.synchronize()
    seqs = kernels.sequences(queries, keys)
    for causal, window in ((True, None), (True, 333), (False, None)):
        got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim, kv_head_count=kv,
                                                         causal=causal, window_size=window)).double()
        want = attention64(q, k, finite, heads, kv, queries, keys, causal=causal, window=window)
        first = sum(queries) - (1 if causal else queries[-1])
        for h in range(heads // kv):
            assert (got[first:, h * dim] == math.inf).all() and (got[first:, h * dim + 1] == -math.inf).all(), (causal, window)
            got[first:, h * dim:h * dim + 2] = want[first:, h * dim:h * dim + 2]
        assert torch.isfinite(got).all()
        assert rel(got, want) <= ATTENTION_TOL[dtype], (causal, window)


def test_more_shared_keys_than_memory_holds_copies_of(kernels):
    """3000 sequences of three queries over the same 70000 rows: the copies that f32 prompts make of their keys would
    take 215 GB."""
    n, m, dim = 3000, 70000, 128
    q, k, v = randn((3 * n, dim), "f32", 271), randn((m, dim), "f32", 272), randn((m, dim), "f32", 273)
    seqs = kernels.sequences([3] * n, [m] * n, [0] * n)
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, 1, dim))
    some = [0, 1, 1500, n - 1]
    rows = torch.tensor([3 * i + j for i in some for j in range(3)], device="cuda")
    assert rel(got[rows], attention64(q[rows], k, v, 1, 1, [3] * 4, [m] * 4, [0] * 4)) <= ATTENTION_TOL["f32"]
    assert torch.isfinite(got).all()
    prompt = kernels.sequences([100, 30])  # ordinary calls go on
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t[:130]) for t in (q, k, v)), prompt, 1, dim))
    assert rel(got, attention64(q[:130], k, v, 1, 1, [100, 30], [100, 30])) <= ATTENTION_TOL["f32"]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,queries,keys,window", [
    (40, 40, 64, [300], [20000], None),             # a CTA has all keys of its rows
    (24, 8, 128, [600, 1, 400], [17000, 9, 18500], None),
    (40, 40, 64, [700], [24000], 18000),
    (8, 8, 128, [8], [70000], None),                # the keys are split, and a part is still long
    (32, 8, 128, [4, 2], [50000, 300], 45000),
])
def test_sums_over_many_keys(kernels, dtype, heads, kv, dim, queries, keys, window):
    """Tens of thousands of keys, values that do not cancel (sums on the tensor cores lose a little of themselves with
    every addition), later keys with ever higher scores (what has been summed is scaled down)."""
    q = randn((sum(queries), heads * dim), dtype, 291)
    k, v = randn((sum(keys), kv * dim), dtype, 292), randn((sum(keys), kv * dim), "f32", 293)
    v = (v + 1).to(DT[dtype])
    some = torch.cat([torch.arange(b - n, b, max(1, n // 12), device="cuda") for n, b in zip(queries, np.cumsum(queries).tolist())])
    for rising in (False, True):
        if rising:
            k = (k.float() * torch.linspace(0.2, 2.5, sum(keys), device="cuda")[:, None]).to(DT[dtype])
        torch.cuda.synchronize()
        got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), kernels.sequences(queries, keys), heads, dim,
                                                         kv_head_count=kv, window_size=window))
        assert torch.isfinite(got).all()
        at_q = at_k = 0
        for n, m in zip(queries, keys):  # a row at a time: it is the last of its own keys
            rows = [int(r) for r in some if at_q <= r < at_q + n]
            for r in rows:
                seen = m - n + (r - at_q) + 1
                want = attention64(q[r:r + 1], k[at_k:at_k + seen], v[at_k:at_k + seen], heads, kv, [1], [seen], window=window)
                assert rel(got[r], want[0]) <= ATTENTION_TOL[dtype], (rising, r)
            at_q, at_k = at_q + n, at_k + m


def test_sums_over_many_keys_in_a_captured_step(kernels, executor, mpc):
    """A step captured over a few keys, replayed where they are many."""
    inv = mpc.KernelInvocation
    heads, dim, slot, n = 8, 64, 40000, 4
    q, k, v = randn((n, heads * dim), "f32", 295), randn((slot, heads * dim), "f32", 296), randn((slot, heads * dim), "f32", 297) + 1
    torch.cuda.synchronize()
    for name, t in (("q", q), ("k", k), ("v", v)):
        executor.write_tensor(name, t.cpu().numpy())
    executor.adopt("seqs", kernels.sequences([n], [10], [0]))
    node = inv("attention-packed", ["q", "k", "v", "seqs"], "out", {"head_count": heads, "head_dimension": dim, "causal": True})
    executor.run(node)
    executor.begin_step_capture(["key_count"])
    executor.run(node)
    executor.end_step_capture()
    for offset in (0, 2040, 2300, 39990):
        executor.replay_step(offset=offset)
        got = torch.from_numpy(executor.read_tensor("out")).cuda()
        assert rel(got, attention64(q, k, v, heads, heads, [n], [10 + offset])) <= ATTENTION_TOL["f32"], offset


_F32_CHILD = r"""
import importlib, json, sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import torch
from test_batch_ops_gpu import attention64, quantise64, randn, rel, to_torch
ks = importlib.import_module("magnetar-provider-cuda_b200").CudaKernels(0)
out = []
for heads, kv, dim, queries, keys in ((8, 2, 128, [300, 5, 41], [300, 700, 41]), (4, 4, 64, [130, 1], [130, 3000]), (3, 1, 64, [3, 4, 0], [999, 64, 7]),
                                      (2, 1, 80, [50], [50])):
    q, k, v = randn((sum(queries), heads * dim), "f32", 281), randn((sum(keys), kv * dim), "f32", 282), randn((sum(keys), kv * dim), "f32", 283)
    seqs = ks.sequences(queries, keys)
    for window in (None, 60):
        got = to_torch(ks, ks.attention_packed(*(ks.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim, kv_head_count=kv, window_size=window))
        out.append(rel(got, attention64(q, k, v, heads, kv, queries, keys, window=window)))
        if dim % 64 == 0:
            stores = [ks.kv_write(ks.kv_store_q4(sum(keys), kv, dim), ks.wrap_tensor(t), 0) for t in (k, v)]
            got = to_torch(ks, ks.attention_packed(ks.wrap_tensor(q), *stores, seqs, heads, dim, kv_head_count=kv, window_size=window))
            out.append(rel(got, attention64(q, quantise64(k), quantise64(v), heads, kv, queries, keys, window=window)))
print(json.dumps(out))
"""


def test_f32_throughout_by_its_switch():
    """Scores are sums of up to 128 products in four chains of f32, some 2^-21 off; weights, sums and means round by 2^-23:
    2e-6 of the output bounds them, which two-term operands (2e-6 to 6e-6) do not reach."""
    import json
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = lambda env: subprocess.run([sys.executable, "-c", _F32_CHILD, root], env=env, capture_output=True, text=True, timeout=300)
    for value, bound in (("1", 2e-6), ("0", ATTENTION_TOL["f32"])):
        res = run(dict(os.environ, MAGNETAR_CUDA_PACKED_F32=value))
        assert res.returncode == 0, res.stderr[-2000:]
        errors = json.loads(res.stdout.strip().splitlines()[-1])
        assert len(errors) == 14 and max(errors) <= bound, errors


def test_a_refused_allocation_leaves_the_memory_free(kernels, mpc):
    """More than the GPU has, and all that it has (of which the process itself has a part): refused, and nothing is kept of it."""
    torch.cuda.empty_cache()
    kernels.synchronize()
    before = kernels.info()
    for size in (before["total_bytes"] + 2 ** 32, before["total_bytes"] - 2 ** 20):
        with pytest.raises(mpc.CudaError) as e:
            kernels.empty((size // 4,))
        assert e.value.code == "OutOfDeviceMemory"
        assert kernels.info()["free_bytes"] >= before["free_bytes"] - 2 ** 28
    assert not kernels.download(kernels.zeros((1000,))).any()


# ---------------------------------------------------------------------------- outputs over inputs
def test_outputs_that_share_memory_with_inputs_are_refused(kernels, mpc):
    """Blocks would read what others have written; rope in place is the one form that is in order."""
    q, k = randn((8, 64), "f32", 261), randn((8, 64), "f32", 262)
    whole = randn((20, 64), "f32", 263)
    x, y = kernels.wrap_tensor(q), kernels.wrap_tensor(k)
    seqs = kernels.sequences([8])
    part = lambda first, rows: kernels.wrap_tensor(whole[first:first + rows])
    logits, two = randn((6, 4), "f32", 264), randn((4, 2), "f32", 265)
    lb, pb = kernels.wrap_tensor(logits), kernels.wrap_tensor(two)
    calls = [lambda: kernels.attention_packed(x, y, y, seqs, 1, 64, out=x), lambda: kernels.attention_packed(x, y, y, seqs, 1, 64, out=y),
             lambda: kernels.attention_packed(x, part(0, 8), part(8, 8), seqs, 1, 64, out=part(12, 8)),
             lambda: kernels.kv_write_packed(part(0, 20), part(3, 8), seqs),
             lambda: kernels.token_logprobs(lb, top=1, out=lb),
             lambda: kernels.rope_axes(pb, pb, [1, 0], out=pb),
             lambda: kernels.rope_axes(part(0, 8), kernels.zeros((8, 1)), [32], out=part(1, 8))]
    before = [t.clone() for t in (q, k, whole, logits, two)]
    for i, call in enumerate(calls):
        with pytest.raises(mpc.CudaError) as e:
            call()
        assert e.value.code == "InvalidArgument", i
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k, whole, logits, two)))
    # neighbours are apart
    kernels.attention_packed(part(0, 4), part(4, 8), part(4, 8), kernels.sequences([4], [8]), 1, 64, out=part(12, 4))
    kernels.kv_write_packed(part(0, 8), part(8, 8), seqs)
    kernels.rope_axes(part(0, 8), kernels.zeros((8, 1)), [32], out=part(0, 8))
    kernels.synchronize()
