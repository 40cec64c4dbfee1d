"""The serving operators for batches of packed sequences, as cases that can be measured.

Each case is one pass of one operator on inputs made from a seed: attention over packed prompts, attention
over a key/value store held in 4 bits, writing rows into such a store, rotary positions with several axes, and
log probabilities of given tokens with entropy and top alternatives.  ``run`` computes it either in a plain
form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own`` set, by the calls a user
of this package makes.  ``exact`` gives the results in 64 bits.
"""
import importlib
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_Q4_BLOCK = 64  # values of a row that share one scale in a 4-bit store
_kernels = None


def _framework():
    """The package's kernels of cuda:0, enqueuing on torch's current stream (1 names the legacy default stream,
    whose handle in torch is 0)."""
    global _kernels
    if _kernels is None:
        _kernels = importlib.import_module("magnetar-provider-cuda_b200").CudaKernels(0)
    _kernels.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return _kernels


def _counts(text):
    return [int(x) for x in text.split(",")]


# ---- the cases ------------------------------------------------------------------------------------------------
def listed():
    return [
        # A few short prompts of the decoder layer's own shape (8 heads of 64, up to 128 tokens) in one call.
        {"name": "prompts_small_f32", "op": "attention_packed", "dtype": "f32", "heads": 8, "kv_heads": 8, "dim": 64,
         "queries": "128,77,1,33", "keys": "128,77,1,33", "window": 0, "causal": True},
        # The prefill batch (4 sequences of 2048, 32 heads of 128) as one packed call.
        {"name": "prompts_prefill_f32", "op": "attention_packed", "dtype": "f32", "heads": 32, "kv_heads": 32, "dim": 128,
         "queries": "2048,2048,2048,2048", "keys": "2048,2048,2048,2048", "window": 0, "causal": True},
        # A serving batch of prompts of very different lengths, grouped heads, half precision.
        {"name": "prompts_ragged_bf16", "op": "attention_packed", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "queries": "8192,1,1500,613,4096,37,2049,255,1024,5", "keys": "8192,1,1500,613,4096,37,2049,255,1024,5",
         "window": 0, "causal": True},
        # One token of each of four young sequences: latency counts.
        {"name": "decode4_small_f32", "op": "attention_q4", "dtype": "f32", "heads": 8, "kv_heads": 8, "dim": 64,
         "queries": "1,1,1,1", "keys": "129,17,500,64", "window": 0, "causal": True},
        # One token of each of 32 sequences of very different ages, grouped heads.
        {"name": "decode4_batch_f32", "op": "attention_q4", "dtype": "f32", "heads": 32, "kv_heads": 8, "dim": 128,
         "queries": ",".join(["1"] * 32), "keys": ",".join(str(v) for v in _ages(32, 100, 16000)), "window": 0, "causal": True},
        # A long-context batch: the cache is far larger than the L2.
        {"name": "decode4_long_bf16", "op": "attention_q4", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "queries": ",".join(["1"] * 16), "keys": ",".join(["32768"] * 15 + ["131071"]), "window": 0, "causal": True},
        # The new keys of one step of a batch, one row for each sequence.
        {"name": "write4_step_f32", "op": "write_q4", "dtype": "f32", "heads": 8, "kv_heads": 8, "dim": 128,
         "queries": ",".join(["1"] * 32), "keys": ",".join(str(v) for v in _ages(32, 100, 4000)), "window": 0, "causal": True},
        # The keys of whole prompts.
        {"name": "write4_prompt_bf16", "op": "write_q4", "dtype": "bf16", "heads": 8, "kv_heads": 8, "dim": 128,
         "queries": "8192,1,1500,613,4096,37,2049,255,1024,5", "keys": "8192,1,1500,613,4096,37,2049,255,1024,5",
         "window": 0, "causal": True},
        # Patches of one small image: two axes, each with frequencies of its own.
        {"name": "rope_image_f32", "op": "rope_axes", "dtype": "f32", "rows": 729, "heads": 16, "width": 64, "dimension": 64,
         "sections": "16,16", "order": "blocks", "ladder": "per_axis", "pairing": "half_split", "inverse": False},
        # Queries of text mixed with video: time, height and width dealt out in turn over one set of frequencies.
        {"name": "rope_video_bf16", "op": "rope_axes", "dtype": "bf16", "rows": 32768, "heads": 32, "width": 128, "dimension": 128,
         "sections": "24,20,20", "order": "cyclic", "ladder": "shared", "pairing": "half_split", "inverse": False},
        # The tokens of one step of a small batch over the decoder layer's vocabulary.
        {"name": "logprobs_step_f32", "op": "logprobs", "dtype": "f32", "rows": 8, "vocab": 32000, "top": 5, "temperature": 1.0},
        # Scoring whole prompts.
        {"name": "logprobs_prompt_bf16", "op": "logprobs", "dtype": "bf16", "rows": 8192, "vocab": 32000, "top": 20, "temperature": 1.0},
    ]


def _ages(count, low, high):
    """`count` lengths spread over the logarithm of [low, high], in a mixed order."""
    return [int(low * (high / low) ** (((i * 7) % count) / max(1, count - 1))) for i in range(count)]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention_packed", "attention_packed", "attention_q4", "attention_q4", "write_q4", "rope_axes", "logprobs"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "rope_axes":
        width = rng.choice([32, 64, 80, 96, 128])
        axes = rng.choice([1, 2, 3])
        pairs = width // 2 if rng.random() < 0.7 else width // 4
        per = pairs // axes
        sections = [pairs - per * (axes - 1)] + [per] * (axes - 1)
        heads = rng.choice([1, 4, 8, 16, 32])
        return {"op": op, "dtype": dtype, "rows": _spread(rng, 1, 32768), "heads": heads, "width": width, "dimension": 2 * pairs,
                "sections": ",".join(str(s) for s in sections), "order": rng.choice(["blocks", "cyclic"]),
                "ladder": rng.choice(["shared", "per_axis"]), "pairing": rng.choice(["half_split", "interleaved"]),
                "inverse": rng.random() < 0.3}
    if op == "logprobs":
        vocab = _spread(rng, 1000, 131072)
        return {"op": op, "dtype": dtype, "rows": _spread(rng, 1, max(1, 131072000 // vocab)), "vocab": vocab,
                "top": rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([1.0, 0.7])}
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    if op == "attention_packed":
        n = _spread(rng, 1, 24)
        longest = _spread(rng, 1, 4096)
        queries = [_spread(rng, 1, longest) for _ in range(n)]
        keys = [q + (_spread(rng, 1, 1024) if rng.random() < 0.2 else 0) for q in queries]
        while sum(q * k for q, k in zip(queries, keys)) > 24_000_000:
            queries, keys = queries[1:], keys[1:]
        causal = rng.random() < 0.8
        window = _spread(rng, 16, 2048) if causal and rng.random() < 0.3 else 0
    else:
        n = _spread(rng, 1, 48)
        longest = _spread(rng, 16, 32768)
        most = 4 if op == "attention_q4" and rng.random() < 0.3 else 1
        if op == "write_q4" and rng.random() < 0.5:
            most = 1024
        queries = [_spread(rng, 1, most) for _ in range(n)]
        keys = [q + _spread(rng, 1, longest) for q in queries]
        while sum(keys) > 400_000:
            queries, keys = queries[1:], keys[1:]
        causal, window = True, 0
    return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "queries": ",".join(map(str, queries)),
            "keys": ",".join(map(str, keys)), "window": window, "causal": causal}


# ---- inputs ---------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype="f32", scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(_DTYPES[dtype])


def _inputs(case, seed):
    """The tensors a case's operator reads, from the seed alone."""
    g = _generator(seed)
    op = case["op"]
    if op == "rope_axes":
        axes = len(_counts(case["sections"]))
        x = _normal(g, (case["rows"], case["heads"] * case["width"]), case["dtype"])
        # time runs slowly, rows and columns of a frame faster
        pos = torch.floor(torch.rand((case["rows"], axes), generator=g, device="cuda") * 512.0)
        return {"x": x, "positions": pos}
    if op == "logprobs":
        logits = _normal(g, (case["rows"], case["vocab"]), case["dtype"], 2.0)
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda").to(torch.float32)
        # a part of the vocabulary is excluded in some rows, as by a grammar
        logits[::5, : case["vocab"] // 3] = -math.inf
        return {"logits": logits, "tokens": tokens}
    queries, keys = _counts(case["queries"]), _counts(case["keys"])
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "attention_packed":
        return {"q": _normal(g, (sum(queries), heads * dim), case["dtype"]), "k": _normal(g, (sum(keys), kv * dim), case["dtype"]),
                "v": _normal(g, (sum(keys), kv * dim), case["dtype"])}
    if op == "attention_q4":
        # some channels of the keys are large, as those of real keys are
        gain = 1.0 + 3.0 * (torch.rand((kv * dim,), generator=g, device="cuda") > 0.95).float()
        return {"q": _normal(g, (sum(queries), heads * dim), case["dtype"]), "k": _normal(g, (sum(keys), kv * dim)) * gain,
                "v": _normal(g, (sum(keys), kv * dim))}
    return {"rows": _normal(g, (sum(queries), kv * dim), case["dtype"])}


def _starts(counts):
    at, out = 0, []
    for c in counts:
        out.append(at)
        at += c
    return out


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    op = case["op"]
    if op in ("attention_packed", "attention_q4", "write_q4"):
        s["queries"], s["keys"] = _counts(case["queries"]), _counts(case["keys"])
        total, kv, dim = sum(s["queries"]), case["kv_heads"], case["dim"]
        if op == "write_q4":
            s["out"] = torch.empty((total, kv * dim), device="cuda")
        else:
            s["out"] = torch.empty_like(s["q"])
    if op == "attention_q4" and not own:
        s["k"], s["v"] = _quantise(s["k"]), _quantise(s["v"])
    if op == "rope_axes":
        s["out"] = torch.empty_like(s["x"])
    if op == "logprobs":
        s["out"] = torch.empty((case["rows"], 2 + 2 * case["top"]), device="cuda")
    if not own:
        return s
    ks = _framework()
    b = s["buffers"] = {n: ks.wrap_tensor(t) for n, t in s.items() if isinstance(t, torch.Tensor)}
    if op in ("attention_packed", "attention_q4", "write_q4"):
        b["sequences"] = ks.sequences(s["queries"], s["keys"])
    if op == "attention_q4":
        for n in ("k", "v"):
            store = ks.kv_store_q4(s[n].shape[0], kv, dim)
            ks.kv_write(store, b[n], 0)
            b[n] = store
        torch.cuda.synchronize()
        del s["k"], s["v"]
    if op == "write_q4":
        b["store"] = ks.kv_store_q4(sum(s["keys"]), kv, dim)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    case, b, ks = s["case"], s["buffers"], _framework()
    op = case["op"]
    if op in ("attention_packed", "attention_q4"):
        ks.attention_packed(b["q"], b["k"], b["v"], b["sequences"], case["heads"], case["dim"], kv_head_count=case["kv_heads"],
                            causal=case["causal"], window_size=case["window"] or None, out=b["out"])
    elif op == "write_q4":
        ks.kv_write_packed(b["store"], b["rows"], b["sequences"])
        ks.kv_read_packed(b["store"], b["sequences"], out=b["out"])
    elif op == "rope_axes":
        ks.rope_axes(b["x"], b["positions"], _counts(case["sections"]), dimension=case["dimension"], head_count=case["heads"],
                     pairing=case["pairing"], order=case["order"], ladder=case["ladder"], inverse=case["inverse"], out=b["out"])
    else:
        ks.token_logprobs(b["logits"], b["tokens"], top=case["top"], temperature=case["temperature"], out=b["out"])
        return _columns(s["out"], case["top"])
    return s["out"]


def _columns(out, top):
    return {"logprob": out[:, 0], "entropy": out[:, 1], "top": out[:, 2:2 + top], "ids": out[:, 2 + top:]}


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "attention_packed":
        return _attention(case, s["q"], s["k"], s["v"], torch.float32)
    if op == "attention_q4":
        return _attention(case, s["q"], s["k"], s["v"], torch.float32)
    if op == "write_q4":
        return _dequantise(_quantise(s["rows"].float()))
    if op == "rope_axes":
        return _rope(case, s["x"].float(), s["positions"]).to(s["x"].dtype)
    return _logprobs(case, s["logits"].float(), s["tokens"])


def _quantise(x):
    """Blocks of 64 values of a row: the scale is the value of largest magnitude (the first of several) over -8, as
    bfloat16; each value is its quotient with the scale, rounded to the nearest whole number (ties to even) in [-8, 7]."""
    blocks = x.view(x.shape[0], -1, _Q4_BLOCK)
    at = blocks.abs().argmax(dim=2, keepdim=True)
    scale = (blocks.gather(2, at) / -8.0).to(torch.bfloat16)
    d = scale.float()
    codes = torch.where(d == 0, torch.zeros_like(blocks), torch.round(blocks / d).clamp_(-8, 7))
    return codes.to(torch.int8), scale


def _dequantise(packed, dtype=torch.float32):
    codes, scale = packed
    return (codes.to(dtype) * scale.to(dtype)).view(codes.shape[0], -1)


def _rows(kv, start, count, dtype):
    """Rows [start, start + count) of a tensor, or of a quantised store, in `dtype`."""
    if isinstance(kv, tuple):
        return _dequantise((kv[0][start:start + count], kv[1][start:start + count]), dtype)
    return kv[start:start + count].to(dtype)


def _attention(case, q, k, v, dtype):
    """softmax(q k^T / sqrt(dim)) v for each sequence; query i of n over m keys stands at position m - n + i."""
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    queries, keys = _counts(case["queries"]), _counts(case["keys"])
    out = torch.empty(q.shape, dtype=q.dtype if dtype == torch.float32 else dtype, device=q.device)
    for qs, n, ks, m in zip(_starts(queries), queries, _starts(keys), keys):
        qh = q[qs:qs + n].to(dtype).view(n, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)  # [kv, group * n, dim]
        kh = _rows(k, ks, m, dtype).view(m, kv, dim).permute(1, 2, 0)
        vh = _rows(v, ks, m, dtype).view(m, kv, dim).permute(1, 0, 2)
        scores = torch.bmm(qh, kh).mul_(1.0 / math.sqrt(dim)).view(kv, heads // kv, n, m)
        if case["causal"]:
            at = torch.arange(m - n, m, device=q.device).view(n, 1)
            key = torch.arange(m, device=q.device).view(1, m)
            hidden = key > at
            if case["window"]:
                hidden |= key <= at - case["window"]
            scores.masked_fill_(hidden, -math.inf)
        scores -= scores.amax(dim=3, keepdim=True)
        scores.exp_()
        scores /= scores.sum(dim=3, keepdim=True)
        o = torch.bmm(scores.view(kv, -1, m), vh).view(kv, heads // kv, n, dim)
        out[qs:qs + n] = o.permute(2, 0, 1, 3).reshape(n, heads * dim).to(out.dtype)
    return out


def _axis_of_pairs(sections, order):
    """The axis of each pair, and its place among the pairs of that axis."""
    pairs, axes = sum(sections), len(sections)
    if order == "blocks":
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    else:
        axis = [i % axes if i % axes and i // axes < sections[i % axes] else 0 for i in range(pairs)]
    seen, place = [0] * axes, []
    for a in axis:
        place.append(seen[a])
        seen[a] += 1
    return axis, place


def _frequencies(case):
    sections = _counts(case["sections"])
    axis, place = _axis_of_pairs(sections, case["order"])
    if case["ladder"] == "shared":
        freq = [10000.0 ** (-i / len(axis)) for i in range(len(axis))]
    else:
        freq = [10000.0 ** (-j / sections[a]) for a, j in zip(axis, place)]
    return axis, freq


def _rope(case, x, positions):
    """Pairs of each head rotated by (position on the pair's axis) x (frequency of the pair, rounded to 32 bits)."""
    rows, heads, width, dim = case["rows"], case["heads"], case["width"], case["dimension"]
    axis, freq = _frequencies(case)
    f = torch.tensor(freq, dtype=torch.float64).to(torch.float32).to(x.device)
    angle = positions.to(x.dtype)[:, torch.tensor(axis, device=x.device)] * f.to(x.dtype)
    c, s = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    if case["inverse"]:
        s = -s
    out = x.clone().view(rows, heads, width)
    h = x.view(rows, heads, width)
    half = dim // 2
    first, second = (slice(0, half), slice(half, dim)) if case["pairing"] == "half_split" else (slice(0, dim, 2), slice(1, dim, 2))
    out[..., first] = h[..., first] * c - h[..., second] * s
    out[..., second] = h[..., first] * s + h[..., second] * c
    return out.view(rows, -1)


def _top(x, k):
    """Columns of the k largest values of each row, ties to the lowest column."""
    bits = (x.to(torch.float32) + 0.0).view(torch.int32)
    bits = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    key = (bits << 32) | (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))
    return x.shape[1] - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)


def _logprobs(case, x, tokens):
    ids = _top(x, case["top"])
    x = x / case["temperature"]
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=1, keepdim=True)
    lse = top + total.log()
    p = e / total
    entropy = lse.squeeze(1) - torch.where(p > 0, p * x, torch.zeros_like(x)).sum(dim=1)
    return {"logprob": (x.gather(1, tokens.long().unsqueeze(1)) - lse).squeeze(1), "entropy": entropy,
            "top": x.gather(1, ids) - lse, "ids": ids.to(torch.float32)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def _pairs(case):
    """Query rows times the keys each of them sees."""
    total = 0
    for n, m in zip(_counts(case["queries"]), _counts(case["keys"])):
        if not case["causal"]:
            total += n * m
            continue
        w = case["window"] or m
        first = m - n + 1  # keys up to and with the first query's own
        short = max(0, min(n, w - first))  # queries that see fewer than w keys
        total += short * first + short * (short - 1) // 2 + (n - short) * w
    return total


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "rope_axes":
        n = case["rows"] * case["heads"] * case["width"]
        return {"bytes": 2 * n * size + 4 * case["rows"] * len(_counts(case["sections"])), "flops": 3 * n}
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + 4 * case["rows"] * (3 + 2 * case["top"]), "flops": 5 * n}
    total, keys, width = sum(_counts(case["queries"])), sum(_counts(case["keys"])), case["kv_heads"] * case["dim"]
    row = width // 2 + 2 * (width // _Q4_BLOCK)
    if op == "write_q4":
        return {"bytes": total * (width * size + row + row + 4 * width), "flops": 6 * total * width}
    q = total * case["heads"] * case["dim"]
    kv = 2 * keys * (row if op == "attention_q4" else width * size)
    return {"bytes": 2 * q * size + kv, "flops": 4 * case["heads"] * case["dim"] * _pairs(case)}


# ---- 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "rope_axes":
        return _exact_rope(case, s["x"].double(), s["positions"].double())
    if op == "logprobs":
        return _exact_logprobs(case, s["logits"], s["tokens"])
    if op == "write_q4":
        return _exact_q4(s["rows"])
    k, v = (_exact_q4(s["k"]), _exact_q4(s["v"])) if op == "attention_q4" else (s["k"].double(), s["v"].double())
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    at_q = at_k = 0
    for n, m in zip(_counts(case["queries"]), _counts(case["keys"])):
        for h in range(heads):
            g = h // (heads // kv)
            a = q[at_q:at_q + n, h * dim:(h + 1) * dim] @ k[at_k:at_k + m, g * dim:(g + 1) * dim].T / math.sqrt(dim)
            if case["causal"]:
                a += torch.full((n, m), -math.inf, dtype=torch.float64, device="cuda").triu_(m - n + 1)
                if case["window"]:
                    a += torch.full((n, m), -math.inf, dtype=torch.float64, device="cuda").tril_(m - n - case["window"])
            out[at_q:at_q + n, h * dim:(h + 1) * dim] = torch.softmax(a, dim=1) @ v[at_k:at_k + m, g * dim:(g + 1) * dim]
        at_q, at_k = at_q + n, at_k + m
    return out


def _exact_q4(x):
    """The values a 4-bit store holds for rows x; the scale and the quotients are rounded as the format says."""
    x = x.double()
    b = x.reshape(-1, _Q4_BLOCK)
    most, low = b.amax(dim=1), b.amin(dim=1)
    # the signed value of largest magnitude; where +m and -m both occur, the first of them
    first = torch.where(b == most[:, None], 1, 0).argmax(dim=1) < torch.where(b == low[:, None], 1, 0).argmax(dim=1)
    m = torch.where((most > -low) | ((most == -low) & first), most, low)
    d = (m / -8).float().to(torch.bfloat16).double()[:, None]
    q = (b / torch.where(d == 0, 1.0, d)).float().double().round().clamp(-8, 7)
    return torch.where(d == 0, 0.0, q * d).view(x.shape)


def _exact_rope(case, x, pos):
    axis, freq = _frequencies(case)
    half, out = case["dimension"] // 2, x.clone().view(case["rows"], case["heads"], case["width"])
    h = out.clone()
    for i, (a, f) in enumerate(zip(axis, freq)):
        p, r = (i, i + half) if case["pairing"] == "half_split" else (2 * i, 2 * i + 1)
        f32 = float(torch.tensor(f, dtype=torch.float64).float())
        turn = torch.polar(torch.ones_like(pos[:, a]), pos[:, a] * f32 * (-1 if case["inverse"] else 1))[:, None]
        z = torch.complex(h[:, :, p], h[:, :, r]) * turn
        out[:, :, p], out[:, :, r] = z.real, z.imag
    return out.view(x.shape)


def _exact_logprobs(case, logits, tokens):
    k, parts = case["top"], []
    for rows, ids in zip(logits.split(512), tokens.split(512)):
        order = torch.sort(rows.float(), dim=1, descending=True, stable=True).indices[:, :k]
        logp = torch.log_softmax(rows.double() / case["temperature"], dim=1)
        entropy = -torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(dim=1)
        parts.append((logp.gather(1, ids.long()[:, None])[:, 0], entropy, logp.gather(1, order), order.double()))
    a, b, c, d = (torch.cat(p) for p in zip(*parts))
    return {"logprob": a, "entropy": b, "top": c, "ids": d}
