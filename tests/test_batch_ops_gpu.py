"""GPU: the operators for batches of packed sequences -- attention over packed sequences, 4-bit key/value
stores, rope with several axes, token log probabilities -- against plain implementations in 64 bits.

Tolerances, from the kernels' own roundings.  Attention, relative L2: in f32 the tensor cores take each
operand as two bfloat16 terms (together within 2^-17 of it), in q, k, the weights and v: 4 * 2^-17 = 3.1e-5
at the worst, independent errors well below; the bound is 2e-5.  In bfloat16 and f16 the weights and the output
are each rounded once, by 2^-9 and 2^-12 of their value in the mean: 2 * 2^-9 and 2 * 2^-12.  Rope: sine, cosine
and three operations in f32, 8 * 2^-24; one output rounding for the half types, by at most 2^-8 and 2^-11.  Log probabilities: weights
2^d with |d| up to some 40 carry 40 * 2^-24 of relative error into the sum, a log-sum up to 16 rounds by
2^-21: 1e-5 absolute.  Writes into a 4-bit store are exact."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ATTENTION_TOL = {"f32": 2e-5, "bf16": 2 * 2.0 ** -9, "f16": 2 * 2.0 ** -12}
ROPE_TOL = {"f32": 8 * 2.0 ** -24, "bf16": 2.0 ** -8 + 1e-6, "f16": 2.0 ** -11 + 1e-6}


def randn(shape, dtype="f32", seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = (torch.randn(shape, generator=g, device="cuda") * scale).to(DT[dtype])
    torch.cuda.synchronize()
    return t


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def to_torch(kernels, buf, like=None):
    """A buffer's values as a torch tensor (a copy through the host)."""
    if buf.dtype == "f32":
        return torch.from_numpy(kernels.download(buf).copy()).cuda()
    raw = torch.from_numpy(kernels.download_raw(buf).astype(np.int32).astype(np.int16)).cuda()
    return raw.view(DT[buf.dtype])


def attention64(q, k, v, heads, kv, queries, keys, starts=None, causal=True, window=None, scale=None):
    """softmax(q k^T scale) v for each sequence, in f64; rows that see no key give zeros."""
    q, k, v = q.double(), k.double(), v.double()
    dim, vdim = q.shape[1] // heads, v.shape[1] // kv
    scale = scale or 1.0 / math.sqrt(dim)
    out = torch.zeros((q.shape[0], heads * vdim), dtype=torch.float64, device=q.device)
    at_q = at_k = 0
    for i, (n, m) in enumerate(zip(queries, keys)):
        k0 = starts[i] if starts else at_k
        for h in range(heads):
            g = h // (heads // kv)
            qs = q[at_q:at_q + n, h * dim:(h + 1) * dim]
            s = qs @ k[k0:k0 + m, g * dim:(g + 1) * dim].T * scale
            pos = torch.arange(m - n, m, device=q.device)[:, None]
            key = torch.arange(m, device=q.device)[None, :]
            seen = torch.ones((n, m), dtype=torch.bool, device=q.device)
            if causal:
                seen = key <= pos
                if window:
                    seen &= key > pos - window
            s = s.masked_fill(~seen, -math.inf)
            p = torch.where(seen.any(1, keepdim=True), torch.softmax(s, 1), torch.zeros_like(s)) if m else s
            out[at_q:at_q + n, h * vdim:(h + 1) * vdim] = p @ v[k0:k0 + m, g * vdim:(g + 1) * vdim]
        at_q, at_k = at_q + n, at_k + m
    return out


# ---------------------------------------------------------------------------- attention, plain keys and values
SHAPES = [(1, 1, 64), (4, 2, 64), (8, 8, 128), (8, 2, 128), (5, 1, 64), (16, 1, 128), (6, 2, 128), (2, 1, 80), (4, 4, 16), (2, 2, 256), (3, 1, 33)]
LENGTHS = [([1], None), ([128, 77, 1, 33], None), ([0, 5, 0, 300, 1, 0], None), ([129, 257, 64], [129, 300, 500]),
           ([3, 1, 1], [700, 1, 0]), ([9, 40], [4, 40])]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("queries,keys", LENGTHS)
def test_attention_packed(kernels, dtype, heads, kv, dim, queries, keys):
    keys = keys or queries
    q = randn((sum(queries), heads * dim), dtype, 1)
    k, v = randn((max(1, sum(keys)), kv * dim), dtype, 2), randn((max(1, sum(keys)), kv * dim), dtype, 3)
    seqs = kernels.sequences(queries, keys)
    for causal, window in ((True, None), (True, 50), (False, None)):
        out = kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim, kv_head_count=kv,
                                       causal=causal, window_size=window)
        assert out.dtype == dtype and out.shape == (sum(queries), heads * dim)
        got = to_torch(kernels, out)
        want = attention64(q, k, v, heads, kv, queries, keys, causal=causal, window=window)
        assert torch.isfinite(got).all()
        assert rel(got, want) <= ATTENTION_TOL[dtype], (causal, window)
        assert (got[want.abs().sum(1) == 0] == 0).all()  # rows that see no key


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (8, 4, 64), (3, 3, 80), (2, 1, 200)])
@pytest.mark.parametrize("queries,keys", [([1], [5000]), ([1, 1, 3], [2000, 1, 900]), ([40, 0, 1], [3000, 5, 64]), ([2, 300], [2, 1500])])
def test_attention_packed_few_queries_over_many_keys(kernels, dtype, heads, kv, dim, queries, keys):
    """Few rows, whose keys are split; a value of NaN that the last query of a sequence alone sees, and NaN behind its keys."""
    q = randn((sum(queries), heads * dim), dtype, 11)
    k, v = randn((sum(keys) + 1, kv * dim), dtype, 12), randn((sum(keys) + 1, kv * dim), dtype, 13)
    k[-1], v[-1] = math.nan, math.nan
    torch.cuda.synchronize()
    seqs = kernels.sequences(queries, keys)
    finite = v.clone()
    for poison in (False, True):
        if poison:
            finite[sum(keys) - 1, 0] = 0
            v[sum(keys) - 1, 0] = math.nan
            torch.cuda.synchronize()
        for causal, window in ((True, None), (True, 333), (False, None)):
            got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim,
                                                             kv_head_count=kv, causal=causal, window_size=window))
            want = attention64(q, k, finite, heads, kv, queries, keys, causal=causal, window=window)
            if poison:
                first = sum(queries) - (1 if causal else queries[-1])
                for h in range(heads // kv):  # the heads of that value column
                    want[first:, h * dim] = math.nan
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (poison, causal, window)
            fine = ~torch.isnan(want)
            assert rel(got[fine], want[fine]) <= ATTENTION_TOL[dtype], (poison, causal, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_packed_reads_its_own_keys_only(kernels, dtype, dim):
    """Keys in slots with NaN between them, in another order than the queries; a long sequence beside short ones."""
    heads, kv = 8, 2
    queries, keys, starts = [200, 3, 1, 70], [1000, 3, 513, 70], [600, 5, 40, 1700]
    q = randn((sum(queries), heads * dim), dtype, 4)
    k, v = randn((1801, kv * dim), dtype, 5), randn((1801, kv * dim), dtype, 6)
    used = torch.zeros(1801, dtype=torch.bool, device="cuda")
    for s, m in zip(starts, keys):
        used[s:s + m] = True
    k[~used] = math.nan
    v[~used] = math.nan
    torch.cuda.synchronize()
    seqs = kernels.sequences(queries, keys, starts)
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim, kv_head_count=kv))
    want = attention64(q, k, v, heads, kv, queries, keys, starts)
    assert rel(got, want) <= ATTENTION_TOL[dtype]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_packed_masked_values_do_not_leak(kernels, dtype):
    """Infinities and NaN in later keys (which the causal mask hides) leave the earlier rows as they are."""
    n, heads, dim = 300, 2, 128
    q, k, v = (randn((n, heads * dim), dtype, s) for s in (7, 8, 9))
    k[200:], v[200:] = math.inf, math.nan
    torch.cuda.synchronize()
    seqs = kernels.sequences([n])
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), seqs, heads, dim))
    want = attention64(q[:200], k[:200], v[:200], heads, heads, [200], [200])
    assert rel(got[:200], want) <= ATTENTION_TOL[dtype]
    assert torch.isnan(got[200:]).all()


@pytest.mark.parametrize("dtype,big", [("f32", 1e38), ("bf16", 1e38), ("f16", 6e4)])
def test_attention_packed_large_values_and_scores(kernels, dtype, big):
    """Values near the type's largest give a mean of them, not infinity; scores of thousands pick one key."""
    n, dim = 700, 128
    q, k = randn((n, dim), dtype, 10, 60.0), randn((n, dim), dtype, 11, 60.0)
    v = (randn((n, dim), "f32", 12).clamp(-1, 1) * big).to(DT[dtype])
    torch.cuda.synchronize()
    for scale in (None, 1e-4):
        got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), kernels.sequences([n]), 1, dim, scale=scale))
        want = attention64(q, k, v / big, 1, 1, [n], [n], scale=scale)
        assert torch.isfinite(got).all()
        # scores of up to s carry s * 2^-17 (f32's two terms) of absolute error into the weights
        tol = ATTENTION_TOL[dtype] + (6e4 * 2.0 ** -17 * 0.1 if scale is None and dtype == "f32" else 0.0)
        assert rel(got.double() / big, want) <= tol


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_packed_unaligned_buffers(kernels, dtype):
    """Buffers that start one element past an aligned address."""
    n, heads, kv, dim = 150, 4, 2, 64
    tensors = [torch.cat([randn(1, dtype), randn((n * w * dim,), dtype, 13 + w)])[1:] for w in (heads, kv, kv)]
    torch.cuda.synchronize()
    bufs = [kernels.wrap(t.data_ptr(), (n, w * dim), dtype, owner=t) for t, w in zip(tensors, (heads, kv, kv))]
    got = to_torch(kernels, kernels.attention_packed(*bufs, kernels.sequences([100, 50]), heads, dim, kv_head_count=kv))
    q, k, v = (t.view(n, -1) for t in tensors)
    assert rel(got, attention64(q, k, v, heads, kv, [100, 50], [100, 50])) <= ATTENTION_TOL[dtype]


def test_attention_packed_value_dimension_and_scale(kernels):
    q, k, v = randn((60, 4 * 64), "f32", 20), randn((60, 2 * 64), "f32", 21), randn((60, 2 * 24), "f32", 22)
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), kernels.sequences([20, 40]), 4, 64,
                                                     kv_head_count=2, value_dimension=24, scale=0.3))
    assert rel(got, attention64(q, k, v, 4, 2, [20, 40], [20, 40], scale=0.3)) <= ATTENTION_TOL["f32"]


def test_attention_packed_matches_attention_of_each_sequence(kernels):
    """The same rows as the framework's one-sequence attention gives."""
    heads, dim, lengths = 8, 64, [130, 1, 64]
    q, k, v = (randn((sum(lengths), heads * dim), "f32", s) for s in (30, 31, 32))
    got = to_torch(kernels, kernels.attention_packed(*(kernels.wrap_tensor(t) for t in (q, k, v)), kernels.sequences(lengths), heads, dim))
    at = 0
    for n in lengths:
        one = kernels.attention(*(kernels.wrap_tensor(t[at:at + n]) for t in (q, k, v)), heads, dim, causal=True)
        assert rel(got[at:at + n], to_torch(kernels, one)) <= 2 * ATTENTION_TOL["f32"]
        at += n


# ---------------------------------------------------------------------------- 4-bit stores
def quantise64(x):
    """The values a 4-bit store holds for x (the scale rounded to bfloat16, the quotient to f32)."""
    x = x.double()
    b = x.reshape(-1, 64)
    at = b.abs().argmax(1, keepdim=True)
    first = (b.abs() == b.abs().gather(1, at)).double().argmax(1, keepdim=True)  # argmax of a 0/1 row: its first 1
    d = (b.gather(1, first) / -8).float().bfloat16().double()
    q = (b / torch.where(d == 0, 1.0, d)).float().double().round().clamp(-8, 7)
    return torch.where(d == 0, 0.0, q * d).view(x.shape)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width,offset", [(1, 64, 0), (1, 128, 200), (63, 192, 1), (65, 1024, 100), (300, 256, 5)])
def test_kv_write_q4_is_exact(kernels, dtype, rows, width, offset):
    x = randn((rows, width), dtype, 40)
    x[0, :64] = 0
    x[-1, -3], x[-1, -2] = 9.0, -9.0  # two values of the same magnitude: the first one sets the scale
    torch.cuda.synchronize()
    store = kernels.kv_store_q4(400, width // 64, 64)
    assert store.dtype == "q4" and store.shape == (400, width)
    assert not kernels.download(store).any()
    kernels.kv_write(store, kernels.wrap_tensor(x), offset)
    got = torch.from_numpy(kernels.download(store)).cuda()
    want = torch.zeros((400, width), dtype=torch.float64, device="cuda")
    want[offset:offset + rows] = quantise64(x)
    assert torch.equal(got.double(), want)
    assert float((got[offset:offset + rows].double() - x.double()).abs().max()) <= 0.13 * float(x.double().abs().max())


def test_kv_write_q4_extremes(kernels):
    """Blocks of the smallest and the largest f32 values, of one repeated value, and with values that are not finite."""
    x = randn((8, 128), "f32", 41)
    x[0] *= 1e-36
    x[1] = x[1].clamp(-3, 3) * 1e38
    x[2] = 0.7
    x[3] = -0.7
    x[4, 5] = math.nan
    x[5, 70] = -math.inf
    x[6, 0] = 1e-44  # a denormal beside larger ones
    x[7] = 1e-44
    torch.cuda.synchronize()
    store = kernels.kv_store_q4(8, 1, 128)
    kernels.kv_write(store, kernels.wrap_tensor(x), 0)
    got = torch.from_numpy(kernels.download(store)).cuda().double()
    for r, c in ((4, 0), (5, 1)):
        assert torch.isnan(got[r, 64 * c:64 * c + 64]).all()
        assert torch.isfinite(got[r, 64 * (1 - c):64 * (1 - c) + 64]).all()
    fine = [0, 1, 2, 3, 6]
    assert torch.equal(got[fine], quantise64(x[fine]))
    assert torch.isfinite(got[7]).all() and float(got[7].abs().max()) <= 2e-44


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_kv_write_packed_and_read(kernels, dtype):
    queries, keys, starts = [1, 0, 70, 3, 1], [100, 4, 70, 64, 1], [300, 0, 130, 200, 64]
    x = randn((sum(queries), 256), dtype, 42)
    store = kernels.kv_store_q4(401, 2, 128)
    seqs = kernels.sequences(queries, keys, starts)
    kernels.kv_write_packed(store, kernels.wrap_tensor(x), seqs)
    want = quantise64(x)
    assert torch.equal(to_torch(kernels, kernels.kv_read_packed(store, seqs)).double(), want)
    whole, at = torch.zeros((401, 256), dtype=torch.float64, device="cuda"), 0
    for n, m, s in zip(queries, keys, starts):
        whole[s + m - n:s + m] = want[at:at + n]
        at += n
    assert torch.equal(torch.from_numpy(kernels.download(store)).cuda().double(), whole)
    # a store of the rows' own type
    plain = kernels.wrap_tensor(torch.zeros((401, 256), dtype=DT[dtype], device="cuda"))
    torch.cuda.synchronize()
    kernels.kv_write_packed(plain, kernels.wrap_tensor(x), seqs)
    got, at = to_torch(kernels, plain), 0
    for n, m, s in zip(queries, keys, starts):
        assert torch.equal(got[s + m - n:s + m], x[at:at + n])
        at += n
    assert float(got.double().abs().sum()) == pytest.approx(float(x.double().abs().sum()), rel=1e-12)


Q4_LENGTHS = [([1], [1]), ([1], [64]), ([1], [1000]), ([1, 1, 1, 1], [129, 17, 500, 64]), ([1, 0, 3, 1], [5000, 0, 70, 0]),
              ([4, 2, 33], [300, 2, 1000]), ([40], [20]), ([1] * 40, list(range(1, 41)))]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 8, 64), (8, 2, 128), (16, 2, 128), (5, 1, 128), (24, 1, 64), (2, 1, 192), (3, 3, 256)])
@pytest.mark.parametrize("queries,keys", Q4_LENGTHS)
def test_attention_over_q4_stores(kernels, dtype, heads, kv, dim, queries, keys):
    # slots of their own, starting at any row, with NaN between them
    starts, at = [], 7
    for m in keys:
        starts.append(at)
        at += m + 5
    q = randn((sum(queries), heads * dim), dtype, 50)
    k, v = randn((at, kv * dim), "f32", 51), randn((at, kv * dim), "f32", 52, 1e-3)
    hole = torch.ones(at, dtype=torch.bool, device="cuda")
    for s, m in zip(starts, keys):
        hole[s:s + m] = False
    k[hole], v[hole] = math.nan, math.nan
    torch.cuda.synchronize()
    ks, vs = kernels.kv_store_q4(at, kv, dim), kernels.kv_store_q4(at, kv, dim)
    kernels.kv_write(ks, kernels.wrap_tensor(k), 0)
    kernels.kv_write(vs, kernels.wrap_tensor(v), 0)
    seqs = kernels.sequences(queries, keys, starts)
    k64, v64 = quantise64(k), quantise64(v)
    for causal, window in ((True, None), (True, 100), (False, None)):
        got = to_torch(kernels, kernels.attention_packed(kernels.wrap_tensor(q), ks, vs, seqs, heads, dim, kv_head_count=kv,
                                                         causal=causal, window_size=window))
        want = attention64(q, k64, v64, heads, kv, queries, keys, starts, causal, window)
        assert torch.isfinite(got).all()
        # values of a thousandth: f16 outputs lie in its denormals, whose step is 2^-24
        tol = ATTENTION_TOL[dtype] + (2.0 ** -25 / 1e-4 if dtype == "f16" else 0.0)
        assert rel(got, want) <= tol, (causal, window)
        assert (got[want.abs().sum(1) == 0] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_over_q4_masked_rows_do_not_leak(kernels, dtype):
    """A later key of NaN, hidden from the first queries by the causal mask; a large score; large values."""
    heads, kv, dim, n, m = 4, 2, 128, 3, 200
    q = randn((n, heads * dim), dtype, 53)
    k, v = randn((m, kv * dim), "f32", 54, 30.0), randn((m, kv * dim), "f32", 55).clamp(-3, 3) * 1e38
    k[m - 1], v[m - 1] = math.nan, math.nan
    torch.cuda.synchronize()
    ks, vs = kernels.kv_store_q4(m, kv, dim), kernels.kv_store_q4(m, kv, dim)
    kernels.kv_write(ks, kernels.wrap_tensor(k), 0)
    kernels.kv_write(vs, kernels.wrap_tensor(v), 0)
    got = to_torch(kernels, kernels.attention_packed(kernels.wrap_tensor(q), ks, vs, kernels.sequences([n], [m]), heads, dim, kv_head_count=kv))
    want = attention64(q[:2], quantise64(k[:m - 1]), quantise64(v[:m - 1]) / 1e38, heads, kv, [2], [m - 1])
    # scores of some hundreds: f32's two terms leave 300 * 2^-17 in the weights
    assert rel(got[:2].double() / 1e38, want) <= ATTENTION_TOL[dtype] + 300 * 2.0 ** -17
    assert torch.isnan(got[2]).all()


# ---------------------------------------------------------------------------- rope with several axes
def rope64(x, pos, sections, heads, dimension, pairing, order, ladder, inverse, base=10000.0, scale=1.0):
    half, axes = dimension // 2, len(sections)
    if order == "blocks":
        axis = [a for a in range(axes) for _ in range(sections[a])]
    else:
        axis = [i % axes if i % axes and i // axes < sections[i % axes] else 0 for i in range(half)]
    place = [sum(1 for b in axis[:i] if b == a) for i, a in enumerate(axis)]
    f = [base ** (-i / half) if ladder == "shared" else base ** (-place[i] / sections[axis[i]]) for i in range(half)]
    f = torch.tensor(f, dtype=torch.float64, device="cuda").float()
    angle = ((pos * scale)[:, axis] * f).double()[:, None, :]  # rounded to f32, as the operator says
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    h = x.double().view(x.shape[0], heads, -1)
    out = h.clone()
    a, b = (slice(0, half), slice(half, dimension)) if pairing == "half_split" else (slice(0, dimension, 2), slice(1, dimension, 2))
    out[..., a] = h[..., a] * c - h[..., b] * s
    out[..., b] = h[..., a] * s + h[..., b] * c
    return out.view(x.shape)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pairing", ["interleaved", "half_split"])
@pytest.mark.parametrize("rows,heads,width,dimension,sections,order,ladder", [
    (1, 1, 2, 2, [1], "blocks", "shared"), (729, 16, 64, 64, [16, 16], "blocks", "per_axis"),
    (50, 4, 128, 128, [24, 20, 20], "cyclic", "shared"), (33, 3, 80, 40, [8, 6, 6], "blocks", "shared"),
    (7, 2, 13, 6, [2, 1], "cyclic", "per_axis"), (5, 1, 256, 256, [32, 32, 32, 32], "cyclic", "per_axis"),
    (1000, 1, 32, 32, [16, 0], "blocks", "shared")])
def test_rope_axes(kernels, dtype, pairing, rows, heads, width, dimension, sections, order, ladder):
    x = randn((rows, heads * width), dtype, 60)
    pos = torch.floor(randn((rows, len(sections)), "f32", 61).abs() * 300)
    torch.cuda.synchronize()
    kw = dict(dimension=dimension, head_count=heads, pairing=pairing, order=order, ladder=ladder)
    xb, pb = kernels.wrap_tensor(x), kernels.wrap_tensor(pos)
    for inverse in (False, True):
        out = kernels.rope_axes(xb, pb, sections, inverse=inverse, **kw)
        assert out.dtype == dtype
        want = rope64(x, pos, sections, heads, dimension, pairing, order, ladder, inverse)
        assert rel(to_torch(kernels, out), want) <= ROPE_TOL[dtype]
    # unaligned, and in place
    flat = torch.cat([randn(1, dtype), x.reshape(-1)])[1:]
    torch.cuda.synchronize()
    ub = kernels.wrap(flat.data_ptr(), x.shape, dtype, owner=flat)
    assert kernels.rope_axes(ub, pb, sections, out=ub, **kw) is ub
    assert rel(flat.view(x.shape), rope64(x, pos, sections, heads, dimension, pairing, order, ladder, False)) <= ROPE_TOL[dtype]


def test_rope_axes_one_axis_is_rope(kernels):
    """One axis with positions 0, 1, 2, ...: the framework's rope (whose frequency powf rounds in f32)."""
    x = randn((100, 4 * 64), "f32", 62)
    pos = torch.arange(100, device="cuda", dtype=torch.float32).view(100, 1)
    torch.cuda.synchronize()
    for pairing in ("interleaved", "half_split"):
        a = kernels.rope_axes(kernels.wrap_tensor(x), kernels.wrap_tensor(pos), [32], head_count=4, pairing=pairing)
        b = kernels.rope(kernels.wrap_tensor(x), head_count=4, pairing=pairing)
        assert rel(to_torch(kernels, a), to_torch(kernels, b)) <= 1e-5


def test_rope_axes_gradient(kernels):
    """The inverse rotation is the gradient: against the formula's and against differences."""
    rows, heads, width, sections = 6, 2, 16, [3, 3, 2]
    x, y = randn((rows, heads * width), "f32", 63), randn((rows, heads * width), "f32", 64)
    pos = torch.floor(randn((rows, 3), "f32", 65).abs() * 40)
    torch.cuda.synchronize()
    kw = dict(sections=sections, head_count=heads, pairing="half_split", order="cyclic")
    pb = kernels.wrap_tensor(pos)
    grad = to_torch(kernels, kernels.rope_axes(kernels.wrap_tensor(y), pb, inverse=True, **kw)).double()
    xd = x.double().requires_grad_(True)
    (rope64(xd, pos, sections, heads, width, "half_split", "cyclic", "shared", False) * y.double()).sum().backward()
    assert rel(grad, xd.grad) <= ROPE_TOL["f32"]
    # the map is linear: a difference along e gives <y, R e> up to f32's rounding
    e = randn(x.shape, "f32", 66)
    torch.cuda.synchronize()
    f = [to_torch(kernels, kernels.rope_axes(kernels.wrap_tensor((x + s * e).contiguous()), pb, **kw)).double() for s in (0.5, -0.5)]
    assert float(((f[0] - f[1]) * y.double()).sum()) == pytest.approx(float((grad * e.double()).sum()), abs=1e-4)


# ---------------------------------------------------------------------------- token log probabilities
def logprobs64(x, tokens, top, temperature):
    z = x.double() / temperature
    logp = torch.log_softmax(z, 1)
    entropy = -torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(1)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    chosen = torch.full((x.shape[0],), math.nan, dtype=torch.float64, device="cuda")
    ok = (tokens >= 0) & (tokens < x.shape[1]) & (tokens == tokens.floor())
    chosen[ok] = logp[ok].gather(1, tokens[ok].long()[:, None])[:, 0]
    return torch.cat([chosen[:, None], entropy[:, None], logp.gather(1, order), order.double()], 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,top,temperature", [(1, 1, 1, 1.0), (3, 5, 5, 0.7), (8, 32000, 5, 1.0), (5, 50001, 20, 1.3), (300, 999, 64, 1.0),
                                                        (2, 131073, 32, 1.0), (4, 64, 0, 2.0), (160, 1024, 1, 1.0)])
def test_token_logprobs(kernels, dtype, rows, vocab, top, temperature):
    x = randn((rows, vocab), dtype, 70, 3.0)
    x[::3, : vocab // 2] = -math.inf
    if vocab > 8:
        x[1::3, ::2] = torch.finfo(DT[dtype]).min if temperature >= 1 else -1e4  # a mask of the type's lowest value
    tokens = torch.randint(0, vocab, (rows,), device="cuda").float()
    tokens[1::4] = -1
    torch.cuda.synchronize()
    out = kernels.token_logprobs(kernels.wrap_tensor(x), kernels.wrap_tensor(tokens), top=top, temperature=temperature)
    assert out.shape == (rows, 2 + 2 * top)
    got, want = to_torch(kernels, out).double(), logprobs64(x, tokens, top, temperature)
    assert torch.equal(got[:, 2 + top:], want[:, 2 + top:])
    a, b = got[:, :2 + top], want[:, :2 + top]
    assert torch.equal(torch.isnan(a), torch.isnan(b))
    far = b < -1e30  # the log probability of a lowest value: only f32's range
    assert torch.equal(torch.isinf(a) & ~far, torch.isinf(b) & ~far)
    fine = torch.isfinite(b) & ~far
    assert float((a[fine] - b[fine]).abs().max() / 1e-5) <= 1.0 + float(b[fine].abs().max()) * 0.1
    # without tokens: NaN in the first column, the rest as before
    none = to_torch(kernels, kernels.token_logprobs(kernels.wrap_tensor(x), top=top, temperature=temperature)).double()
    assert torch.isnan(none[:, 0]).all() and torch.equal(none[:, 1:], got[:, 1:])


def test_token_logprobs_ties_and_rows_without_a_distribution(kernels):
    vocab = 20000
    x = torch.zeros((8, vocab), device="cuda")
    x[1, 7::7] = 1.0             # many equal largest values
    x[2] = -math.inf             # nothing left
    x[3, 5] = math.nan
    x[4, 5] = math.inf
    x[5] = -math.inf
    x[5, [3, 19000]] = torch.tensor([1.0, 2.0], device="cuda")  # fewer finite values than asked for
    x[6, ::2] = -0.0             # equal to +0
    x[7] = torch.finfo(torch.float32).min
    tokens = torch.tensor([0, 7, 0, 0, 0, 3, 1, 2], device="cuda", dtype=torch.float32)
    torch.cuda.synchronize()
    got = to_torch(kernels, kernels.token_logprobs(kernels.wrap_tensor(x), kernels.wrap_tensor(tokens), top=4)).double()
    assert torch.isnan(got[2:5]).all()
    n = vocab // 7
    flat = -math.log(vocab)
    assert got[0].tolist() == pytest.approx([flat, -flat] + [flat] * 4 + [0, 1, 2, 3], abs=1e-5)
    assert got[1, 6:].tolist() == [7, 14, 21, 28]
    assert float(got[1, 0]) == pytest.approx(1 - math.log(n * math.e + vocab - n), abs=1e-5)
    assert got[5, 6:].tolist() == [19000, 3, 0, 1] and torch.isinf(got[5, 4:6]).all()
    assert got[6].tolist() == pytest.approx(got[0].tolist(), abs=1e-6)
    assert got[7].tolist() == pytest.approx(got[0].tolist(), abs=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("vocab,top", [(70, 64), (1024, 5), (32000, 20), (32000, 64)])
def test_token_logprobs_of_few_allowed_columns(kernels, dtype, rows, vocab, top):
    """A mask (-inf, or the type's lowest value) that leaves three columns, fewer than the top; a row of one value;
    a row whose finite logits are all in every 256th column: columns of equal logits come in order."""
    x = torch.full((rows, vocab), -math.inf, dtype=DT[dtype], device="cuda")
    x[1] = torch.finfo(DT[dtype]).min
    x[:, [5, vocab // 2, vocab - 1]] = randn((rows, 3), dtype, 75)
    x[2] = 0.5
    x[3, ::256] = randn((vocab + 255) // 256, dtype, 76)
    torch.cuda.synchronize()
    got = to_torch(kernels, kernels.token_logprobs(kernels.wrap_tensor(x), None, top=top))
    want = logprobs64(x, torch.full((rows,), -1.0, device="cuda"), top, 1.0)
    assert torch.equal(got[:, 2 + top:].double(), want[:, 2 + top:])
    finite = torch.isfinite(want[:, 1:2 + top]) & (want[:, 1:2 + top].abs() < 1e30)
    assert torch.equal(got[:, 1:2 + top][~finite].double(), want[:, 1:2 + top][~finite].float().double())
    assert float((got[:, 1:2 + top].double() - want[:, 1:2 + top])[finite].abs().max()) <= 1e-5


def test_token_logprobs_rows_on_odd_addresses(kernels):
    x = randn((1 + 3 * 1001,), "bf16", 71)[1:].view(3, 1001)
    tokens = torch.tensor([0.0, 1000.0, 500.5], device="cuda")
    torch.cuda.synchronize()
    buf = kernels.wrap(x.data_ptr(), (3, 1001), "bf16", owner=x)
    got = to_torch(kernels, kernels.token_logprobs(buf, kernels.wrap_tensor(tokens), top=3)).double()
    want = logprobs64(x, tokens, 3, 1.0)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert float(torch.nan_to_num(got - want).abs().max()) <= 1e-5


# ---------------------------------------------------------------------------- refusals
def test_refusals(kernels, mpc):
    def refused(code, f, *a, **kw):
        with pytest.raises(mpc.CudaError) as e:
            f(*a, **kw)
        assert e.value.code == code, e.value

    f32, bf16 = kernels.zeros((10, 256)), kernels.zeros((10, 256), "bf16")
    seqs = kernels.sequences([4, 6])
    store = kernels.kv_store_q4(10, 2, 128)
    att = kernels.attention_packed
    refused("ShapeUnsupported", kernels.sequences, [])
    refused("ShapeUnsupported", kernels.sequences, [2 ** 31])
    refused("ShapeUnsupported", kernels.sequences, [1], [1], [2 ** 31])
    refused("ShapeUnsupported", kernels.sequences, [2 ** 30, 2 ** 30])
    refused("ShapeUnsupported", kernels.write_sequences, seqs, [1])
    refused("DTypeUnsupported", kernels.write_sequences, f32, [1])
    refused("DTypeUnsupported", att, f32, bf16, bf16, seqs, 2, 128)
    refused("DTypeUnsupported", att, f32, store, f32, seqs, 2, 128)
    refused("DTypeUnsupported", att, store, store, store, seqs, 2, 128)
    refused("DTypeUnsupported", att, f32, f32, f32, f32, 2, 128)
    refused("ShapeUnsupported", att, f32, f32, f32, kernels.sequences([4, 5]), 2, 128)
    refused("ShapeUnsupported", att, f32, f32, f32, kernels.sequences([4, 6], [4, 7]), 2, 128)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 2, 64)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 3, 128)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 0, 128)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 2, 128, kv_head_count=3)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 2, 128, window_size=0)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 2, 128, window_size=4, causal=False)
    refused("ShapeUnsupported", att, f32, f32, f32, seqs, 2, 128, scale=-1.0)
    refused("ShapeUnsupported", att, f32, store, store, seqs, 8, 32)
    refused("ShapeUnsupported", kernels.kv_store_q4, 10, 1, 96)
    refused("ShapeUnsupported", kernels.kv_store_q4, 0, 1, 64)
    refused("ShapeUnsupported", kernels.kv_write, store, f32, 1)
    refused("ShapeUnsupported", kernels.kv_write, store, kernels.zeros((1, 128)), 0)
    refused("ShapeUnsupported", kernels.kv_write_packed, store, f32, kernels.sequences([4, 6], [4, 7]))
    refused("ShapeUnsupported", kernels.kv_write_packed, store, f32, kernels.sequences([4, 6], [4, 5]))
    refused("ShapeUnsupported", kernels.kv_write_packed, store, kernels.zeros((9, 256)), seqs)
    refused("DTypeUnsupported", kernels.kv_write_packed, bf16, f32, seqs)
    refused("DTypeUnsupported", kernels.kv_write_packed, store, store, seqs)
    refused("DTypeUnsupported", kernels.kv_read_packed, f32, seqs)
    # opaque buffers have no elements of their own, and no other operator reads them
    refused("DTypeUnsupported", kernels.add, store, store)
    refused("DTypeUnsupported", kernels.add_half, store, store)
    refused("DTypeUnsupported", kernels.matmul, f32, store, transpose_b=True)
    refused("DTypeUnsupported", kernels.download, seqs)
    refused("DTypeUnsupported", kernels.empty, (4, 64), "q4")
    refused("DTypeUnsupported", kernels.wrap, f32.data_ptr(), (4, 64), "q4")
    refused("LayoutUnsupported", store.reshape, (2560,))
    refused("DTypeUnsupported", store.write, np.zeros((10, 256), np.float32))
    # rope and log probabilities
    pos = kernels.zeros((10, 2))
    refused("ShapeUnsupported", kernels.rope_axes, f32, pos, [10, 20], head_count=2)
    refused("ShapeUnsupported", kernels.rope_axes, f32, pos, [64], head_count=2)
    refused("ShapeUnsupported", kernels.rope_axes, f32, pos, [1, 63], head_count=2, order="cyclic")
    refused("ShapeUnsupported", kernels.rope_axes, f32, pos, [32, 32], head_count=3)
    refused("ShapeUnsupported", kernels.rope_axes, f32, pos, [32, 32], head_count=2, base=0.0)
    refused("DTypeUnsupported", kernels.rope_axes, f32, bf16, [32, 32], head_count=2)
    refused("DTypeUnsupported", kernels.rope_axes, store, pos, [32, 32], head_count=2)
    refused("ShapeUnsupported", kernels.token_logprobs, f32, top=65)
    refused("ShapeUnsupported", kernels.token_logprobs, kernels.zeros((2, 3)), top=4)
    refused("ShapeUnsupported", kernels.token_logprobs, f32, kernels.zeros((9,)))
    refused("ShapeUnsupported", kernels.token_logprobs, f32, temperature=0.0)
    refused("DTypeUnsupported", kernels.token_logprobs, store)
    refused("DTypeUnsupported", kernels.token_logprobs, f32, kernels.zeros((10,), "bf16"))


# ---------------------------------------------------------------------------- streams, tables, the executor
def test_operators_on_another_stream(kernels):
    """On a caller's stream, behind work that is still running there."""
    side = torch.cuda.Stream()
    n, heads, dim = 400, 4, 128
    a = torch.randn((2048, 2048), device="cuda")
    q, k, v = (randn((n, heads * dim), "f32", s) for s in (80, 81, 82))
    want = attention64(q, k, v, heads, heads, [n], [n])
    kernels.set_stream(side.cuda_stream)
    try:
        with torch.cuda.stream(side):
            late = torch.zeros_like(q)
            for _ in range(20):
                a = a @ a * 1e-3
            late.copy_(q)
            out = torch.empty_like(q)
            kernels.attention_packed(kernels.wrap_tensor(late), kernels.wrap_tensor(k), kernels.wrap_tensor(v), kernels.sequences([n]),
                                     heads, dim, out=kernels.wrap_tensor(out))
            got = out * 1.0
        side.synchronize()
    finally:
        kernels.set_stream(None)
    assert rel(got, want) <= ATTENTION_TOL["f32"]


def test_table_rewritten_between_calls(kernels):
    heads, dim = 2, 64
    q, k, v = (randn((100, heads * dim), "bf16", s) for s in (83, 84, 85))
    bufs = [kernels.wrap_tensor(t) for t in (q, k, v)]
    seqs = kernels.sequences([100, 0])
    for lengths in ([100, 0], [1, 99], [50, 50], [99, 1]):
        kernels.write_sequences(seqs, lengths)
        got = to_torch(kernels, kernels.attention_packed(*bufs, seqs, heads, dim))
        assert rel(got, attention64(q, k, v, heads, heads, lengths, lengths)) <= ATTENTION_TOL["bf16"]


def test_executor_decode_loop_over_a_q4_store(kernels, executor, mpc):
    """Captured once, replayed for token after token of three sequences in slots of one store: the new keys and
    values are written, then attended to; the key counts advance with the replay's offset."""
    heads, kv, dim, slot, ages = 4, 2, 64, 200, [70, 1, 130]
    inv = mpc.KernelInvocation
    total = slot * 3
    k, v = randn((total, kv * dim), "f32", 90), randn((total, kv * dim), "f32", 91)
    starts = [0, slot, 2 * slot]
    for name, t in (("ks", k), ("vs", v)):
        store = kernels.kv_store_q4(total, kv, dim)
        for s, m in zip(starts, ages):
            kernels.kv_write(store, kernels.wrap_tensor(t[s:s + m - 1]), s)
        executor.adopt(name, store)
    executor.adopt("seqs", kernels.sequences([1, 1, 1], ages, starts))
    steps = 40
    q = randn((steps, 3, heads * dim), "f32", 92)
    torch.cuda.synchronize()
    host = {"q": q.cpu().numpy(), "k": k.cpu().numpy(), "v": v.cpu().numpy()}
    for name, w in (("q", heads), ("kn", kv), ("vn", kv)):
        executor.write_zeroed_tensor(name, (3, w * dim))
    nodes = [inv("kv-write-packed", ["ks", "kn", "seqs"], "ks"), inv("kv-write-packed", ["vs", "vn", "seqs"], "vs"),
             inv("attention-packed", ["q", "ks", "vs", "seqs"], "out",
                 {"head_count": heads, "head_dimension": dim, "kv_head_count": kv, "causal": True})]
    for n in nodes:
        executor.run(n)
    executor.begin_step_capture(["key_count"])
    for n in nodes:
        executor.run(n)
    executor.end_step_capture()
    assert executor.step_max_offset() == min(slot - m for m in ages)
    k64, v64 = quantise64(k), quantise64(v)
    out = np.empty((3, heads * dim), np.float32)
    for i in range(steps):
        rows = [s + m - 1 + i for s, m in zip(starts, ages)]
        executor.replay_step_io({"q": host["q"][i].copy(), "kn": host["k"][rows].copy(), "vn": host["v"][rows].copy()}, {"out": out}, offset=i)
        want = attention64(q[i], k64, v64, heads, kv, [1] * 3, [m + i for m in ages], starts)
        assert rel(torch.from_numpy(out).cuda(), want) <= ATTENTION_TOL["f32"], i
    with pytest.raises(mpc.CudaError) as e:
        executor.replay_step(offset=slot)
    assert e.value.code == "CaptureUnsupported"
    with pytest.raises(mpc.CudaError) as e:
        kernels.write_sequences(executor.buffer("seqs"), [1, 1, 1], ages, starts)
    assert e.value.code == "CaptureUnsupported"


def test_executor_kernels(kernels, executor, mpc):
    inv = mpc.KernelInvocation
    x = randn((6, 2 * 32), "f32", 93)
    pos = torch.floor(randn((6, 3), "f32", 94).abs() * 50)
    torch.cuda.synchronize()
    executor.write_tensor("x", x.cpu().numpy())
    executor.write_tensor("pos", pos.cpu().numpy())
    executor.run(inv("rope-axes", ["x", "pos"], "xr", {"dimension": 32, "head_count": 2, "sections": "6,5,5", "section_order": "cyclic",
                                                       "rotation_pairing": "half_split", "frequency_ladder": "per_axis"}))
    want = rope64(x, pos, [6, 5, 5], 2, 32, "half_split", "cyclic", "per_axis", False)
    assert rel(torch.from_numpy(executor.read_tensor("xr")).cuda(), want) <= ROPE_TOL["f32"]
    executor.write_tensor("ids", np.arange(6, dtype=np.float32))
    executor.run(inv("token-logprobs", ["x", "ids"], "lp", {"top": 3, "temperature": 0.5}))
    want = logprobs64(x, torch.arange(6, device="cuda").float(), 3, 0.5)
    assert float((torch.from_numpy(executor.read_tensor("lp")).cuda() - want).abs().max()) <= 1e-5
    # a kv-write-packed that does not end in its store leaves it as it was
    executor.adopt("store", kernels.kv_store_q4(6, 1, 64))
    executor.adopt("seqs", kernels.sequences([2, 4]))
    executor.run(inv("kv-write-packed", ["store", "x", "seqs"], "store2"))
    assert not executor.read_tensor("store").any()
    executor.copy_tensor("store2", "store3")
    executor.run(inv("kv-read-packed", ["store3", "seqs"], "back"))
    assert torch.equal(torch.from_numpy(executor.read_tensor("back")).cuda().double(), quantise64(x))
    executor.run(inv("kv-write", ["store", "x"], "store", {"row_offset": 0}))
    assert np.array_equal(executor.read_tensor("store"), executor.read_tensor("back"))
    for bad, code in ((inv("rope-axes", ["x", "pos"], "o", {"dimension": 32, "head_count": 2, "sections": "6,x"}), "KernelAttributeUnsupported"),
                      (inv("rope-axes", ["x", "pos"], "o", {"dimension": 32, "head_count": 2}), "KernelAttributeUnsupported"),
                      (inv("rope-axes", ["x", "pos"], "o", {"dimension": 32, "head_count": 2, "sections": "6,5,5", "section_order": "odd"}),
                       "KernelAttributeUnsupported"),
                      (inv("token-logprobs", ["x"], "o", {"top": -1}), "KernelAttributeUnsupported"),
                      (inv("attention-packed", ["x", "x", "x"], "o", {"head_count": 2, "head_dimension": 32}), "ExecutionFailed"),
                      (inv("attention-packed", ["x", "x", "x", "seqs"], "o", {"head_count": 2, "head_dimension": 32, "key_count": 3}),
                       "ShapeUnsupported"),
                      (inv("add", ["store", "store"], "o"), "DTypeUnsupported")):
        assert executor.submit_kernel(bad).error_code == code


def test_executor_decode_loop_over_long_plain_stores(kernels, executor, mpc):
    """The same loop over f32 stores, with slots so long that the keys are split: the parts follow the key counts."""
    heads, kv, dim, slot, ages = 4, 2, 64, 3000, [1500, 10, 700]
    inv = mpc.KernelInvocation
    total, starts = slot * 3, [0, slot, 2 * slot]
    k, v = randn((total, kv * dim), "f32", 95), randn((total, kv * dim), "f32", 96)
    for name, t in (("ks", k), ("vs", v)):
        store = torch.full((total, kv * dim), math.nan, device="cuda")
        for s, m in zip(starts, ages):
            store[s:s + m - 1] = t[s:s + m - 1]
        torch.cuda.synchronize()
        executor.write_tensor(name, store.cpu().numpy())
    executor.adopt("seqs", kernels.sequences([1, 1, 1], ages, starts))
    offsets = [0, 1, 2, 600, 601, 1499, 1500]
    q = randn((len(offsets), 3, heads * dim), "f32", 97)
    torch.cuda.synchronize()
    for name, w in (("q", heads), ("kn", kv), ("vn", kv)):
        executor.write_zeroed_tensor(name, (3, w * dim))
    nodes = [inv("kv-write-packed", ["ks", "kn", "seqs"], "ks"), inv("kv-write-packed", ["vs", "vn", "seqs"], "vs"),
             inv("attention-packed", ["q", "ks", "vs", "seqs"], "out",
                 {"head_count": heads, "head_dimension": dim, "kv_head_count": kv, "causal": True})]
    for n in nodes:
        executor.run(n)
    executor.begin_step_capture(["key_count"])
    for n in nodes:
        executor.run(n)
    executor.end_step_capture()
    out, last = np.empty((3, heads * dim), np.float32), -1
    for i, offset in enumerate(offsets):
        for o in range(last + 1, offset + 1):  # every token is written, those at `offsets` are looked at
            rows = [s + m - 1 + o for s, m in zip(starts, ages)]
            executor.replay_step_io({"q": q[i].cpu().numpy(), "kn": k[rows].cpu().numpy(), "vn": v[rows].cpu().numpy()}, {"out": out}, offset=o)
        last = offset
        want = attention64(q[i], k, v, heads, kv, [1] * 3, [m + offset for m in ages], starts)
        assert rel(torch.from_numpy(out).cuda(), want) <= ATTENTION_TOL["f32"], offset
