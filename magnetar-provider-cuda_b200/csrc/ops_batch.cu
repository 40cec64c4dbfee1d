// C ABI of the operators for batches of packed sequences: the table of sequences, 4-bit key/value
// stores, packed kv-write / kv-read, attention of packed sequences, rope with several axes, and
// token log probabilities.  Each entry validates its operands on the host (shape errors ->
// ShapeUnsupported, types -> DTypeUnsupported), picks the output by the output-offer rule and
// enqueues its kernels; none of them waits for the device.  The reference serves one sequence per
// call and has no counterpart of these entries.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <new>
#include <numeric>

#include "internal.h"

using namespace mg;

namespace {

using ull = unsigned long long;

mg_status need(Device* d, const mg_buffer* b, const char* what) {
    if (!b) return fail(MG_INVALID_ARGUMENT, "null %s buffer", what);
    if (buf(b)->device != d) return fail(MG_INVALID_ARGUMENT, "buffer belongs to another device");
    return MG_OK;
}

mg_status need_rows(const Buffer* b, const char* what, uint64_t* rows, uint64_t* cols) {
    if (b->rank != 2) return fail(MG_SHAPE_UNSUPPORTED, "%s must have rank 2, got shape %s", what, shape_str(b).c_str());
    *rows = b->shape[0];
    *cols = b->shape[1];
    return MG_OK;
}

mg_status need_float(const Buffer* b, const char* what) {
    if (!is_float(b->dtype)) return fail(MG_DTYPE_UNSUPPORTED, "%s cannot be %s", what, dtype_name(b->dtype));
    return MG_OK;
}

// An offered output (or a store that is written) that shares memory with something the call reads: blocks of the
// launch would read what others have already written.
mg_status need_apart(const Buffer* written, std::initializer_list<const Buffer*> read) {
    auto bytes = [](const Buffer* b) { return b->dtype == MG_Q4 ? q4_bytes(b->shape[0], b->shape[1]) : b->count * dtype_size(b->dtype); };
    const uint8_t* w = (const uint8_t*)written->ptr;
    for (const Buffer* b : read) {
        if (!b || !bytes(b)) continue;
        const uint8_t* r = (const uint8_t*)b->ptr;
        if (w < r + bytes(b) && r < w + bytes(written))
            return fail(MG_INVALID_ARGUMENT, "the memory that is written (%s) overlaps an input (%s)", shape_str(written).c_str(),
                        shape_str(b).c_str());
    }
    return MG_OK;
}

mg_status need_table(Device* d, const mg_buffer* s, const SequenceTable** host, k::SeqTable* table) {
    MG_TRY(need(d, s, "sequences"));
    const Buffer* b = buf(s);
    if (b->dtype != MG_SEQUENCES || !b->seq)
        return fail(MG_DTYPE_UNSUPPORTED, "%s is not a table of sequences", dtype_name(b->dtype));
    *host = b->seq;
    table->rows = (const SeqRow*)b->ptr;
    table->count = (uint32_t)b->seq->rows.size();
    table->ordered = table->rows + table->count;
    table->order = (const uint32_t*)(table->ordered + table->count);
    table->key_prefix = table->order + table->count;
    table->step = nullptr;
    return MG_OK;
}

// The host side of a table, or the reason there is none.
mg_status make_table(uint64_t count, const uint64_t* query_counts, const uint64_t* key_counts, const uint64_t* key_starts,
                     SequenceTable* t) {
    constexpr uint64_t kLimit = 1ull << 31;
    if (count == 0 || count >= (1u << 24)) return fail(MG_SHAPE_UNSUPPORTED, "a table cannot hold %llu sequences", (ull)count);
    t->rows.resize(count);
    for (uint64_t i = 0; i < count; i++) {
        const uint64_t n = query_counts[i], m = key_counts ? key_counts[i] : n;
        if (n >= kLimit || m >= kLimit) return fail(MG_SHAPE_UNSUPPORTED, "sequence %llu has 2^31 rows or more", (ull)i);
        const uint64_t at = key_starts ? key_starts[i] : t->keys;
        if (t->queries + n >= kLimit || at >= kLimit || at + m >= kLimit)
            return fail(MG_SHAPE_UNSUPPORTED, "the rows of sequence %llu do not lie below 2^31", (ull)i);
        t->rows[i] = {(uint32_t)t->queries, (uint32_t)n, (uint32_t)at, (uint32_t)m};
        t->queries += n;
        t->keys += m;
        t->key_end = std::max(t->key_end, at + m);
        t->max_queries = std::max(t->max_queries, n);
        if (m < n) t->writable = false;
    }
    // What each sequence with queries may grow by: up to the first row another one starts at, at or past its end
    // (a sequence without queries is neither read nor written).
    std::vector<std::pair<uint32_t, uint32_t>> spans, written;  // [start, end) of all keys, by their starts; of the written rows
    spans.reserve(count);
    written.reserve(count);
    for (const SeqRow& r : t->rows) {
        const uint32_t end = r.k_start + r.k_count;
        if (r.k_count) spans.emplace_back(r.k_start, end);
        if (r.q_count && r.q_count <= r.k_count) written.emplace_back(end - r.q_count, end);
    }
    std::sort(spans.begin(), spans.end());
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); i++) t->shared_rows = t->shared_rows || written[i].first < written[i - 1].second;
    std::vector<uint32_t> farthest(spans.size());  // end of the spans up to each
    for (size_t i = 0; i < spans.size(); i++) farthest[i] = std::max(spans[i].second, i ? farthest[i - 1] : 0u);
    for (const SeqRow& r : t->rows) {
        if (!r.q_count) continue;
        const uint32_t end = r.k_start + r.k_count;
        const size_t i = std::lower_bound(spans.begin(), spans.end(), std::make_pair(end, 0u)) - spans.begin();
        if (i < spans.size()) t->slack = std::min<uint64_t>(t->slack, spans[i].first - end);
        if (i && farthest[i - 1] > end) t->write_slack = 0;
    }
    t->write_slack = std::min(t->write_slack, t->slack);
    return MG_OK;
}

mg_status upload_table(Device* d, Buffer* b) {
    const SequenceTable& t = *b->seq;
    const size_t n = t.rows.size();
    std::vector<uint32_t> words(n * kSeqBytes / sizeof(uint32_t));
    memcpy(words.data(), t.rows.data(), n * sizeof(SeqRow));
    uint32_t* order = words.data() + 8 * n;
    std::iota(order, order + n, 0u);
    std::stable_sort(order, order + n, [&](uint32_t x, uint32_t y) { return t.rows[x].k_count > t.rows[y].k_count; });
    uint32_t keys = 0;
    for (size_t i = 0; i < n; i++) {
        memcpy(words.data() + 4 * (n + i), &t.rows[order[i]], sizeof(SeqRow));
        order[n + i] = keys;
        keys += t.rows[i].k_count;
    }
    // pageable memory: the copy has read it when the call returns
    MG_CUDA(cudaMemcpyAsync(b->ptr, words.data(), words.size() * 4, cudaMemcpyHostToDevice, d->stream), "uploading a table");
    d->uploads.fetch_add(1);
    return MG_OK;
}

// Host allocation failures must not cross the C ABI.
template <class F>
mg_status guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(MG_EXECUTION_FAILED, "host allocation failed");
    }
}

}  // namespace

namespace mg {

mg_status kv_write_q4_plan(mg_device* h, mg_buffer* sh, const mg_buffer* rh, uint64_t row_offset, k::KvPackedArgs* a,
                           uint64_t* headroom) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, sh, "store"));
    MG_TRY(need(d, rh, "rows"));
    const Buffer *store = buf(sh), *rows = buf(rh);
    MG_TRY(need_float(rows, "kv-write's rows"));
    uint64_t count, width;
    MG_TRY(need_rows(rows, "kv-write's rows", &count, &width));
    const uint64_t capacity = store->shape[0];
    if (width != store->shape[1])
        return fail(MG_SHAPE_UNSUPPORTED, "kv-write rows have width %llu, the store %llu", (ull)width, (ull)store->shape[1]);
    if (row_offset > capacity || count > capacity - row_offset)
        return fail(MG_SHAPE_UNSUPPORTED, "kv-write of %llu rows at %llu exceeds the store's %llu rows", (ull)count,
                    (ull)row_offset, (ull)capacity);
    *headroom = capacity - row_offset - count;
    a->rows = rows->ptr;
    a->dtype = rows->dtype;
    a->store = store->ptr;
    a->store_dtype = MG_Q4;
    a->queries = count;
    a->width = width;
    a->table = {};
    a->row_offset = row_offset;
    return MG_OK;
}

mg_status kv_write_packed_plan(mg_device* h, mg_buffer* sh, const mg_buffer* rh, const mg_buffer* seqs, k::KvPackedArgs* a,
                               uint64_t* headroom) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, sh, "store"));
    MG_TRY(need(d, rh, "rows"));
    const Buffer *store = buf(sh), *rows = buf(rh);
    MG_TRY(need_float(rows, "kv-write's rows"));
    if (store->dtype != MG_Q4 && store->dtype != rows->dtype)
        return fail(MG_DTYPE_UNSUPPORTED, "kv-write cannot put %s rows into a %s store", dtype_name(rows->dtype),
                    dtype_name(store->dtype));
    const SequenceTable* t;
    MG_TRY(need_table(d, seqs, &t, &a->table));
    uint64_t capacity, store_width, count, width;
    MG_TRY(need_rows(store, "the store", &capacity, &store_width));
    MG_TRY(need_rows(rows, "kv-write's rows", &count, &width));
    if (width != store_width)
        return fail(MG_SHAPE_UNSUPPORTED, "kv-write rows have width %llu, the store %llu", (ull)width, (ull)store_width);
    if (count != t->queries)
        return fail(MG_SHAPE_UNSUPPORTED, "the sequences have %llu rows, got %llu", (ull)t->queries, (ull)count);
    if (!t->writable) return fail(MG_SHAPE_UNSUPPORTED, "a sequence has fewer keys than rows to write");
    if (t->shared_rows) return fail(MG_SHAPE_UNSUPPORTED, "two sequences would write the same rows of the store");
    if (t->key_end > capacity)
        return fail(MG_SHAPE_UNSUPPORTED, "the sequences' keys end at row %llu of the store's %llu", (ull)t->key_end,
                    (ull)capacity);
    MG_TRY(need_apart(store, {rows}));
    *headroom = std::min(t->write_slack, capacity - t->key_end);
    a->rows = rows->ptr;
    a->dtype = rows->dtype;
    a->store = store->ptr;
    a->store_dtype = store->dtype;
    a->queries = count;
    a->width = width;
    a->row_offset = 0;
    return MG_OK;
}

mg_status kv_read_packed_plan(mg_device* h, const mg_buffer* sh, const mg_buffer* seqs, mg_buffer** out, k::KvPackedArgs* a,
                              float** values, uint64_t* headroom) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, sh, "store"));
    const Buffer* store = buf(sh);
    if (store->dtype != MG_Q4) return fail(MG_DTYPE_UNSUPPORTED, "kv-read reads 4-bit stores, got %s", dtype_name(store->dtype));
    const SequenceTable* t;
    MG_TRY(need_table(d, seqs, &t, &a->table));
    if (!t->writable) return fail(MG_SHAPE_UNSUPPORTED, "a sequence has fewer keys than rows to read");
    if (t->key_end > store->shape[0])
        return fail(MG_SHAPE_UNSUPPORTED, "the sequences' keys end at row %llu of the store's %llu", (ull)t->key_end,
                    (ull)store->shape[0]);
    *headroom = std::min(t->slack, store->shape[0] - t->key_end);
    const uint64_t shape[2] = {t->queries, store->shape[1]};
    Buffer* o;
    MG_TRY(output_for(d, MG_F32, 2, shape, out, &o));
    a->rows = nullptr;
    a->dtype = MG_F32;
    a->store = store->ptr;
    a->store_dtype = MG_Q4;
    a->queries = t->queries;
    a->width = store->shape[1];
    a->row_offset = 0;
    *values = (float*)o->ptr;
    return MG_OK;
}

mg_status attention_packed_plan(mg_device* h, const mg_buffer* qh, const mg_buffer* kh, const mg_buffer* vh,
                                const mg_buffer* seqs, const mg_attention_params* pp, mg_buffer** out,
                                k::PackedAttentionArgs* a, uint64_t* headroom) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, qh, "q"));
    MG_TRY(need(d, kh, "k"));
    MG_TRY(need(d, vh, "v"));
    if (!pp) return fail(MG_INVALID_ARGUMENT, "null attention parameters");
    const mg_attention_params& p = *pp;
    const Buffer *q = buf(qh), *kb = buf(kh), *v = buf(vh);
    MG_TRY(need_float(q, "attention's q"));
    if (kb->dtype != v->dtype || (kb->dtype != q->dtype && kb->dtype != MG_Q4))
        return fail(MG_DTYPE_UNSUPPORTED, "attention cannot read %s keys and %s values with %s queries", dtype_name(kb->dtype),
                    dtype_name(v->dtype), dtype_name(q->dtype));
    const SequenceTable* t;
    MG_TRY(need_table(d, seqs, &t, &a->table));
    const uint64_t heads = p.head_count, dim = p.head_dimension, kv = p.kv_head_count ? p.kv_head_count : heads;
    const uint64_t vdim = p.value_dimension ? p.value_dimension : dim;
    if (heads == 0 || dim == 0)
        return fail(MG_SHAPE_UNSUPPORTED, "head_count, kv_head_count, and head_dimension must all be positive");
    if (heads % kv != 0)
        return fail(MG_SHAPE_UNSUPPORTED, "head_count %llu must be an exact multiple of kv_head_count %llu", (ull)heads, (ull)kv);
    if (heads > 65535) return fail(MG_SHAPE_UNSUPPORTED, "attention head_count exceeds the launch grid");
    if (dim > k::kPackedMaxDim || vdim > k::kPackedMaxDim)
        return fail(MG_SHAPE_UNSUPPORTED, "packed attention's dimensions are at most %llu, got %llu and %llu",
                    (ull)k::kPackedMaxDim, (ull)dim, (ull)vdim);
    if (p.key_count >= 0) return fail(MG_SHAPE_UNSUPPORTED, "packed attention takes its key counts from the sequences");
    if (p.window_size == 0) return fail(MG_SHAPE_UNSUPPORTED, "window_size must be positive; a zero window admits no keys");
    if (p.window_size > 0 && !p.causal) return fail(MG_SHAPE_UNSUPPORTED, "window_size is only defined for causal attention");
    if (p.has_scale && (!std::isfinite(p.scale) || !(p.scale > 0.0f)))
        return fail(MG_SHAPE_UNSUPPORTED, "attention scale %g must be finite and positive", (double)p.scale);
    uint64_t q_rows, q_width, k_rows, k_width, v_rows, v_width;
    MG_TRY(need_rows(q, "q", &q_rows, &q_width));
    MG_TRY(need_rows(kb, "k", &k_rows, &k_width));
    MG_TRY(need_rows(v, "v", &v_rows, &v_width));
    if (q_rows != t->queries)
        return fail(MG_SHAPE_UNSUPPORTED, "the sequences have %llu queries, q %llu rows", (ull)t->queries, (ull)q_rows);
    if (q_width != heads * dim)
        return fail(MG_SHAPE_UNSUPPORTED, "head_count * head_dimension must equal q row width %llu, got %llu * %llu", (ull)q_width,
                    (ull)heads, (ull)dim);
    if (k_width != kv * dim)
        return fail(MG_SHAPE_UNSUPPORTED, "kv_head_count * head_dimension must equal k row width %llu, got %llu * %llu",
                    (ull)k_width, (ull)kv, (ull)dim);
    if (v_rows != k_rows || v_width != kv * vdim)
        return fail(MG_SHAPE_UNSUPPORTED, "v must hold %llu rows of kv_head_count * value_dimension = %llu * %llu, got %s",
                    (ull)k_rows, (ull)kv, (ull)vdim, shape_str(v).c_str());
    if (kb->dtype == MG_Q4 && (dim % kQ4Block != 0 || vdim != dim))
        return fail(MG_SHAPE_UNSUPPORTED, "attention over 4-bit stores needs a head dimension that is a multiple of 64, and as "
                    "wide values; got %llu and %llu", (ull)dim, (ull)vdim);
    if (t->key_end > k_rows)
        return fail(MG_SHAPE_UNSUPPORTED, "the sequences' keys end at row %llu of k's %llu", (ull)t->key_end, (ull)k_rows);
    *headroom = std::min(t->slack, k_rows - t->key_end);
    const uint64_t shape[2] = {q_rows, heads * vdim};
    Buffer* o;
    MG_TRY(output_for(d, q->dtype, 2, shape, out, &o));
    MG_TRY(need_apart(o, {q, kb, v}));
    a->q = q->ptr;
    a->k = kb->ptr;
    a->v = v->ptr;
    a->out = o->ptr;
    a->dtype = q->dtype;
    a->kv_dtype = kb->dtype;
    a->queries = q_rows;
    a->kv_rows = k_rows;
    a->head_count = heads;
    a->kv_head_count = kv;
    a->head_dim = dim;
    a->value_dim = vdim;
    a->causal = p.causal ? 1 : 0;
    a->window = p.window_size > 0 ? p.window_size : -1;
    a->scale = p.has_scale ? p.scale : 1.0f / sqrtf((float)dim);
    a->host = t;
    a->max_step = 0;
    return MG_OK;
}

}  // namespace mg

extern "C" {

mg_status mg_sequences_create(mg_device* h, uint64_t count, const uint64_t* query_counts, const uint64_t* key_counts,
                              const uint64_t* key_starts, mg_buffer** out) {
    MG_TRY(device_check(h));
    if (!out || !query_counts) return fail(MG_INVALID_ARGUMENT, "null argument");
    *out = nullptr;
    Device* d = dev(h);
    if (d->capturing) return fail(MG_CAPTURE_UNSUPPORTED, "a host-to-device upload cannot be captured");
    return guarded([&]() -> mg_status {
        SequenceTable t;
        MG_TRY(make_table(count, query_counts, key_counts, key_starts, &t));
        const uint64_t shape[2] = {count, 4};
        Buffer* b = nullptr;
        MG_TRY(buffer_new_opaque(d, MG_SEQUENCES, 2, shape, count * kSeqBytes, &b));
        mg_status s = MG_EXECUTION_FAILED;
        try {
            b->seq = new SequenceTable(std::move(t));
            s = upload_table(d, b);
        } catch (const std::bad_alloc&) {
            s = fail(MG_EXECUTION_FAILED, "host allocation failed");
        }
        if (s != MG_OK) {
            buffer_free(b);
            return s;
        }
        *out = reinterpret_cast<mg_buffer*>(b);
        return MG_OK;
    });
}

mg_status mg_sequences_write(mg_buffer* h, uint64_t count, const uint64_t* query_counts, const uint64_t* key_counts,
                             const uint64_t* key_starts) {
    if (!h || !query_counts) return fail(MG_INVALID_ARGUMENT, "null argument");
    Buffer* b = buf(h);
    if (b->dtype != MG_SEQUENCES || !b->seq) return fail(MG_DTYPE_UNSUPPORTED, "%s is not a table of sequences", dtype_name(b->dtype));
    if (count != b->seq->rows.size())
        return fail(MG_SHAPE_UNSUPPORTED, "the table holds %llu sequences, not %llu", (ull)b->seq->rows.size(), (ull)count);
    Device* d = b->device;
    if (d->capturing) return fail(MG_CAPTURE_UNSUPPORTED, "a host-to-device upload cannot be captured");
    {
        std::lock_guard<std::mutex> g(d->mem_lock);
        if (d->graph_refs.count(b->ptr)) return fail(MG_CAPTURE_UNSUPPORTED, "a captured step reads this table");
    }
    MG_CUDA(cudaSetDevice(d->ordinal), "selecting the device");
    return guarded([&]() -> mg_status {
        SequenceTable t;
        MG_TRY(make_table(count, query_counts, key_counts, key_starts, &t));
        std::swap(*b->seq, t);
        mg_status s = MG_EXECUTION_FAILED;
        try {
            s = upload_table(d, b);
        } catch (const std::bad_alloc&) {
            s = fail(MG_EXECUTION_FAILED, "host allocation failed");
        }
        if (s != MG_OK) std::swap(*b->seq, t);  // the device still holds the old rows
        return s;
    });
}

mg_status mg_kv_store_q4(mg_device* h, uint64_t rows, uint64_t head_count, uint64_t head_dimension, mg_buffer** out) {
    MG_TRY(device_check(h));
    if (!out) return fail(MG_INVALID_ARGUMENT, "null output parameter");
    *out = nullptr;
    if (rows == 0 || rows >= (1ull << 31) || head_count == 0 || head_dimension == 0 || head_dimension % kQ4Block != 0 ||
        head_dimension > 65536 || head_count > 65535)
        return fail(MG_SHAPE_UNSUPPORTED,
                    "a 4-bit store needs 1 to 2^31 - 1 rows and heads of a multiple of 64 values, got %llu rows of %llu * %llu",
                    (ull)rows, (ull)head_count, (ull)head_dimension);
    const uint64_t shape[2] = {rows, head_count * head_dimension};
    const uint64_t bytes = q4_bytes(rows, shape[1]);
    Buffer* b = nullptr;
    MG_TRY(buffer_new_opaque(dev(h), MG_Q4, 2, shape, bytes, &b));
    // zero scales: every row reads as zeros until it is written
    mg_status s = k::fill_zero(dev(h), b->ptr, bytes);
    if (s != MG_OK) {
        buffer_free(b);
        return s;
    }
    *out = reinterpret_cast<mg_buffer*>(b);
    return MG_OK;
}

mg_status mg_kv_write_packed(mg_device* h, mg_buffer* store, const mg_buffer* rows, const mg_buffer* sequences) {
    k::KvPackedArgs a;
    uint64_t headroom;
    MG_TRY(kv_write_packed_plan(h, store, rows, sequences, &a, &headroom));
    if (buf(store)->dtype != MG_Q4) buffer_drop_prep(buf(store));  // its contents change
    return k::kv_write_packed(dev(h), a);
}

mg_status mg_kv_read_packed(mg_device* h, const mg_buffer* store, const mg_buffer* sequences, mg_buffer** out) {
    k::KvPackedArgs a;
    float* values;
    uint64_t headroom;
    MG_TRY(kv_read_packed_plan(h, store, sequences, out, &a, &values, &headroom));
    return k::kv_read_packed(dev(h), a, values);
}

mg_status mg_attention_packed(mg_device* h, const mg_buffer* q, const mg_buffer* k, const mg_buffer* v,
                              const mg_buffer* sequences, const mg_attention_params* params, mg_buffer** out) {
    k::PackedAttentionArgs a;
    uint64_t headroom;
    MG_TRY(attention_packed_plan(h, q, k, v, sequences, params, out, &a, &headroom));
    return k::attention_packed(dev(h), a);
}

mg_status mg_rope_axes(mg_device* h, const mg_buffer* xh, const mg_buffer* ph, const mg_rope_axes_params* pp, mg_buffer** out) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, xh, "input"));
    MG_TRY(need(d, ph, "positions"));
    if (!pp) return fail(MG_INVALID_ARGUMENT, "null rope parameters");
    const mg_rope_axes_params& p = *pp;
    const Buffer *x = buf(xh), *pos = buf(ph);
    MG_TRY(need_float(x, "rope's input"));
    if (pos->dtype != MG_F32) return fail(MG_DTYPE_UNSUPPORTED, "rope's positions cannot be %s", dtype_name(pos->dtype));
    uint64_t rows, cols, pos_rows, pos_cols;
    MG_TRY(need_rows(x, "rope's input", &rows, &cols));
    MG_TRY(need_rows(pos, "rope's positions", &pos_rows, &pos_cols));
    if (p.axes < 1 || p.axes > MG_ROPE_MAX_AXES)
        return fail(MG_SHAPE_UNSUPPORTED, "RoPE takes 1 to %d axes, got %d", MG_ROPE_MAX_AXES, p.axes);
    if (pos_rows != rows || pos_cols != (uint64_t)p.axes)
        return fail(MG_SHAPE_UNSUPPORTED, "RoPE positions must be [%llu, %d], got %s", (ull)rows, p.axes, shape_str(pos).c_str());
    if (p.head_count == 0 || cols % p.head_count != 0)
        return fail(MG_SHAPE_UNSUPPORTED, "RoPE head_count %llu must be positive and evenly divide the row width %llu",
                    (ull)p.head_count, (ull)cols);
    const uint64_t head_width = cols / p.head_count, half = p.dimension / 2;
    if (p.dimension == 0 || p.dimension % 2 != 0 || p.dimension > head_width)
        return fail(MG_SHAPE_UNSUPPORTED, "RoPE dimension %llu must be positive, even, and at most the head width %llu",
                    (ull)p.dimension, (ull)head_width);
    if (half > k::kRopeAxesMaxPairs)
        return fail(MG_SHAPE_UNSUPPORTED, "RoPE with several axes rotates at most %llu pairs, got %llu", (ull)k::kRopeAxesMaxPairs,
                    (ull)half);
    if (!std::isfinite(p.base) || p.base <= 0.0f) return fail(MG_SHAPE_UNSUPPORTED, "RoPE base must be finite and positive");
    if (!std::isfinite(p.scale) || p.scale <= 0.0f) return fail(MG_SHAPE_UNSUPPORTED, "RoPE scale must be finite and positive");
    if (p.pairing != 0 && p.pairing != 1) return fail(MG_SHAPE_UNSUPPORTED, "RoPE pairing %d is not implemented", p.pairing);
    if (p.order != 0 && p.order != 1) return fail(MG_SHAPE_UNSUPPORTED, "RoPE section order %d is not implemented", p.order);
    if (p.ladder != 0 && p.ladder != 1) return fail(MG_SHAPE_UNSUPPORTED, "RoPE frequency ladder %d is not implemented", p.ladder);
    uint64_t sum = 0;
    for (int i = 0; i < p.axes; i++) {
        if (p.sections[i] > half) return fail(MG_SHAPE_UNSUPPORTED, "RoPE section %d is larger than the %llu pairs", i, (ull)half);
        sum += p.sections[i];
    }
    if (sum != half) return fail(MG_SHAPE_UNSUPPORTED, "RoPE sections hold %llu pairs, the dimension %llu", (ull)sum, (ull)half);
    return guarded([&]() -> mg_status {
        k::RopeAxesArgs a;
        a.axis.resize(half);
        a.frequency.resize(half);
        uint64_t seen[MG_ROPE_MAX_AXES] = {0};
        uint64_t at = 0, left = p.sections[0];
        for (uint64_t i = 0; i < half; i++) {
            int axis = 0;
            if (p.order == 0) {
                while (left == 0) left = p.sections[++at];
                left--;
                axis = (int)at;
            } else {
                const int turn = (int)(i % (uint64_t)p.axes);
                if (turn != 0 && i / (uint64_t)p.axes < p.sections[turn]) axis = turn;
            }
            const double exponent = p.ladder == 0 ? (double)i / (double)half : (double)seen[axis] / (double)p.sections[axis];
            a.axis[i] = (uint8_t)axis;
            a.frequency[i] = (float)std::pow((double)p.base, -exponent);
            seen[axis]++;
        }
        for (int i = 0; i < p.axes; i++)
            if (seen[i] != p.sections[i])
                return fail(MG_SHAPE_UNSUPPORTED, "dealing the %llu pairs out in turn cannot give axis %d %llu of them", (ull)half, i,
                            (ull)p.sections[i]);
        Buffer* o;
        MG_TRY(output_for(d, x->dtype, 2, x->shape, out, &o));
        MG_TRY(need_apart(o, {o->ptr == x->ptr ? nullptr : x, pos}));
        a.x = x->ptr;
        a.out = o->ptr;
        a.positions = (const float*)pos->ptr;
        a.dtype = x->dtype;
        a.rows = rows;
        a.head_count = p.head_count;
        a.head_width = head_width;
        a.half = half;
        a.scale = p.scale;
        a.axes = p.axes;
        a.half_split = p.pairing;
        a.inverse = p.inverse ? 1 : 0;
        return k::rope_axes(d, a);
    });
}

mg_status mg_token_logprobs(mg_device* h, const mg_buffer* lh, const mg_buffer* th, uint32_t top, float temperature,
                            mg_buffer** out) {
    MG_TRY(device_check(h));
    Device* d = dev(h);
    MG_TRY(need(d, lh, "logits"));
    const Buffer *l = buf(lh), *t = nullptr;
    MG_TRY(need_float(l, "logits"));
    uint64_t rows, vocab;
    MG_TRY(need_rows(l, "logits", &rows, &vocab));
    if (vocab == 0 || vocab > (1u << 24))  // a column is returned as f32, exact up to 2^24
        return fail(MG_SHAPE_UNSUPPORTED, "logits need 1 to 2^24 columns, got %llu", (ull)vocab);
    if (top > MG_LOGPROBS_MAX_TOP || top > vocab)
        return fail(MG_SHAPE_UNSUPPORTED, "%u top columns exceed %d or the %llu columns", top, MG_LOGPROBS_MAX_TOP, (ull)vocab);
    if (!std::isfinite(temperature) || !(temperature > 0.0f))
        return fail(MG_SHAPE_UNSUPPORTED, "temperature %g must be finite and positive", (double)temperature);
    if (temperature < FLT_MIN) return fail(MG_SHAPE_UNSUPPORTED, "temperature %g has no reciprocal in f32", (double)temperature);
    if (th) {
        MG_TRY(need(d, th, "tokens"));
        t = buf(th);
        if (t->dtype != MG_F32) return fail(MG_DTYPE_UNSUPPORTED, "tokens cannot be %s", dtype_name(t->dtype));
        if (t->count != rows)
            return fail(MG_SHAPE_UNSUPPORTED, "%llu rows of logits need as many tokens, got %s", (ull)rows, shape_str(t).c_str());
    }
    const uint64_t shape[2] = {rows, 2 + 2 * (uint64_t)top};
    Buffer* o;
    MG_TRY(output_for(d, MG_F32, 2, shape, out, &o));
    MG_TRY(need_apart(o, {l, t}));
    k::LogprobsArgs a;
    a.logits = l->ptr;
    a.dtype = l->dtype;
    a.tokens = t ? (const float*)t->ptr : nullptr;
    a.out = (float*)o->ptr;
    a.rows = rows;
    a.vocab = vocab;
    a.top = top;
    a.temperature = temperature;
    return k::token_logprobs(d, a);
}

}  // extern "C"
