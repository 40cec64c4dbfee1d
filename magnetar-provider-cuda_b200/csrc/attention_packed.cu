// Attention of packed sequences: softmax(Q K^T * scale) V, each sequence over its own keys, with
// causal / sliding-window masks and grouped heads.
//
// Query j of a sequence with n queries and m keys stands at position m - n + j; causal admits the
// keys up to and with that position, a window of w the last w of those.  A query that sees no key
// gives zeros.
#include <algorithm>

#include "sequences.cuh"

namespace mg {
namespace {

// Keys [lo, hi) of its sequence that the query at `pos` sees (pos < 0: a query in front of all keys).
__device__ __forceinline__ void key_range(int causal, int64_t window, int64_t pos, int64_t keys, int64_t& lo, int64_t& hi) {
    hi = causal ? min(pos + 1, keys) : keys;
    hi = max(hi, (int64_t)0);
    lo = window >= 0 ? max(pos - window + 1, (int64_t)0) : 0;
    lo = min(lo, hi);
}

// One row's values of a key/value tensor, by dimension, in f32.
template <typename T>
struct PlainRows {
    const T* base;
    uint64_t ld;
    __device__ __forceinline__ float at(uint64_t row, uint32_t col) const { return to_f32(base[row * ld + col]); }
};
struct Q4Rows {
    const uint8_t* base;
    uint64_t columns;
    __device__ __forceinline__ float at(uint64_t row, uint32_t col) const {
        const uint8_t* rec = base + (row / kQ4Tile * columns + col / kQ4Block) * kQ4Record;
        const uint32_t r = (uint32_t)(row % kQ4Tile), c = col % kQ4Block;
        const int q = (int)((rec[r * 32 + c / 2] >> (4 * (c & 1))) & 15) - 8;
        const uint32_t slot = (r & ~15u) | ((r & 3u) << 2) | ((r >> 2) & 3u);
        return (float)q * __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rec + kQ4Quants)[slot]);
    }
};

// Any dimensions up to 512, any alignment: one warp per (query, head), lanes over the dimensions,
// keys one at a time.  The output is kept as a weighted mean of V rows (each key moves it by
// its weight over the sum so far), so it never exceeds the largest |v|.
constexpr int kRowThreads = 256;
constexpr int kPerLane = (int)(k::kPackedMaxDim / 32);

template <typename T, typename R>
__global__ void __launch_bounds__(kRowThreads) attention_packed_row_kernel(const k::PackedAttentionArgs a, R kr, R vr) {
    pdl_enter();
    const uint64_t warp = (uint64_t)blockIdx.x * (kRowThreads / 32) + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (warp >= a.queries * a.head_count) return;
    const uint64_t row = warp / a.head_count, head = warp % a.head_count;
    const uint64_t kvh = head / (a.head_count / a.kv_head_count);
    const SeqRow s = seq_load(a.table, seq_of_query(a.table, (uint32_t)row));
    int64_t lo, hi;
    key_range(a.causal, a.window, (int64_t)s.k_count - s.q_count + (int64_t)(row - s.q_start), s.k_count, lo, hi);
    const T* q = (const T*)a.q + (row * a.head_count + head) * a.head_dim;
    float qv[kPerLane], o[kPerLane];
#pragma unroll
    for (int i = 0; i < kPerLane; i++) {
        qv[i] = lane + 32 * i < (int)a.head_dim ? to_f32(q[lane + 32 * i]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = __int_as_float(0xff800000), l = 0.0f;
    for (int64_t key = lo; key < hi; key++) {
        const uint64_t krow = s.k_start + (uint64_t)key;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kPerLane; i++)
            if (lane + 32 * i < (int)a.head_dim) dot = fmaf(qv[i], kr.at(krow, (uint32_t)(kvh * a.head_dim) + lane + 32 * i), dot);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        const float m_new = fmaxf(m, dot);
        const float alpha = m == __int_as_float(0xff800000) ? 0.0f : expf(m - m_new);
        // (a NaN score passes through here, whatever the maximum made of it)
        const float e = dot == __int_as_float(0xff800000) ? 0.0f : expf(dot - m_new);
        const float l_new = l * alpha + e;
        const float keep = l > 0.0f ? l * alpha / l_new : 0.0f, w = l_new != 0.0f ? e / l_new : 0.0f;
#pragma unroll
        for (int i = 0; i < kPerLane; i++)
            if (lane + 32 * i < (int)a.value_dim)
                o[i] = fmaf(w, vr.at(krow, (uint32_t)(kvh * a.value_dim) + lane + 32 * i), o[i] * keep);
        m = m_new;
        l = l_new;
    }
    T* out = (T*)a.out + (row * a.head_count + head) * a.value_dim;
#pragma unroll
    for (int i = 0; i < kPerLane; i++)
        if (lane + 32 * i < (int)a.value_dim) out[lane + 32 * i] = from_f32<T>(o[i]);
}

mg_status attention_packed_rows(Device* d, const k::PackedAttentionArgs& a) {
    const uint64_t blocks = (a.queries * a.head_count + kRowThreads / 32 - 1) / (kRowThreads / 32);
    if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        const uint64_t kw = a.kv_head_count * a.head_dim, vw = a.kv_head_count * a.value_dim;
        if (a.kv_dtype == MG_Q4) {
            const Q4Rows kr{(const uint8_t*)a.k, kw / kQ4Block}, vr{(const uint8_t*)a.v, vw / kQ4Block};
            enqueue(d, attention_packed_row_kernel<T, Q4Rows>, (unsigned)blocks, kRowThreads, 0, a, kr, vr);
        } else {
            const PlainRows<T> kr{(const T*)a.k, kw}, vr{(const T*)a.v, vw};
            enqueue(d, attention_packed_row_kernel<T, PlainRows<T>>, (unsigned)blocks, kRowThreads, 0, a, kr, vr);
        }
        return launched(d, "packed attention launch");
    });
}

}  // namespace

namespace k {

mg_status attention_packed(Device* d, const PackedAttentionArgs& a) {
    if (a.queries == 0) return MG_OK;
    return attention_packed_rows(d, a);
}

}  // namespace k
}  // namespace mg
