// What the kernels of packed attention share: the masks, the readers of keys and values, and one
// query row computed by one warp.
#pragma once

#include "sequences.cuh"

namespace mg {

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
        return (float)q * __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot(r)]);
    }
};

// One (query row, head) by one warp, lanes over the dimensions (at most 32 * N), keys one at a time.
// The output is kept as a weighted mean of V rows (each key moves it by its weight over the sum so
// far), so it never exceeds the largest |v|.
template <typename T, typename R, int N>
__device__ __forceinline__ void attention_row(const k::PackedAttentionArgs& a, const R& kr, const R& vr, const SeqRow& s,
                                              uint64_t row, uint64_t head, int lane) {
    const uint64_t kvh = head / (a.head_count / a.kv_head_count);
    int64_t lo, hi;
    key_range(a.causal, a.window, (int64_t)s.k_count - s.q_count + (int64_t)(row - s.q_start), s.k_count, lo, hi);
    const T* q = (const T*)a.q + (row * a.head_count + head) * a.head_dim;
    float qv[N], o[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        qv[i] = lane + 32 * i < (int)a.head_dim ? to_f32(q[lane + 32 * i]) * a.scale : 0.0f;
        o[i] = 0.0f;
    }
    float m = __int_as_float(0xff800000), l = 0.0f;
    for (int64_t key = lo; key < hi; key++) {
        const uint64_t krow = s.k_start + (uint64_t)key;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++)
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
        for (int i = 0; i < N; i++)
            if (lane + 32 * i < (int)a.value_dim)
                o[i] = fmaf(w, vr.at(krow, (uint32_t)(kvh * a.value_dim) + lane + 32 * i), o[i] * keep);
        m = m_new;
        l = l_new;
    }
    T* out = (T*)a.out + (row * a.head_count + head) * a.value_dim;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane + 32 * i < (int)a.value_dim) out[lane + 32 * i] = from_f32<T>(o[i]);
}

}  // namespace mg
