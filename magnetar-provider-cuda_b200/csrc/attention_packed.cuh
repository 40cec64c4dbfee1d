// What the kernels of packed attention share: the masks, the readers of keys and values, and one
// query row computed by one warp.
#pragma once

#include <type_traits>

#include "sequences.cuh"

namespace mg {

// Keys [lo, hi) of its sequence that the query at `pos` sees (pos < 0: a query in front of all keys).
__device__ __forceinline__ void key_range(int causal, int64_t window, int64_t pos, int64_t keys, int64_t& lo, int64_t& hi) {
    hi = causal ? min(pos + 1, keys) : keys;
    hi = max(hi, (int64_t)0);
    lo = window >= 0 ? max(pos - window + 1, (int64_t)0) : 0;
    lo = min(lo, hi);
}

// One row's values of a key/value tensor in f32: one, or eight from a column on (a multiple of 8 within a head).
template <typename T>
struct PlainRows {
    const T* base;
    uint64_t ld;
    bool vec;  // every head of every row starts on 16 bytes and has a multiple of 8 values
    __device__ __forceinline__ float at(uint64_t row, uint32_t col) const { return to_f32(base[row * ld + col]); }
    __device__ __forceinline__ void eight(uint64_t row, uint32_t col, float (&x)[8]) const {
        const T* src = base + row * ld + col;
        uint4 u[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) u[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = to_f32(reinterpret_cast<const T*>(u)[e]);
    }
};
struct Q4Rows {
    const uint8_t* base;
    uint64_t columns;
    static constexpr bool vec = true;
    __device__ __forceinline__ const uint8_t* record(uint64_t row, uint32_t col, float& scale) const {
        const uint8_t* rec = base + (row / kQ4Tile * columns + col / kQ4Block) * kQ4Record;
        scale = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot((uint32_t)(row % kQ4Tile))]);
        return rec + row % kQ4Tile * 32;
    }
    __device__ __forceinline__ float at(uint64_t row, uint32_t col) const {
        const uint32_t c = col % kQ4Block;
        float scale;
        const uint8_t* quants = record(row, col, scale);
        return (float)((int)((quants[c / 2] >> (4 * (c & 1))) & 15) - 8) * scale;
    }
    __device__ __forceinline__ void eight(uint64_t row, uint32_t col, float (&x)[8]) const {
        float scale;
        const uint8_t* quants = record(row, col, scale);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(quants + col % kQ4Block / 2);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)((int)((word >> (4 * e)) & 15u) - 8) * scale;
    }
};

// One (query row, head) by one warp: the keys from `first` on, 32 at a time, `step` apart.  A lane has a key for
// the scores (q in shared memory, read by all lanes alike) and up to N values of the output, lane, lane +
// 32, ..., for the weighted values, AHEAD keys' loads at a time.  The output is kept as a weighted mean of V rows (each tile moves it by
// its weight over the sum so far), so it never exceeds the largest |v|; m and l are the scores' maximum and sum.
template <typename T, typename R, int N, int AHEAD>
__device__ __forceinline__ void attention_keys(const k::PackedAttentionArgs& a, const R& kr, const R& vr, const SeqRow& s, uint64_t row,
                                               uint64_t head, int lane, float* q_shared, int64_t first, int64_t step, float (&o)[N],
                                               float& m, float& l) {
    const uint64_t kvh = head / (a.head_count / a.kv_head_count);
    const int dim = (int)a.head_dim, vdim = (int)a.value_dim;
    const uint32_t kcol = (uint32_t)kvh * (uint32_t)dim, vcol = (uint32_t)kvh * (uint32_t)vdim;
    const float kNegInf = __int_as_float(0xff800000);
    int64_t lo, hi;
    key_range(a.causal, a.window, (int64_t)s.k_count - s.q_count + (int64_t)(row - s.q_start), s.k_count, lo, hi);
    const T* q = (const T*)a.q + (row * a.head_count + head) * a.head_dim;
    __syncwarp();
    for (int i = lane; i < dim; i += 32) q_shared[i] = to_f32(q[i]) * a.scale;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = 0.0f;
    m = kNegInf;
    l = 0.0f;
    for (int64_t base = lo + first; base < hi; base += step) {
        const int keys = (int)min((int64_t)32, hi - base);
        const uint64_t row0 = s.k_start + (uint64_t)base, krow = row0 + (uint64_t)min(lane, keys - 1);
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (kr.vec) {
#pragma unroll(AHEAD > 1 ? 4 : 1)
            for (int c = 0; c < dim; c += 8) {
                float x[8];
                kr.eight(krow, kcol + c, x);
                const float4 u = *reinterpret_cast<const float4*>(q_shared + c), v = *reinterpret_cast<const float4*>(q_shared + c + 4);
                sums[0] = fmaf(u.x, x[0], fmaf(v.x, x[4], sums[0]));
                sums[1] = fmaf(u.y, x[1], fmaf(v.y, x[5], sums[1]));
                sums[2] = fmaf(u.z, x[2], fmaf(v.z, x[6], sums[2]));
                sums[3] = fmaf(u.w, x[3], fmaf(v.w, x[7], sums[3]));
            }
        } else {
#pragma unroll 8
            for (int c = 0; c < dim; c++) sums[0] = fmaf(q_shared[c], kr.at(krow, kcol + c), sums[0]);
        }
        const float dot = lane < keys ? (sums[0] + sums[1]) + (sums[2] + sums[3]) : kNegInf;
        float m_new = fmaxf(m, dot);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, w));
        const float alpha = m == kNegInf ? 0.0f : expf(m - m_new);
        // (a NaN score passes through here, whatever the maximum made of it)
        const float e = dot == kNegInf ? 0.0f : expf(dot - m_new);
        float sum = e;
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const float l_new = l * alpha + sum;
        const float keep = l > 0.0f ? l * alpha / l_new : 0.0f, weight = l_new != 0.0f ? e / l_new : 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= keep;
        // (addresses are bounded, not the loads: a conditional load is waited for at once; a column past the last
        // is not stored, and a key past the last counts as zeros, since its weight of nothing would not keep an
        // infinite value out)
        auto add = [&](int j0, auto whole) {
            float v[AHEAD][N];
#pragma unroll
            for (int j = 0; j < AHEAD; j++)
#pragma unroll
                for (int i = 0; i < N; i++) v[j][i] = vr.at(row0 + (uint64_t)min(j0 + j, keys - 1), vcol + min(lane + 32 * i, vdim - 1));
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                const float w = __shfl_sync(0xffffffffu, weight, j0 + j);
#pragma unroll
                for (int i = 0; i < N; i++) o[i] = fmaf(w, decltype(whole)::value || j0 + j < keys ? v[j][i] : 0.0f, o[i]);
            }
        };
        int j0 = 0;
#pragma unroll 1
        for (; j0 + AHEAD <= keys; j0 += AHEAD) add(j0, std::true_type{});
        if (j0 < keys) add(j0, std::false_type{});
        m = m_new;
        l = l_new;
    }
}

// All keys by one warp.
template <typename T, typename R, int N, int AHEAD>
__device__ __forceinline__ void attention_row(const k::PackedAttentionArgs& a, const R& kr, const R& vr, const SeqRow& s,
                                              uint64_t row, uint64_t head, int lane, float* q_shared) {
    float o[N], m, l;
    attention_keys<T, R, N, AHEAD>(a, kr, vr, s, row, head, lane, q_shared, 0, 32, o, m, l);
    T* out = (T*)a.out + (row * a.head_count + head) * a.value_dim;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane + 32 * i < (int)a.value_dim) out[lane + 32 * i] = from_f32<T>(o[i]);
}

}  // namespace mg
