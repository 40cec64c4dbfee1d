// Device-side reading of a table of packed sequences and of activations in any float type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"

namespace mg {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A row of `rows` (of the table's rows or ordered rows), with a captured step's advance.
__device__ __forceinline__ SeqRow seq_load(const k::SeqTable& t, const SeqRow* rows, uint32_t i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(rows) + i);
    return SeqRow{v.x, v.y, v.z, v.w + (t.step ? (uint32_t)*t.step : 0u)};
}
__device__ __forceinline__ SeqRow seq_load(const k::SeqTable& t, uint32_t i) { return seq_load(t, t.rows, i); }

// The sequence that owns packed query row `row` (below the table's queries): the last one that
// starts at or before it.  Empty sequences share their start with the next one, which is later.
__device__ __forceinline__ uint32_t seq_of_query(const k::SeqTable& t, uint32_t row) {
    uint32_t lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (__ldg(&t.rows[mid].q_start) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A thread's places in rows of `columns` pieces each, kStride pieces apart: one division at the start, then
// additions (a division by a variable is some 20 instructions, of 64 bits 70).
template <uint32_t kStride>
struct Places {
    uint64_t i;                                    // row
    uint32_t c, step_rows, step_columns, columns;  // piece of the row; the stride
    __device__ __forceinline__ Places(uint64_t first, uint32_t columns_) : columns(columns_) {
        if (first >> 32) {
            i = first / columns;
            c = (uint32_t)(first % columns);
        } else {
            i = (uint32_t)first / columns;
            c = (uint32_t)first % columns;
        }
        step_rows = kStride / columns;
        step_columns = kStride % columns;
    }
    __device__ __forceinline__ void next() {
        i += step_rows;
        c += step_columns;
        if (c >= columns) {
            c -= columns;
            i++;
        }
    }
};

// Work item `item` of a launch that gives a sequence of n queries `items_of(n)` items, sequences with the
// most keys first: the sequence's place in that order and the item's place in the sequence.  All lanes of
// a warp call it together; false past the last item.
template <class F>
__device__ __forceinline__ bool find_item(const k::SeqTable& t, uint32_t item, F&& items_of, uint32_t& seq, uint32_t& place) {
    const uint32_t lane = threadIdx.x % 32;
    uint32_t before = 0;
    for (uint32_t base = 0; base < t.count; base += 32) {
        const uint32_t i = base + lane;
        const uint32_t n = i < t.count ? items_of(__ldg(&t.ordered[i].q_count)) : 0;
        uint32_t sum = n;  // items of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= (uint32_t)o) sum += v;
        }
        const uint32_t owner = __ballot_sync(0xffffffffu, item < before + sum);
        if (owner) {
            const int l = __ffs(owner) - 1;
            seq = base + l;
            place = item - before - __shfl_sync(0xffffffffu, sum - n, l);
            return true;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

// Where a 4-bit store's record keeps the scale of its row r (of 64): of each 16, rows t + 4 e and
// t + 4 e + 8 (e = 0, 1) are neighbours, as the attention kernel's lanes take them.
__device__ __forceinline__ uint32_t q4_scale_slot(uint32_t r) {
    return (r & ~15u) | ((r & 3u) << 2) | ((r >> 1) & 2u) | ((r >> 3) & 1u);
}

// One dtype's kernel by a generic lambda: f(T{}).
template <class F>
inline mg_status by_float(mg_dtype t, F&& f) {
    switch (t) {
        case MG_F16: return f(__half{});
        case MG_BF16: return f(__nv_bfloat16{});
        default: return f(float{});
    }
}

}  // namespace mg
