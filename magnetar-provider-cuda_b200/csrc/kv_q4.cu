// Key/value stores held in 4 bits: writing rows into them and reading them back.
//
// Format (mg_kv_store_q4): 64 consecutive values of a row share the scale d = bf16(m / -8), m being
// the value of largest magnitude, so m itself maps to -8 (up to d's rounding) and the other sign
// reaches 7/8 of it; q = rint(x / d) in [-8, 7].  A bfloat16 scale has f32's range: no block
// overflows or vanishes, and q * d (4 by 8 bits) is exact in f32.  One scale for 64 values rather
// than 32 because the attention that reads the store multiplies every weight by its value's scale:
// the block halves that work, and the store is 4.25 bits a value instead of 4.5.
#include <algorithm>

#include "sequences.cuh"

namespace mg {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint8_t* record(void* store, uint64_t row, uint64_t columns, uint64_t column) {
    return (uint8_t*)store + (row / kQ4Tile * columns + column) * kQ4Record;
}

// The store row that packed row `i` goes to (or is read from).
__device__ __forceinline__ uint64_t store_row(const k::KvPackedArgs& a, uint64_t i) {
    if (a.table.count == 0) return a.row_offset + i + (a.table.step ? *a.table.step : 0);
    const SeqRow s = seq_load(a.table, seq_of_query(a.table, (uint32_t)i));
    return (uint64_t)s.k_start + s.k_count - s.q_count + (i - s.q_start);
}

// Eight values of a block per thread, eight threads to a block, a warp's 32 lanes over four
// neighbouring blocks of one row: one 16-byte (f32: two) load per thread and one word stored.
// Streaming work, bound by the bytes read and written.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) q4_write_kernel(const k::KvPackedArgs a) {
    pdl_enter();
    const uint64_t columns = a.width / kQ4Block;
    const uint64_t total = a.queries * columns * 8;  // threads' worth of work
    const uint64_t stride = (uint64_t)gridDim.x * kThreads;
    const uint32_t part = threadIdx.x & 7;
    // whole groups of eight lanes leave together (total and the stride are multiples of 8)
    for (uint64_t w = (uint64_t)blockIdx.x * kThreads + threadIdx.x; w < total; w += stride) {
        const uint64_t block = w / 8;
        const uint64_t i = block / columns, c = block % columns;
        const T* src = (const T*)a.rows + i * a.width + c * kQ4Block + part * 8;
        float x[8];
        if constexpr (VEC) {
            if constexpr (sizeof(T) == 4) {
                const float4 u = __ldg(reinterpret_cast<const float4*>(src)), v = __ldg(reinterpret_cast<const float4*>(src) + 1);
                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
            } else {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
                const T* p = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = to_f32(p[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = to_f32(src[e]);
        }
        const uint64_t row = store_row(a, i);
        // the value of largest magnitude, the first of several: a strict comparison keeps the
        // earlier value inside the thread, the lower lane between threads
        float m = x[0];
        bool bad = !isfinite(x[0]);
#pragma unroll
        for (int e = 1; e < 8; e++) {
            if (fabsf(x[e]) > fabsf(m)) m = x[e];
            bad = bad || !isfinite(x[e]);
        }
        const uint32_t group = 0xffu << (threadIdx.x & 24);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            const float other = __shfl_xor_sync(group, m, o, 8);
            const bool lower = (part & o) != 0;  // the partner's values come first
            if (lower ? fabsf(other) >= fabsf(m) : fabsf(other) > fabsf(m)) m = other;
        }
        bad = __any_sync(group, bad);
        const __nv_bfloat16 scale = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : __fdiv_rn(m, -8.0f));
        const float d = __bfloat162float(scale);
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float q = d != 0.0f ? rintf(__fdiv_rn(x[e], d)) : 0.0f;
            q = fminf(fmaxf(q, -8.0f), 7.0f);  // NaN (a bad block) gives -8
            word |= (uint32_t)((int)q + 8) << (4 * e);
        }
        uint8_t* rec = record(a.store, row, columns, c);
        const uint32_t r = (uint32_t)(row % kQ4Tile);
        reinterpret_cast<uint32_t*>(rec)[r * 8 + part] = word;
        if (part == 0) reinterpret_cast<__nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot(r)] = scale;
    }
}

// The values rows stand for, as f32: the same split of the work, eight values per thread.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) q4_read_kernel(const k::KvPackedArgs a, float* out) {
    pdl_enter();
    const uint64_t columns = a.width / kQ4Block;
    const uint64_t total = a.queries * columns * 8, stride = (uint64_t)gridDim.x * kThreads;
    for (uint64_t w = (uint64_t)blockIdx.x * kThreads + threadIdx.x; w < total; w += stride) {
        const uint64_t block = w / 8, i = block / columns, c = block % columns;
        const uint32_t part = (uint32_t)(w & 7);
        const uint64_t row = store_row(a, i);
        const uint8_t* rec = record(a.store, row, columns, c);
        const uint32_t r = (uint32_t)(row % kQ4Tile);
        const uint32_t word = reinterpret_cast<const uint32_t*>(rec)[r * 8 + part];
        const float d = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot(r)]);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)((int)((word >> (4 * e)) & 15u) - 8) * d;
        float* dst = out + i * a.width + c * kQ4Block + part * 8;
        if constexpr (VEC) {
            reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) dst[e] = x[e];
        }
    }
}

// Rows copied into a store of their own type.
template <typename V>
__global__ void __launch_bounds__(kThreads) kv_copy_packed_kernel(const k::KvPackedArgs a, uint64_t per_row) {
    pdl_enter();
    const uint64_t n = a.queries * per_row, stride = (uint64_t)gridDim.x * kThreads;
    for (uint64_t w = (uint64_t)blockIdx.x * kThreads + threadIdx.x; w < n; w += stride) {
        const uint64_t i = w / per_row, e = w % per_row;
        ((V*)a.store)[store_row(a, i) * per_row + e] = ((const V*)a.rows)[w];
    }
}

unsigned grid(const Device* d, uint64_t items) {
    const uint64_t want = (items + kThreads - 1) / kThreads, cap = (uint64_t)d->sm_count * 16;
    return (unsigned)std::max<uint64_t>(1, std::min(want, cap));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

namespace k {

mg_status kv_write_packed(Device* d, const KvPackedArgs& a) {
    const uint64_t n = a.queries * a.width;
    if (n == 0) return MG_OK;
    if (a.store_dtype == MG_Q4) {
        const bool vec = aligned16(a.rows);  // rows are multiples of 64 values
        return by_float(a.dtype, [&](auto t) {
            using T = decltype(t);
            enqueue(d, vec ? q4_write_kernel<T, true> : q4_write_kernel<T, false>, grid(d, n / 8), kThreads, 0, a);
            return launched(d, "4-bit kv-write launch");
        });
    }
    const uint64_t bytes = a.width * dtype_size(a.dtype);
    if (aligned16(a.rows) && aligned16(a.store) && bytes % 16 == 0)
        enqueue(d, kv_copy_packed_kernel<uint4>, grid(d, n * dtype_size(a.dtype) / 16), kThreads, 0, a, bytes / 16);
    else if (dtype_size(a.dtype) == 4)
        enqueue(d, kv_copy_packed_kernel<uint32_t>, grid(d, n), kThreads, 0, a, a.width);
    else
        enqueue(d, kv_copy_packed_kernel<uint16_t>, grid(d, n), kThreads, 0, a, a.width);
    return launched(d, "packed kv-write launch");
}

mg_status kv_read_packed(Device* d, const KvPackedArgs& a, float* out) {
    const uint64_t n = a.queries * a.width;
    if (n == 0) return MG_OK;
    enqueue(d, aligned16(out) ? q4_read_kernel<true> : q4_read_kernel<false>, grid(d, n / 8), kThreads, 0, a, out);
    return launched(d, "4-bit kv-read launch");
}

}  // namespace k
}  // namespace mg
