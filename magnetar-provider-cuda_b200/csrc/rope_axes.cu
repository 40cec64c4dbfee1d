// Rotary positions with several axes: pair (a, b) of a head turned by the angle t = position on the
// pair's axis x the pair's frequency, (a cos t - b sin t, a sin t + b cos t).
#include <algorithm>
#include <cstring>

#include "sequences.cuh"

namespace mg {
namespace {

constexpr int kThreads = 256;

struct RopeAxesK {
    const void* x;
    void* out;
    const float* positions;
    uint64_t rows;
    uint32_t heads, width, half, rows_per_block;
    float scale;
    int axes, inverse;
    float frequency[k::kRopeAxesMaxPairs];
    uint8_t axis[k::kRopeAxesMaxPairs];
};

template <typename T, int N>
struct alignas(sizeof(T) * N == 16 ? 16 : sizeof(T)) Vec {
    T v[N];
};

// A block takes rows_per_block rows: first the cosines and sines of their (row, pair)s into shared
// memory, each computed once for all heads, then the rows themselves, N values per access.
// Streaming work: the bytes of x in and out bound it.  HALF: pairs are (i, i + half) of a head,
// else (2i, 2i + 1); a thread owns both values of its pairs, so out may be x.
template <typename T, int N, bool HALF>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesK p) {
    extern __shared__ float2 turn[];
    pdl_enter();
    const uint64_t row0 = (uint64_t)blockIdx.x * p.rows_per_block;
    const uint32_t rows = (uint32_t)min((uint64_t)p.rows_per_block, p.rows - row0);
    for (uint32_t i = threadIdx.x; i < rows * p.half; i += kThreads) {
        const uint32_t r = i / p.half, pair = i % p.half;
        const float angle = p.positions[(row0 + r) * p.axes + p.axis[pair]] * p.scale * p.frequency[pair];
        float s, c;
        sincosf(angle, &s, &c);
        turn[i] = make_float2(c, p.inverse ? -s : s);
    }
    __syncthreads();
    const T* x = (const T*)p.x + row0 * p.heads * p.width;
    T* out = (T*)p.out + row0 * p.heads * p.width;
    using V = Vec<T, N>;
    constexpr int M = sizeof(T) * N == 16 ? N : 1;  // values per access of the rest
    // per head: the rotated values' vectors (half-split: of the first half), then the others
    const uint32_t turned = (HALF ? p.half : 2 * p.half) / N, rest = (p.width - 2 * p.half) / M, per_head = turned + rest;
    const uint32_t total = rows * p.heads * per_head;
    for (uint32_t w = threadIdx.x; w < total; w += kThreads) {
        const uint32_t j = w % per_head, rh = w / per_head, r = rh / p.heads;
        const uint64_t at = (uint64_t)rh * p.width;
        if (j >= turned) {
            const uint64_t e = at + 2 * p.half + (uint64_t)(j - turned) * M;
            if (p.x != p.out) *reinterpret_cast<Vec<T, M>*>(out + e) = *reinterpret_cast<const Vec<T, M>*>(x + e);
            continue;
        }
        const float2* cs = turn + r * p.half;
        if constexpr (HALF) {
            const uint64_t e = at + j * N;
            V a = *reinterpret_cast<const V*>(x + e), b = *reinterpret_cast<const V*>(x + e + p.half);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float2 t = cs[j * N + i];
                const float u = to_f32(a.v[i]), v = to_f32(b.v[i]);
                a.v[i] = from_f32<T>(u * t.x - v * t.y);
                b.v[i] = from_f32<T>(u * t.y + v * t.x);
            }
            *reinterpret_cast<V*>(out + e) = a;
            *reinterpret_cast<V*>(out + e + p.half) = b;
        } else {
            const uint64_t e = at + (uint64_t)j * N;
            V a = *reinterpret_cast<const V*>(x + e);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 t = cs[(j * N + i) / 2];
                const float u = to_f32(a.v[i]), v = to_f32(a.v[i + 1]);
                a.v[i] = from_f32<T>(u * t.x - v * t.y);
                a.v[i + 1] = from_f32<T>(u * t.y + v * t.x);
            }
            *reinterpret_cast<V*>(out + e) = a;
        }
    }
}

template <typename T, int N>
mg_status launch(Device* d, const RopeAxesK& p, uint64_t blocks, uint32_t smem, bool half_split) {
    if (half_split) {
        enqueue(d, rope_axes_kernel<T, N, true>, (unsigned)blocks, kThreads, smem, p);
    } else if constexpr (N % 2 == 0) {
        enqueue(d, rope_axes_kernel<T, N, false>, (unsigned)blocks, kThreads, smem, p);
    }
    return launched(d, "rope launch");
}

}  // namespace

namespace k {

mg_status rope_axes(Device* d, const RopeAxesArgs& a) {
    if (a.rows == 0) return MG_OK;
    const uint64_t row_width = a.head_count * a.head_width;
    if (row_width > 0x7fffffffull / 64) return fail(MG_SHAPE_UNSUPPORTED, "RoPE rows of %llu values are too wide", (unsigned long long)row_width);
    RopeAxesK p;
    p.x = a.x;
    p.out = a.out;
    p.positions = a.positions;
    p.rows = a.rows;
    p.heads = (uint32_t)a.head_count;
    p.width = (uint32_t)a.head_width;
    p.half = (uint32_t)a.half;
    p.scale = a.scale;
    p.axes = a.axes;
    p.inverse = a.inverse;
    memcpy(p.frequency, a.frequency.data(), a.half * sizeof(float));
    memcpy(p.axis, a.axis.data(), a.half);
    // 16-byte accesses where every piece of a row starts on 16 bytes; else single pairs.
    const uint32_t n = 16 / (uint32_t)dtype_size(a.dtype);
    const bool vec = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0 && a.head_width % n == 0 &&
                     (2 * a.half) % n == 0 && (!a.half_split || a.half % n == 0);
    // About two accesses per thread in a block, and shared memory for at most 4096 turns.
    const uint64_t per_row = std::max<uint64_t>(1, row_width / (vec ? n : 2));
    p.rows_per_block = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(2 * kThreads / per_row, 4096 / a.half));
    const uint64_t blocks = (a.rows + p.rows_per_block - 1) / p.rows_per_block;
    if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "RoPE launch size overflows");
    const uint32_t smem = p.rows_per_block * p.half * (uint32_t)sizeof(float2);
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (vec) return launch<T, 16 / (int)sizeof(T)>(d, p, blocks, smem, a.half_split);
        return a.half_split ? launch<T, 1>(d, p, blocks, smem, true) : launch<T, 2>(d, p, blocks, smem, false);
    });
}

}  // namespace k
}  // namespace mg
