// Rotary positions with several axes: pair (a, b) of a head turned by the angle t = position on the
// pair's axis x the pair's frequency, (a cos t - b sin t, a sin t + b cos t).
#include <algorithm>
#include <cstring>

#include "sequences.cuh"

namespace mg {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;   // heads that a thread takes together

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
struct alignas(sizeof(T) * N == 16 ? 16 : alignof(T)) Vec {
    T v[N];
};

// A block takes rows_per_block rows: a thread's first accesses are loaded, then the cosines and sines of
// the block's (row, pair)s go into shared memory, each computed once for all heads, then the values of
// kItems heads are turned, N per access.  Streaming work: the bytes of x in and out bound it.  HALF: pairs are
// (i, i + half) of a head, else (2i, 2i + 1); a thread owns both values of its pairs, so out may be x.
// 32768 rows of 32 x 128 bf16: 84 to 90 us, 6.0 to 6.4 TB/s, nearly a copy's rate.  1, 2, 4 heads at a time take 90, 87 and
// 84 (a turn is read from shared memory once for all of them); blocks of fewer rows, which leave threads
// without a turn to compute, 111 to 132; turns laid out pair after pair (bank conflicts) 140.
template <typename T, int N, bool HALF>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ RopeAxesK p) {
    extern __shared__ float2 turn[];
    pdl_enter();
    const uint64_t row0 = (uint64_t)blockIdx.x * p.rows_per_block;
    const uint32_t rows = (uint32_t)min((uint64_t)p.rows_per_block, p.rows - row0);
    const T* x = (const T*)p.x + row0 * p.heads * p.width;
    T* out = (T*)p.out + row0 * p.heads * p.width;
    using V = Vec<T, N>;
    constexpr int M = sizeof(T) * N == 16 ? N : 1;  // values per access of the rest
    // per head: the rotated values' vectors (half-split: of the first half), then the others
    constexpr int P = HALF ? N : N / 2;  // pairs of an access
    constexpr int Q = P > 1 ? 2 : 1;     // of those read together
    const uint32_t lanes = p.half / P,  rest = (p.width - 2 * p.half) / M, per_head = lanes + rest;
    const uint32_t groups = (p.heads + kItems - 1) / kItems, total = rows * groups * per_head;
    for (uint32_t base = 0; base < total; base += kThreads) {
        const uint32_t w = min(base + threadIdx.x, total - 1), j = w % per_head, g = w / per_head, r = g / groups, h = g % groups * kItems;
        const uint32_t row = r * p.heads * p.width, col = j < lanes ? j * N : 0;
        V a[kItems], b[HALF ? kItems : 1];
#pragma unroll
        for (int k = 0; k < kItems; k++) {
            // (the address is bounded, not the load: a conditional load is waited for at once)
            const uint32_t at = row + min(h + k, p.heads - 1) * p.width + col;
            a[k] = *reinterpret_cast<const V*>(x + at);
            if constexpr (HALF) b[k] = *reinterpret_cast<const V*>(x + at + p.half);
        }
        if (base == 0) {
            // turns of a row, an access's pairs two by two (one by one), so that neighbouring lanes read side by side
            for (uint32_t i = threadIdx.x; i < rows * p.half; i += kThreads) {
                const uint32_t q = i / p.half, f = i % p.half;
                const float angle = p.positions[(row0 + q) * p.axes + p.axis[f]] * p.scale * p.frequency[f];
                float s, c;
                sincosf(angle, &s, &c);
                turn[q * p.half + ((f % P) / Q * lanes + f / P) * Q + f % Q] = make_float2(c, p.inverse ? -s : s);
            }
            __syncthreads();
        }
        if (base + threadIdx.x >= total) break;
        if (j >= lanes) {
            if (p.x == p.out) continue;
            for (uint32_t k = h; k < min(h + kItems, p.heads); k++) {
                const uint32_t e = row + k * p.width + 2 * p.half + (j - lanes) * M;
                *reinterpret_cast<Vec<T, M>*>(out + e) = *reinterpret_cast<const Vec<T, M>*>(x + e);
            }
            continue;
        }
        const Vec<float2, Q>* cs = reinterpret_cast<const Vec<float2, Q>*>(turn + r * p.half) + j;
        Vec<float2, Q> t[P / Q];
#pragma unroll
        for (int i = 0; i < P / Q; i++) t[i] = cs[i * lanes];
#pragma unroll
        for (int k = 0; k < kItems; k++) {
            if (h + k >= p.heads) break;
            T* dst = out + row + (h + k) * p.width + col;
#pragma unroll
            for (int i = 0; i < P; i++) {
                const float2 z = t[i / Q].v[i % Q];
                T& first = a[k].v[HALF ? i : 2 * i];
                T& second = HALF ? b[HALF ? k : 0].v[HALF ? i : 0] : a[k].v[HALF ? 0 : 2 * i + 1];
                const float u = to_f32(first), v = to_f32(second);
                first = from_f32<T>(u * z.x - v * z.y);
                second = from_f32<T>(u * z.y + v * z.x);
            }
            *reinterpret_cast<V*>(dst) = a[k];
            if constexpr (HALF) *reinterpret_cast<V*>(dst + p.half) = b[HALF ? k : 0];
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
    // Eight accesses per thread in a block where the rows fill the SMs, and shared memory for at most 4096 turns.
    const uint64_t per_row = std::max<uint64_t>(1, row_width / (vec ? n : 2));
    p.rows_per_block = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(8 * kThreads / per_row, 4096 / a.half));
    p.rows_per_block = (uint32_t)std::min<uint64_t>(p.rows_per_block, std::max<uint64_t>(1, a.rows / (4 * (uint64_t)d->sm_count)));
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
