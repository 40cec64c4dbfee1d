// Key/value stores held in 4 bits: writing rows into them and reading them back.
//
// Format (mg_kv_store_q4): 64 consecutive values of a row share the scale d = bf16(m / -8), m being
// the value of largest magnitude, so m itself maps to -8 (up to d's rounding) and the other sign
// reaches 7/8 of it; q = rint(x / d) in [-8, 7].  A bfloat16 scale has f32's range: no block
// overflows or vanishes, and q * d (4 by 8 bits) is exact in f32.  One scale for 64 values rather
// than 32 because the attention that reads the store multiplies every weight by its value's scale:
// the block halves that work, and the store is 4.25 bits a value instead of 4.5.
#include <algorithm>
#include <type_traits>

#include "sequences.cuh"
#include "sm100.cuh"

namespace mg {
namespace {

using namespace sm100;

constexpr int kThreads = 256;
constexpr uint32_t kPerBlock = 4;  // threads of a block of 64 values, as q4_write_kernel takes it
constexpr uint32_t kWriteBlocks = kThreads / kPerBlock, kReadBlocks = kThreads / 8;
constexpr int kWriteBytes = 64;             // loaded by a thread of q4_write_kernel before it works on them
constexpr int kReadPieces = 4, kCopyPieces = 4;
constexpr float kToInteger = 12582912.0f;  // 1.5 x 2^23: added to a small f32, it leaves its integer in the low bits

__device__ __forceinline__ uint8_t* record(void* store, uint64_t row, uint64_t columns, uint64_t column) {
    return (uint8_t*)store + (row / kQ4Tile * columns + column) * kQ4Record;
}

// A thread's places in packed rows, and the store rows they belong to.
template <uint32_t kStride>
struct Walk : Places<kStride> {
    using Places<kStride>::i;
    uint64_t advance;
    SeqRow s{0, 0, 0, 0};
    __device__ __forceinline__ Walk(const k::KvPackedArgs& a, uint64_t first, uint32_t columns) : Places<kStride>(first, columns) {
        advance = a.row_offset + (a.table.count == 0 && a.table.step ? *a.table.step : 0);
    }
    // The store row that packed row i goes to (or is read from).
    __device__ __forceinline__ uint64_t row(const k::KvPackedArgs& a) {
        if (a.table.count == 0) return advance + i;
        if ((uint32_t)i - s.q_start >= s.q_count) s = seq_load(a.table, seq_of_query(a.table, (uint32_t)i));
        return (uint64_t)s.k_start + (s.k_count - s.q_count + ((uint32_t)i - s.q_start));
    }
};

// A thread's sixteen values of a block, as they lie in memory.
template <typename T, bool VEC>
struct Sixteen {
    static constexpr int kWords = 4 * (int)sizeof(T);
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* src) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(src) + i / 4);
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            }
        } else {
            T* x = reinterpret_cast<T*>(w);
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = src[e];
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return to_f32(reinterpret_cast<const T*>(w)[e]); }
    // The largest value of the block's four threads and the negated smallest; NaN if there is one.
    __device__ __forceinline__ float2 ends(uint32_t group) const {
        if constexpr (sizeof(T) == 4) {
            float hi = (*this)[0], lo = -hi;
#pragma unroll
            for (int e = 1; e < 16; e++) {
                hi = max_nan(hi, (*this)[e]);
                lo = max_nan(lo, -(*this)[e]);
            }
#pragma unroll
            for (int o = 1; o < kPerBlock; o <<= 1) {
                hi = max_nan(hi, __shfl_xor_sync(group, hi, o, kPerBlock));
                lo = max_nan(lo, __shfl_xor_sync(group, lo, o, kPerBlock));
            }
            return make_float2(hi, lo);
        } else {
            constexpr uint32_t kSigns = 0x80008000u;
            uint32_t hi = w[0], lo = w[0] ^ kSigns;
#pragma unroll
            for (int i = 1; i < kWords; i++) {
                hi = max2(hi, w[i]);
                lo = max2(lo, w[i] ^ kSigns);
            }
            uint32_t both = max2(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
#pragma unroll
            for (int o = 1; o < kPerBlock; o <<= 1) both = max2(both, __shfl_xor_sync(group, both, o, kPerBlock));
            const T* v = reinterpret_cast<const T*>(&both);
            return make_float2(to_f32(v[0]), to_f32(v[1]));
        }
    }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t d;
        if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
};

// Sixteen values of a block per thread, four threads to a block, a warp's 32 lanes over eight neighbouring
// blocks: 16-byte loads, two words stored.  Streaming work, bound by the bytes read and written once the
// instructions per value are few: a thread loads all that it takes before it works on it, finds the rows by
// adding (no division), takes the largest magnitude as a largest and a smallest value (of 16-bit types
// two at a time), and divides by a reciprocal.  With eight values per thread what a block needs once
// outweighs its values (9.8 M instructions against 13.9 M).  17772 rows of 1024 bf16 written and read back:
// 28 us for 129 MB, 4.5 TB/s; half of the issue slots are taken.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) q4_write_kernel(const k::KvPackedArgs a) {
    constexpr int kPieces = kWriteBytes / (16 * (int)sizeof(T));
    pdl_enter();
    const uint32_t columns = (uint32_t)(a.width / kQ4Block);
    const uint64_t total = a.queries * columns;  // blocks
    const uint32_t part = threadIdx.x % kPerBlock, group = 0xfu << (threadIdx.x & 28);
    const uint64_t first = (uint64_t)blockIdx.x * (kPieces * kWriteBlocks) + threadIdx.x / kPerBlock;
    if (first >= total) return;  // (a block's lanes together, as below)
    Sixteen<T, VEC> piece[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; j++)
        piece[j].load((const T*)a.rows + min(first + j * kWriteBlocks, total - 1) * kQ4Block + part * 16);
    Walk<kWriteBlocks> at(a, first, columns);
#pragma unroll
    for (int j = 0; j < kPieces; j++) {
        if (j) at.next();
        if (at.i >= a.queries) return;
        const uint64_t row = at.row(a);
        // the value of largest magnitude, the first of several
        const float2 ends = piece[j].ends(group);
        const float hi = ends.x, lo = -ends.y;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = piece[j][e];
        float m = hi > -lo ? hi : lo;
        if (hi == -lo) {
            int sign = 0;
#pragma unroll
            for (int e = 15; e >= 0; e--) sign = x[e] == hi ? 1 : x[e] == lo ? -1 : sign;
            const uint32_t has = __ballot_sync(group, sign != 0) & group;
            m = __shfl_sync(group, sign, __ffs(has) - 1) > 0 ? hi : lo;
        }
        // an infinity or a NaN in the block: the scale is NaN
        const __nv_bfloat16 scale = __float2bfloat16_rn(fabsf(m) < __int_as_float(0x7f800000) ? m * -0.125f : __int_as_float(0x7fc00000));
        // x / d as x r + x s with r + s = 1 / d to twice the bits of an f32: a quotient that is a half exactly
        // comes out exact, the others on their side of it (x of 24 bits and d of 8 leave no quotient nearer to
        // a half than an f32 shows).  Blocks of small or large values are scaled, so that no part leaves the
        // range; where d is so small that its own rounding is coarse, quotients beyond 8 are cut to it.
        float d = __bfloat162float(scale);
        if (!(fabsf(m) >= 0x1p-60f && fabsf(m) <= 0x1p60f)) {
            const float by = fabsf(m) > 1.0f ? 0x1p-64f : 0x1p64f;
            d *= by;
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = fminf(fmaxf(x[e] * by, -8.0f * fabsf(d)), 8.0f * fabsf(d));
        }
        const float inv = d != 0.0f ? __frcp_rn(d) : 0.0f;  // no scale: everything is zero
        const float rest = fmaf(-d, inv, 1.0f) * inv;
        const uint64_t inv2 = f2(inv, inv), rest2 = f2(rest, rest), to_integer = f2(kToInteger, kToInteger);
        uint32_t word[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            word[h] = 0x88888888u - __float_as_uint(kToInteger) * 0x11111111u;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint64_t v = f2(x[8 * h + e], x[8 * h + e + 1]);
                uint64_t y = f2mul(v, rest2);
                f2fma(y, v, inv2);
                // q in [-8, 8] (d's rounding), 8 becomes 7; to an integer, ties to even, in the low bits of a float
                const float2 q = f2split(y), n = f2split(f2add(f2(fminf(q.x, 7.0f), fminf(q.y, 7.0f)), to_integer));
                word[h] += __float_as_uint(n.x) << (4 * e);
                word[h] += __float_as_uint(n.y) << (4 * e + 4);
            }
        }
        uint8_t* rec = record(a.store, row, columns, at.c);
        const uint32_t r = (uint32_t)(row % kQ4Tile);
        reinterpret_cast<uint2*>(rec)[r * kPerBlock + part] = make_uint2(word[0], word[1]);
        if (part == 0) reinterpret_cast<__nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot(r)] = scale;
    }
}

// The values rows stand for, as f32: eight threads to a block, each with two times four values, so that a
// warp's stores are whole lines.  A quant n is the float 16 + n by its bits (a conversion runs at a quarter of the rate).
// Bound by the 73 MB that it writes for 17772 rows of 1024 (written and read back, with 1, 2 or 4 pieces at a
// time: 31.7, 29.7 and 28.4 us).
template <bool VEC>
__global__ void __launch_bounds__(kThreads) q4_read_kernel(const k::KvPackedArgs a, float* out) {
    pdl_enter();
    const uint32_t columns = (uint32_t)(a.width / kQ4Block), part = threadIdx.x % 8;
    const uint64_t total = a.queries * columns, first = (uint64_t)blockIdx.x * (kReadPieces * kReadBlocks) + threadIdx.x / 8;
    if (first >= total) return;
    Walk<kReadBlocks> at(a, first, columns);
    uint32_t four[kReadPieces][2];
    float d[kReadPieces];
#pragma unroll
    for (int j = 0; j < kReadPieces; j++) {
        if (at.i >= a.queries) at.i = a.queries - 1;  // (read, not written)
        const uint64_t row = at.row(a);
        const uint8_t* rec = record(a.store, row, columns, at.c);
        const uint32_t r = (uint32_t)(row % kQ4Tile);
        const uint16_t* quants = reinterpret_cast<const uint16_t*>(rec) + r * 16 + part;
        four[j][0] = quants[0];
        four[j][1] = quants[8];
        d[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(rec + kQ4Quants)[q4_scale_slot(r)]);
        at.next();
    }
#pragma unroll
    for (int j = 0; j < kReadPieces; j++) {
        if (first + j * kReadBlocks >= total) return;
        float* dst = out + (first + j * kReadBlocks) * kQ4Block + part * 4;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = (__uint_as_float((four[j][h] << (19 - 4 * e) & 0x780000u) | 0x41800000u) - 24.0f) * d[j];
            if constexpr (VEC) {
                reinterpret_cast<float4*>(dst)[8 * h] = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) dst[32 * h + e] = x[e];
            }
        }
    }
}

// Rows copied into a store of their own type, a value V per thread and piece.
template <typename V>
__global__ void __launch_bounds__(kThreads) kv_copy_packed_kernel(const k::KvPackedArgs a, uint32_t per_row) {
    pdl_enter();
    const uint64_t total = a.queries * per_row, first = (uint64_t)blockIdx.x * (kCopyPieces * kThreads) + threadIdx.x;
    if (first >= total) return;
    V v[kCopyPieces];
#pragma unroll
    for (int j = 0; j < kCopyPieces; j++) v[j] = ((const V*)a.rows)[min(first + j * kThreads, total - 1)];
    Walk<kThreads> at(a, first, per_row);
#pragma unroll
    for (int j = 0; j < kCopyPieces; j++) {
        if (j) at.next();
        if (at.i >= a.queries) return;
        ((V*)a.store)[at.row(a) * per_row + at.c] = v[j];
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

namespace k {

// A launch over `pieces` of work, per_block to a block.
template <class... P>
static mg_status over(Device* d, void (*kernel)(P...), uint64_t pieces, uint64_t per_block, const char* what, P... params) {
    const uint64_t blocks = (pieces + per_block - 1) / per_block;
    if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "%s of too many values", what);
    enqueue(d, kernel, (unsigned)blocks, kThreads, 0, params...);
    return launched(d, what);
}

mg_status kv_write_packed(Device* d, const KvPackedArgs& a) {
    const uint64_t size = dtype_size(a.dtype), n = a.queries * a.width;
    if (n == 0) return MG_OK;
    if (a.width >> 32) return fail(MG_SHAPE_UNSUPPORTED, "kv-write rows of %llu values are too wide", (unsigned long long)a.width);
    if (a.store_dtype == MG_Q4) {
        return by_float(a.dtype, [&](auto t) {
            using T = decltype(t);
            // (rows are multiples of 64 values)
            return over(d, aligned16(a.rows) ? q4_write_kernel<T, true> : q4_write_kernel<T, false>, n / kQ4Block,
                        kWriteBytes / (16 * size) * kWriteBlocks, "4-bit kv-write launch", a);
        });
    }
    constexpr uint64_t per_block = kCopyPieces * kThreads;
    if (aligned16(a.rows) && aligned16(a.store) && a.width * size % 16 == 0)
        return over(d, kv_copy_packed_kernel<uint4>, n * size / 16, per_block, "packed kv-write launch", a, (uint32_t)(a.width * size / 16));
    return size == 4 ? over(d, kv_copy_packed_kernel<uint32_t>, n, per_block, "packed kv-write launch", a, (uint32_t)a.width)
                     : over(d, kv_copy_packed_kernel<uint16_t>, n, per_block, "packed kv-write launch", a, (uint32_t)a.width);
}

mg_status kv_read_packed(Device* d, const KvPackedArgs& a, float* out) {
    if (a.queries * a.width == 0) return MG_OK;
    if (a.width >> 32) return fail(MG_SHAPE_UNSUPPORTED, "kv-read rows of %llu values are too wide", (unsigned long long)a.width);
    return over(d, aligned16(out) ? q4_read_kernel<true> : q4_read_kernel<false>, a.queries * (a.width / kQ4Block), kReadPieces * kReadBlocks,
                "4-bit kv-read launch", a, out);
}

}  // namespace k
}  // namespace mg
