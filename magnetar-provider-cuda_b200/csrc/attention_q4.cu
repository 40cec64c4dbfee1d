// Attention of packed sequences over 4-bit key/value stores: head dimensions 64 and 128, any number of
// queries per sequence (a decode step has one).
//
// Each byte of the store is read once per 16 score rows, so a decode step is bound by memory: 0.53
// bytes a value against some 4 us of L2 and DRAM latency to cover, and, closer than for wider caches,
// by the instructions that turn 4 bits into an operand.  The products run on the warp-level tensor
// instructions (m16n8k16, f32 accumulators): their operands are registers, so a quant goes from shared
// memory to an operand without being written back, which the tcgen05 forms (operands in shared or
// tensor memory, 128 rows) would need; 16 rows are all a decode step has.
//
// Numbers: a quant q in [-8, 7] is a bfloat16 exactly, K's scale multiplies the scores of its block of
// 64 and V's scale its weights, both in f32.  bfloat16 queries and their weights are single terms, 16
// score rows.  f32 and f16 queries, and the weights, are two bfloat16 terms (hi in rows 0-7, lo in
// rows 8-15: together within 2^-17), 8 score rows.  A score row is one (query, head) of a kv head.
//
// A warp takes tiles of 64 keys on its own, with its own maximum, sum and output; the eight warps' and the
// splits' partial results are merged at the end, those of the splits by the CTA that finishes last.
#include <algorithm>

#include "attention_packed.cuh"
#include "sm100.cuh"

namespace mg {
namespace {

using namespace sm100;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;  // tiles of K and V a warp has in flight or in use

template <int D>
struct Q4Shape {
    static constexpr int kGroups = D / 64;                       // blocks of a head's row
    static constexpr int kTile = kGroups * (int)kQ4Record;       // a head's K (or V) of 64 keys
    static constexpr int kRing = kStages * 2 * kTile;            // of one warp
    static constexpr int kLd = D + 4;                            // floats of a merged output row (in bank-conflict-free steps)
    static constexpr int kMerge = kWarps * 16 * (kLd + 2) * 4;   // the warps' outputs, maxima and sums, over the rings
    static constexpr int kSmem = kWarps * kRing > kMerge ? kWarps * kRing : kMerge;
};

struct Q4Params {
    k::PackedAttentionArgs a;
    uint32_t group;        // heads per kv head
    uint32_t chunk;        // keys of a split, a multiple of 64
    uint32_t max_splits;   // of any row block
    float scale2;          // scores to log2 units
    float* partial;        // per (row block, kv head, split): rows x (D + 2)
    unsigned* counters;    // per (row block, kv head)
    int* error;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Nibbles i and i + 4 of a word, as the bfloat16 pair (q_i, q_{i+4}): 128 + (q + 8) by its bits, less 136.
__device__ __forceinline__ uint32_t dequant(uint32_t word, int i) {
    uint32_t x = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0x43084308u));
    return x;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attention_q4_kernel(const __grid_constant__ Q4Params p) {
    using S = Q4Shape<D>;
    constexpr bool kTwo = sizeof(T) == 4 || std::is_same<T, __half>::value;
    constexpr int R = kTwo ? 8 : 16;  // score rows
    constexpr int G = S::kGroups;
    constexpr float kNegInf = -__builtin_huge_valf();
    // the reference maximum moves only when a tile passes it by more than 2^8; weights are 2^(s - m - 40),
    // so that sums of large finite values stay finite
    constexpr float kLazy = 8.0f, kOffset = 40.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][kStages];
    __shared__ uint32_t s_seq, s_place, s_last;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t kvh = blockIdx.y;

    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int s = 0; s < kStages; s++) mbar_init(smem_u32(&bars[w][s]), 1);
        fence_barrier_init();
    }
    pdl_enter();
    const uint32_t step = p.a.table.step ? (uint32_t)*p.a.table.step : 0u;
    // Splits of a sequence's keys (as every row block of it sees them: its last rows see them all).
    auto splits_of = [&](uint32_t i) {
        const uint32_t keys = __ldg(&p.a.table.rows[i].k_count) + step;
        return max(1u, (keys + p.chunk - 1) / p.chunk);
    };
    auto blocks_of = [&](uint32_t i) { return (__ldg(&p.a.table.rows[i].q_count) * p.group + R - 1) / R; };
    if (warp == 0) {
        uint32_t seq, place;
        const bool found = find_item(p.a.table, blockIdx.x, [&](uint32_t i) { return blocks_of(i) * splits_of(i); }, seq, place);
        if (lane == 0) {
            s_seq = found ? seq : 0xffffffffu;
            s_place = found ? place : 0;
        }
    }
    __syncthreads();
    if (s_seq == 0xffffffffu) return;
    const SeqRow seq = seq_load(p.a.table, s_seq);
    const uint32_t splits = splits_of(s_seq), split = s_place % splits, block = s_place / splits;
    const int rows = (int)(seq.q_count * p.group), row0 = (int)block * R;  // score rows of the sequence; this block's first
    const int m_keys = (int)seq.k_count, shift = m_keys - (int)seq.q_count;
    const int window = p.a.window > 0 && p.a.window < 0x7fffffff ? (int)p.a.window : 0;

    // Keys [lo, hi) of the sequence that a score row sees.
    auto range = [&](int r, int& lo, int& hi) {
        const int pos = shift + r / (int)p.group;
        hi = r >= rows ? 0 : p.a.causal ? max(0, min(m_keys, pos + 1)) : m_keys;
        lo = window ? min(max(0, pos - window + 1), hi) : 0;
    };
    int b_lo, b_hi, x;  // of the block: its first row's lower end, its last row's upper end
    range(row0, b_lo, x);
    range(min(row0 + R, rows) - 1, x, b_hi);
    // This split's share of them.
    const int k_lo = max(b_lo, (int)(split * p.chunk)), k_hi = min(b_hi, (int)min((uint64_t)(split + 1) * p.chunk, (uint64_t)0x7fffffff));
    // Tiles lie on the store's own boundaries; sequences may start anywhere in one.
    const int64_t abs_lo = (int64_t)seq.k_start + k_lo;
    const int tile0 = (int)(abs_lo / 64);
    const int tiles = k_hi > k_lo ? (int)(((int64_t)seq.k_start + k_hi + 63) / 64) - tile0 : 0;

    // ---- each warp: tiles warp, warp + kWarps, ... ------------------------------------------------
    const int mine = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
    const uint64_t columns = p.a.kv_head_count * (uint64_t)G;  // records of a tile
    const uint8_t* kbase = (const uint8_t*)p.a.k + ((uint64_t)(tile0 + warp) * columns + kvh * G) * kQ4Record;
    const uint8_t* vbase = (const uint8_t*)p.a.v + ((uint64_t)(tile0 + warp) * columns + kvh * G) * kQ4Record;
    const uint64_t stride = (uint64_t)kWarps * columns * kQ4Record;
    uint8_t* ring = smem + warp * S::kRing;
    auto load = [&](int i) {  // (by lane 0)
        const int s = i % kStages;
        const uint32_t bar = smem_u32(&bars[warp][s]), dst = smem_u32(ring + s * 2 * S::kTile);
        mbar_arrive_expect_tx(bar, 2 * S::kTile);
        bulk_load(dst, kbase + (uint64_t)i * stride, S::kTile, bar);
        bulk_load(dst + S::kTile, vbase + (uint64_t)i * stride, S::kTile, bar);
    };
    if (lane == 0)
        for (int i = 0; i < min(kStages - 1, mine); i++) load(i);

    // The queries as MMA operands: in group gr and step st (16 columns), the lane's word at row g (and
    // g + 8) holds columns 64 gr + 16 t + 8 (st / 2) + {i, i + 4} and {i + 1, i + 5}, i = 2 (st % 2) --
    // the nibbles that one word of K gives at a time.
    uint32_t qf[G][4][4];
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const int r = row0 + g + (kTwo ? 0 : 8 * half);
        const bool live = r < rows;
        const int rr = min(r, rows - 1);
        const T* q = (const T*)p.a.q + ((uint64_t)(seq.q_start + (uint32_t)(rr / (int)p.group)) * p.a.head_count + kvh * p.group + (uint32_t)(rr % (int)p.group)) * D;
#pragma unroll
        for (int gr = 0; gr < G; gr++)
#pragma unroll
            for (int st = 0; st < 4; st++)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const int c = 64 * gr + 16 * t + 8 * (st / 2) + 2 * (st % 2) + w;
                    const float x0 = live ? to_f32(q[c]) : 0.0f, x1 = live ? to_f32(q[c + 4]) : 0.0f;
                    const uint32_t hi = pack_bf16(x0, x1);
                    const uint32_t lo = pack_bf16(x0 - lo_f(hi), x1 - hi_f(hi));
                    qf[gr][st][2 * w + half] = kTwo && half ? lo : hi;
                }
    }
    // Rows g (h = 0) and g + 8 (h = 1): the keys they see, relative to the sequence.
    constexpr int H = kTwo ? 1 : 2;
    int lo[H], hi[H];
#pragma unroll
    for (int h = 0; h < H; h++) {
        range(row0 + g + 8 * h, lo[h], hi[h]);
        lo[h] = max(lo[h], k_lo);
        hi[h] = min(hi[h], k_hi);
    }
    // (all rows see the keys [in_lo, in_hi))
    int in_lo, in_hi;
    range(min(row0 + R, rows) - 1, in_lo, x);
    range(row0, x, in_hi);
    in_lo = max(in_lo, k_lo);
    in_hi = min(in_hi, k_hi);

    float m[H], l[H];
    float o[G][8][4];
#pragma unroll
    for (int h = 0; h < H; h++) m[h] = kNegInf, l[h] = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G; gr++)
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[gr][j][e] = 0.0f;

    bool failed = false;
    for (int i = 0; i < mine; i++) {
        if (lane == 0 && i + kStages - 1 < mine) {
            fence_proxy_async();  // the stage's last reads come before the copy that overwrites it
            load(i + kStages - 1);
        }
        const int s = i % kStages;
        if (!mbar_wait(smem_u32(&bars[warp][s]), (uint32_t)(i / kStages) & 1u)) failed = true;
        failed = __any_sync(0xffffffffu, failed);
        if (failed) break;
        const uint8_t* kt = ring + s * 2 * S::kTile;
        const uint8_t* vt = kt + S::kTile;
        const int key0 = (int)((int64_t)(tile0 + warp + i * kWarps) * 64 - seq.k_start);  // of the tile, in the sequence (may be < 0)
        const bool whole = key0 >= in_lo && key0 + 64 <= in_hi;

        // ---- scores: 16 keys at a time, n-tiles of keys (t' , t' + 4) and (t' + 8, t' + 12) ----------
        // Accumulator column n of n-tile u is key 8 u + n / 2 + 4 (n % 2) of the 16, so lane (g, t)
        // has row g's scores of keys t, t + 4 (u = 0) and t + 8, t + 12 (u = 1).
        float sc[4][H][4];
        float mx[H];
#pragma unroll
        for (int h = 0; h < H; h++) mx[h] = kNegInf;
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[c][h][e] = 0.0f;
#pragma unroll
            for (int gr = 0; gr < G; gr++) {
                const uint8_t* rec = kt + gr * (int)kQ4Record;
                // scales of keys t, t + 4, t + 8, t + 12
                const uint2 sw = *reinterpret_cast<const uint2*>(rec + kQ4Quants + (16 * c + 4 * t) * 2);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint2 w = *reinterpret_cast<const uint2*>(rec + (16 * c + 8 * u + (g >> 1) + 4 * (g & 1)) * 32 + 8 * t);
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int st = 0; st < 4; st++) {
                        const uint32_t word = st < 2 ? w.x : w.y;
                        const int i2 = 2 * (st % 2);
                        mma16816(acc, qf[gr][st], dequant(word, i2), dequant(word, i2 + 1));
                    }
                    const uint32_t pair = u ? sw.y : sw.x;
                    const float d0 = lo_f(pair), d1 = hi_f(pair);
                    if constexpr (kTwo) {
                        sc[c][0][2 * u] = fmaf(d0, acc[0] + acc[2], sc[c][0][2 * u]);
                        sc[c][0][2 * u + 1] = fmaf(d1, acc[1] + acc[3], sc[c][0][2 * u + 1]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            sc[c][h][2 * u] = fmaf(d0, acc[2 * h], sc[c][h][2 * u]);
                            sc[c][h][2 * u + 1] = fmaf(d1, acc[2 * h + 1], sc[c][h][2 * u + 1]);
                        }
                    }
                }
            }
        }
        if (!whole) {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = key0 + 16 * c + t + 4 * e;
                        if (key < lo[h] || key >= hi[h]) sc[c][h][e] = kNegInf;
                    }
        }
        // ---- the rows' maxima, in log2 units; NaN stays NaN -------------------------------------------
#pragma unroll
        for (int h = 0; h < H; h++) {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx[h]) : "f"(sc[c][h][e]));
#pragma unroll
            for (int w = 1; w < 4; w <<= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, mx[h], w);
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(mx[h]) : "f"(other));
            }
            mx[h] *= p.scale2;
        }
        bool move[H];
        bool any = false;
#pragma unroll
        for (int h = 0; h < H; h++) {
            move[h] = mx[h] != kNegInf && !(mx[h] <= m[h] + kLazy);
            any = any || move[h];
        }
        if (__any_sync(0xffffffffu, any)) {
            float f[H];
#pragma unroll
            for (int h = 0; h < H; h++) {
                f[h] = !move[h] ? 1.0f : m[h] == kNegInf ? 0.0f : ex2(m[h] - mx[h]);
                if (move[h]) m[h] = fmaf(mx[h], 0.0f, mx[h]);  // (+inf becomes NaN)
                l[h] *= f[h];
            }
#pragma unroll
            for (int gr = 0; gr < G; gr++)
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[gr][j][e] *= f[kTwo ? 0 : e / 2];
        }
        // ---- weights, and O += P V ----------------------------------------------------------------------
        float ref[H];
#pragma unroll
        for (int h = 0; h < H; h++) ref[h] = m[h] == kNegInf ? 0.0f : -(m[h] + kOffset);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float w[H][4];
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[h][e] = ex2(fmaf(sc[c][h][e], p.scale2, ref[h]));
                    l[h] += w[h][e];
                }
#pragma unroll
            for (int gr = 0; gr < G; gr++) {
                const uint8_t* rec = vt + gr * (int)kQ4Record;
                const uint2 sw = *reinterpret_cast<const uint2*>(rec + kQ4Quants + (16 * c + 4 * t) * 2);
                float d[4] = {lo_f(sw.x), hi_f(sw.x), lo_f(sw.y), hi_f(sw.y)};
                float pw[H][4];
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        pw[h][e] = w[h][e] * d[e];
                        // a weight of nothing keeps out whatever the row holds
                        if (!whole && w[h][e] == 0.0f) pw[h][e] = 0.0f;
                    }
                uint32_t a[4];
                a[0] = pack_bf16(pw[0][0], pw[0][1]);  // row g, keys t, t + 4
                a[2] = pack_bf16(pw[0][2], pw[0][3]);  // row g, keys t + 8, t + 12
                if constexpr (kTwo) {
                    a[1] = pack_bf16(pw[0][0] - lo_f(a[0]), pw[0][1] - hi_f(a[0]));
                    a[3] = pack_bf16(pw[0][2] - lo_f(a[2]), pw[0][3] - hi_f(a[2]));
                } else {
                    a[1] = pack_bf16(pw[1][0], pw[1][1]);
                    a[3] = pack_bf16(pw[1][2], pw[1][3]);
                }
                // lane g's word of a key: columns 8 g .. 8 g + 7 of the block; two keys' halves side by side
                uint32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = *reinterpret_cast<const uint32_t*>(rec + (16 * c + t + 4 * e) * 32 + 4 * g);
                const uint32_t b0l = __byte_perm(v[0], v[1], 0x5410), b0h = __byte_perm(v[0], v[1], 0x7632);
                const uint32_t b1l = __byte_perm(v[2], v[3], 0x5410), b1h = __byte_perm(v[2], v[3], 0x7632);
#pragma unroll
                for (int j = 0; j < 8; j++) mma16816(o[gr][j], a, dequant(j < 4 ? b0l : b0h, j % 4), dequant(j < 4 ? b1l : b1h, j % 4));
            }
        }
        __syncwarp();  // all lanes have read the stage
    }
    if (failed && lane == 0) atomicExch(p.error, 1);

    // ---- the warps' results, merged --------------------------------------------------------------------
    // Accumulator j of block gr: columns 64 gr + 16 t + j (elements 0 and 2) and + 8 + j (1 and 3).
    __syncthreads();  // the rings are free
    float* so = reinterpret_cast<float*>(smem);                   // [warp][16 rows][kLd]
    float* sm = so + kWarps * 16 * S::kLd;                        // [warp][16][2]: m, l
#pragma unroll
    for (int h = 0; h < H; h++) {
        float sum = l[h];
#pragma unroll
        for (int w = 1; w < 4; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        float* row = so + (warp * 16 + g + 8 * h) * S::kLd;
#pragma unroll
        for (int gr = 0; gr < G; gr++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int c = 64 * gr + 16 * t + j;
                row[c] = kTwo ? o[gr][j][0] + o[gr][j][2] : o[gr][j][2 * h];
                row[c + 8] = kTwo ? o[gr][j][1] + o[gr][j][3] : o[gr][j][2 * h + 1];
            }
        if (t == 0) {
            sm[(warp * 16 + g + 8 * h) * 2] = m[h];
            sm[(warp * 16 + g + 8 * h) * 2 + 1] = sum;
        }
    }
    __syncthreads();
    // The merge of n (m, l, o) triples of a row: o / l weighed by 2^(m - max m).  NaN stays NaN.
    const uint32_t slot = 0;
    (void)slot;
    // rows of the block before this sequence's: every sequence's blocks have their own counters and partials
    const bool single = splits == 1;
    T* out = (T*)p.a.out;
    const uint64_t part = (uint64_t)blockIdx.x * p.a.kv_head_count + kvh;  // this CTA's partial
    constexpr int kPart = R * (D + 2);
    for (int e = threadIdx.x; e < R * (D / 4); e += kThreads) {
        const int r = e / (D / 4), c = 4 * (e % (D / 4));
        if (row0 + r >= rows) continue;
        float mm = kNegInf;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float mw = sm[(w * 16 + r) * 2];
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(mm) : "f"(mw));
        }
        float ll = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float mw = sm[(w * 16 + r) * 2], f = mw == kNegInf ? 0.0f : ex2(mw - mm);
            ll += f * sm[(w * 16 + r) * 2 + 1];
            const float4 v = *reinterpret_cast<const float4*>(so + (w * 16 + r) * S::kLd + c);
            acc[0] = fmaf(f, v.x, acc[0]);
            acc[1] = fmaf(f, v.y, acc[1]);
            acc[2] = fmaf(f, v.z, acc[2]);
            acc[3] = fmaf(f, v.w, acc[3]);
        }
        if (single) {
            const float inv = mm == kNegInf ? 0.0f : 1.0f / ll;
            const int rr = row0 + r;
            T* dst = out + ((uint64_t)(seq.q_start + (uint32_t)(rr / (int)p.group)) * p.a.head_count + kvh * p.group + (uint32_t)(rr % (int)p.group)) * D + c;
#pragma unroll
            for (int i = 0; i < 4; i++) dst[i] = from_f32<T>(acc[i] * inv);
        } else {
            float* dst = p.partial + part * kPart + r * (D + 2);
#pragma unroll
            for (int i = 0; i < 4; i++) dst[c + i] = acc[i];
            if (c == 0) {
                dst[D] = mm;
                dst[D + 1] = ll;
            }
        }
    }
    if (single) return;
    // ---- the splits' results, merged by the CTA that finishes last ----------------------------------------
    const uint32_t first = blockIdx.x - split;  // the block's first split's item, which also counts for the block
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned* counter = p.counters + (uint64_t)first * p.a.kv_head_count + kvh;
        s_last = atomicAdd(counter, 1u) == splits - 1;
        if (s_last) *counter = 0u;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const float* parts = p.partial + ((uint64_t)first * p.a.kv_head_count + kvh) * kPart;
    const uint64_t next = p.a.kv_head_count * (uint64_t)kPart;
    for (int e = threadIdx.x; e < R * (D / 2); e += kThreads) {
        const int r = e / (D / 2), c = 2 * (e % (D / 2));
        const int rr = row0 + r;
        if (rr >= rows) continue;
        const float* src = parts + r * (D + 2);
        float mm = kNegInf;
        for (uint32_t i = 0; i < splits; i++) {
            const float mw = __ldcg(src + i * next + D);
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(mm) : "f"(mw));
        }
        float ll = 0.0f, a0 = 0.0f, a1 = 0.0f;
        for (uint32_t i = 0; i < splits; i++) {
            const float* q = src + i * next;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + D)), v = __ldcg(reinterpret_cast<const float2*>(q + c));
            const float f = ml.x == kNegInf ? 0.0f : ex2(ml.x - mm);
            ll = fmaf(f, ml.y, ll);
            a0 = fmaf(f, v.x, a0);
            a1 = fmaf(f, v.y, a1);
        }
        const float inv = mm == kNegInf ? 0.0f : 1.0f / ll;
        T* dst = out + ((uint64_t)(seq.q_start + (uint32_t)(rr / (int)p.group)) * p.a.head_count + kvh * p.group + (uint32_t)(rr % (int)p.group)) * D + c;
        dst[0] = from_f32<T>(a0 * inv);
        dst[1] = from_f32<T>(a1 * inv);
    }
}

template <typename T, int D>
mg_status launch(Device* d, const k::PackedAttentionArgs& a) {
    using S = Q4Shape<D>;
    constexpr int R = sizeof(T) == 4 || std::is_same<T, __half>::value ? 8 : 16;
    static bool configured[64] = {false};
    if (!configured[d->ordinal & 63]) {
        MG_CUDA(cudaFuncSetAttribute(attention_q4_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
                "configuring the 4-bit attention kernel");
        configured[d->ordinal & 63] = true;
    }
    Q4Params p;
    p.a = a;
    p.group = (uint32_t)(a.head_count / a.kv_head_count);
    p.scale2 = a.scale * 1.4426950408889634f;
    p.counters = d->counters;
    p.error = d->flags + 2;
    // Splits: enough CTAs for the machine, of equal numbers of keys.
    uint64_t work = 0, blocks = 0;
    for (const SeqRow& r : a.host->rows) {
        const uint64_t b = ((uint64_t)r.q_count * p.group + R - 1) / R;
        blocks += b;
        work += b * (r.k_count + a.max_step);
    }
    constexpr uint64_t kUnit = 64 * kWarps;  // keys that give each warp a tile
    const uint64_t slots = (uint64_t)d->sm_count * 2;
    uint64_t chunk = (work * a.kv_head_count + slots - 1) / slots;
    chunk = std::max<uint64_t>(kUnit, (chunk + kUnit - 1) / kUnit * kUnit);
    auto items_at = [&](uint64_t c) {
        uint64_t n = 0;
        for (const SeqRow& r : a.host->rows)
            n += ((uint64_t)r.q_count * p.group + R - 1) / R * std::max<uint64_t>(1, (r.k_count + a.max_step + c - 1) / c);
        return n;
    };
    uint64_t items = items_at(chunk);
    if (items * a.kv_head_count > (1u << 16)) {  // more than there are counters: no splits, there are CTAs enough
        chunk = 1ull << 31;
        items = items_at(chunk);
    }
    if (items > 0x7fffffffull || a.kv_head_count > 65535) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    p.chunk = (uint32_t)chunk;
    p.max_splits = 0;
    MG_TRY(scratch(d, 9, chunk == 1ull << 31 ? 16 : items * a.kv_head_count * R * (D + 2) * sizeof(float), (void**)&p.partial));
    enqueue(d, attention_q4_kernel<T, D>, dim3((unsigned)items, (unsigned)a.kv_head_count), kThreads, S::kSmem, p);
    return launched(d, "4-bit attention launch");
}

}  // namespace

namespace k {

bool attention_q4_eligible(const PackedAttentionArgs& a) {
    return a.kv_dtype == MG_Q4 && (a.head_dim == 64 || a.head_dim == 128);
}

mg_status attention_q4(Device* d, const PackedAttentionArgs& a) {
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        return a.head_dim == 64 ? launch<T, 64>(d, a) : launch<T, 128>(d, a);
    });
}

}  // namespace k
}  // namespace mg
