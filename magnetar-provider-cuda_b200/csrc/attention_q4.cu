// Attention of packed sequences over 4-bit key/value stores: head dimensions 64 and 128, any number of
// queries per sequence (a decode step has one).
//
// A decode step reads each byte of the store once: 0.53 bytes a value of DRAM traffic, against which stand
// the instructions that make an operand of 4 bits.  The products run on the warp-level tensor
// instructions (m16n8k16, f32 accumulators): their operands are registers, so a quant goes from shared
// memory to an operand without being written back, which the tcgen05 forms (operands in shared or
// tensor memory, 128 rows) would need.  Keys, and V's columns, are the 16 rows of an instruction and
// queries its 8 columns (S^T = K Q^T, O^T = V^T P^T): the quants, of which there are many, take the large
// side, and each is made an operand once.  With keys as columns and 16 queries as rows, a step of 4 heads
// per kv head issued twice the products and softmax instructions (189 us for 16 sequences of 32768
// keys and more, in bfloat16).
//
// Numbers: a quant q in [-8, 7] is a bfloat16 exactly.  For bfloat16 queries K's operands are 136 + q, one
// step short of it, and the accumulators start at -136 times the query's sum instead; the rounding at
// that size (some 2^-18 of a score) is lost in the outputs' own, but not in f32's, and V's many keys would
// make it grow.  K's scale multiplies the scores of its block of 64 and V's scale its weights, both in
// f32.  bfloat16 queries and their weights are single terms, a column each.  f32 and f16 queries, and the
// weights, are two bfloat16 terms (together within 2^-17) in neighbouring columns.  A score row
// is one (query, head) of a kv head.
//
// The tiles (64 keys on the store's own boundaries) of all sequences and row blocks form one line per kv
// head, each row block with a length for its own cost in front, and the line is cut into equal shares,
// one per CTA: however ragged the batch, all CTAs have as much to do.  A captured step's grid is sized for the
// keys it may grow to; of its CTAs as many have a share as the line's present length asks for.  In
// a share a warp takes every fourth tile on its own, with its own maximum, sum and output.  The four warps'
// results are merged in shared memory, those of a row block that was cut by the CTA that finishes last.
//
// (One bfloat16 term for the weights is what their products' rate allows: outputs are 2.3e-3 off, of which their own
// rounding is 1.7e-3; two terms leave 3.8e-6 where f32 arithmetic has 5e-7.)
//
// One query each, 32 heads over 8 of 128: 16 sequences, 15 of 32768 keys and one of 131071, bfloat16, 147 to 156 us,
// 4.4 to 4.6 TB/s of the store (half of the ALU's slots); 32 sequences of some 100 to 16000 keys, f32, 41 us.
#include <algorithm>
#include <type_traits>

#include "attention_packed.cuh"
#include "sm100.cuh"

namespace mg {
namespace {

using namespace sm100;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;  // tiles of K and V a warp has in flight or in use
constexpr int kBlockCost = 12;  // a row block's queries and merge cost as much as so many tiles
constexpr uint64_t kLeastShare = kBlockCost + kWarps;  // units: a tile for each warp, beside a row block's cost
constexpr int kPerSm = 3;   // CTAs of an SM: as many as shared memory holds

template <int D>
struct Q4Shape {
    static constexpr int kGroups = D / 64;                       // blocks of a head's row
    static constexpr int kTile = kGroups * (int)kQ4Record;       // a head's K (or V) of 64 keys
    static constexpr int kRing = kStages * 2 * kTile;            // of one warp
    static constexpr int kLd = D + 4;                            // floats of a row in the merge
    static constexpr int kMerge = kWarps * 16 * (kLd + 2) * 4;   // the warps' outputs, maxima and sums (16 rows at most), over the rings
    static constexpr int kSmem = kWarps * kRing > kMerge ? kWarps * kRing : kMerge;
};

struct Q4Params {
    k::PackedAttentionArgs a;
    uint32_t group;        // heads per kv head
    uint64_t units;        // of all row blocks (without a captured step's advance)
    float scale2;          // scores to log2 units
    float* partial;        // two per CTA: R x (D + 2)
    unsigned* counters;    // per CTA, for the row block that runs on past its share
    int* error;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// The same from other accumulators.
__device__ __forceinline__ void mma16816_from(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Values i and i + 4 of a word as a bfloat16 pair: 128 + (q + 8) by its bits ...  (One and-or per pair: its
// second constant has to come from a register, here one that the compiler does not know the value of.)
__device__ __forceinline__ uint32_t biased(uint32_t word, int i, uint32_t magic) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(x) : "r"(word >> (4 * i)), "r"(magic));
    return x;
}
// ... and q itself.
__device__ __forceinline__ uint32_t dequant(uint32_t word, int i, uint32_t magic) {
    uint32_t x = biased(word, i, magic);
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0x43084308u));  // less 136
    return x;
}

// The transpose of an 8 x 8 matrix of 16-bit values, two of a row in each lane's word.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// NT: column tiles of 8, that is 8 NT bfloat16 score rows of a block, or 4 NT of the two-term types.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? kPerSm : 2) attention_q4_kernel(const __grid_constant__ Q4Params p) {
    using S = Q4Shape<D>;
    constexpr bool kTwo = !std::is_same<T, __nv_bfloat16>::value;
    constexpr int R = (kTwo ? 4 : 8) * NT;  // score rows
    constexpr int H = kTwo ? 1 : 2;         // rows of a lane in a column tile: t, or 2 t and 2 t + 1
    constexpr int G = S::kGroups;
    constexpr int kPart = R * (D + 2);
    constexpr float kNegInf = -__builtin_huge_valf();
    // the reference maximum moves only when a tile passes it by more than 2^8; weights are 2^(s - m - 40),
    // so that sums of large finite values stay finite
    constexpr float kLazy = 8.0f, kOffset = 40.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][kStages];
    __shared__ uint32_t s_order;
    __shared__ uint64_t s_at, s_units;
    __shared__ uint32_t s_last;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const uint32_t kvh = blockIdx.y;
    const k::SeqTable& tab = p.a.table;
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(magic));

    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; w++)
            for (int s = 0; s < kStages; s++) mbar_init(smem_u32(&bars[w][s]), 1);
        fence_barrier_init();
    }
    if (tab.step) pdl_enter();  // (the table itself was written by copies, which a launch never overtakes)
    // A sequence's units (its tiles, and what a row block costs beside them), and its row blocks.
    auto units_of = [&](const SeqRow& q) { return kBlockCost + (uint32_t)(((uint64_t)q.k_start + q.k_count + 63) / 64 - q.k_start / 64); };
    auto blocks_of = [&](const SeqRow& q) { return (q.q_count * p.group + R - 1) / R; };
    // CTAs that have a share: all of an eager launch's grid.  No share of theirs is empty, so the last one to
    // finish a row block is one of those that it was cut among.
    auto shares_of = [&](uint64_t units) { return min((uint64_t)gridDim.x, max((uint64_t)1, (units + kLeastShare - 1) / kLeastShare)); };
    if (warp == 0) {
        // The line's length, and this CTA's share of it: from unit `begin` on; then the sequence it lies in.
        uint64_t units = p.units;
        if (tab.step) {
            units = 0;
            for (uint32_t i = lane; i < tab.count; i += 32) {
                const SeqRow q = seq_load(tab, i);
                units += (uint64_t)blocks_of(q) * units_of(q);
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) units += __shfl_xor_sync(0xffffffffu, units, w);
        }
        const uint64_t begin = units * blockIdx.x / shares_of(units);
        uint64_t before = 0;
        uint32_t order = 0xffffffffu;
        for (uint32_t base = 0; base < tab.count && order == 0xffffffffu; base += 32) {
            const uint32_t i = base + lane;
            uint64_t sum = 0;
            if (i < tab.count) {
                const SeqRow q = seq_load(tab, tab.ordered, i);
                sum = (uint64_t)blocks_of(q) * units_of(q);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const uint32_t owner = __ballot_sync(0xffffffffu, begin < before + sum);
            if (owner) {
                const int l = __ffs(owner) - 1;
                order = base + l;
                if (l > 0) before += __shfl_sync(0xffffffffu, sum, l - 1);
            } else {
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        if (lane == 0) {
            s_order = order;
            s_at = begin - before;  // units of the sequence before the share
            s_units = units;
        }
    }
    if (!tab.step) pdl_enter();
    __syncthreads();
    const uint64_t units = s_units, grid = shares_of(units);
    // (past the last share: past the line's end, where there is no sequence)
    uint64_t pos = units * blockIdx.x / grid;
    const uint64_t end = units * (blockIdx.x + 1) / grid;
    uint32_t order = s_order;
    uint64_t at = s_at;
    const int window = p.a.window > 0 && p.a.window < 0x7fffffff ? (int)p.a.window : 0;
    const uint64_t columns = p.a.kv_head_count * (uint64_t)G;  // records of a tile
    uint8_t* ring = smem + warp * S::kRing;
    uint32_t filled = 0;  // tiles this warp has had (the phase of its ring)
    bool failed = false;
    uint32_t missing = 0;  // the first tile that did not come
    T* out = (T*)p.a.out;

    // ---- row blocks, or the shares of them, one after another ---------------------------------------
    while (pos < end && order < tab.count) {
        const SeqRow seq = seq_load(tab, tab.ordered, order);
        const uint32_t all_units = units_of(seq);
        const uint64_t seq_units = (uint64_t)blocks_of(seq) * all_units;
        if (at >= seq_units) {  // (an empty sequence, or the last one done)
            at = 0;
            order++;
            continue;
        }
        const uint32_t block = (uint32_t)(at / all_units), first = (uint32_t)(at % all_units);
        const uint32_t count = (uint32_t)min((uint64_t)(all_units - first), end - pos);
        const uint64_t block_begin = pos - first;  // the row block's units on the line
        const int rows = (int)(seq.q_count * p.group), row0 = (int)block * R;  // score rows of the sequence; this block's first
        const int m_keys = (int)seq.k_count, shift = m_keys - (int)seq.q_count;

        // Keys [lo, hi) of the sequence that a score row sees.
        auto range = [&](int r, int& lo, int& hi) {
            const int pos_r = shift + r / (int)p.group;
            hi = r >= rows ? 0 : p.a.causal ? max(0, min(m_keys, pos_r + 1)) : m_keys;
            lo = window ? min(max(0, pos_r - window + 1), hi) : 0;
        };
        const int last_row = min(row0 + R, rows) - 1;
        int b_lo, b_hi, in_lo, in_hi;  // keys some row sees, and keys all rows see
        range(row0, b_lo, in_hi);
        range(last_row, in_lo, b_hi);
        // The tiles of this share that hold keys some row sees.
        const int tile_first = (int)(seq.k_start / 64);
        const int see_lo = (int)((seq.k_start + (uint32_t)b_lo) / 64) - tile_first;
        const int see_hi = b_hi > b_lo ? (int)(((uint64_t)seq.k_start + (uint32_t)b_hi + 63) / 64) - tile_first : see_lo;
        const int tile0 = tile_first + max((int)first - kBlockCost, see_lo), tile1 = tile_first + min((int)(first + count) - kBlockCost, see_hi);
        const int tiles = tile1 - tile0;
        // tiles warp, warp + kWarps, ...; none after a wait has run out (the shares' arrivals still have to be counted)
        const int mine = tiles > warp && !failed ? (tiles - warp + kWarps - 1) / kWarps : 0;

        const uint8_t* kbase = (const uint8_t*)p.a.k + ((uint64_t)(tile0 + warp) * columns + kvh * G) * kQ4Record;
        const uint8_t* vbase = (const uint8_t*)p.a.v + ((uint64_t)(tile0 + warp) * columns + kvh * G) * kQ4Record;
        const uint64_t stride = (uint64_t)kWarps * columns * kQ4Record;
        auto load = [&](int i) {  // (by lane 0)
            const uint32_t s = (filled + (uint32_t)i) % kStages;
            const uint32_t bar = smem_u32(&bars[warp][s]), dst = smem_u32(ring + s * 2 * S::kTile);
            mbar_arrive_expect_tx(bar, 2 * S::kTile);
            bulk_load(dst, kbase + (uint64_t)i * stride, S::kTile, bar);
            bulk_load(dst + S::kTile, vbase + (uint64_t)i * stride, S::kTile, bar);
        };
        if (lane == 0) {
            fence_proxy_async();  // what was read and written here comes before the copies
            for (int i = 0; i < min(kStages, mine); i++) load(i);
        }

        // The queries as MMA operands: in group gr and step st (16 columns of q), column g of a tile, the lane's
        // words hold columns 64 gr + 16 t + 8 (st / 2) + {i, i + 4} and {i + 1, i + 5}, i = 2 (st % 2) --
        // the quants that one word of K gives at a time.  And what the accumulators start from.
        uint32_t qf[NT][G][4][2];
        float start[NT][G][4];  // (four registers, as an accumulator has)
#pragma unroll
        for (int x = 0; x < NT; x++) {
            const int r = row0 + (kTwo ? 4 * x + g / 2 : 8 * x + g), rr = min(r, rows - 1);
            const bool live = r < rows;
            const T* q = (const T*)p.a.q + ((uint64_t)(seq.q_start + (uint32_t)(rr / (int)p.group)) * p.a.head_count + kvh * p.group +
                                            (uint32_t)(rr % (int)p.group)) * D + 16 * t;
#pragma unroll
            for (int gr = 0; gr < G; gr++) {
                float v[16], sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e++) v[e] = to_f32(q[64 * gr + e]);
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    v[e] = live ? v[e] : 0.0f;
                    sum += v[e];
                }
#pragma unroll
                for (int st = 0; st < 4; st++)
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const int c = 8 * (st / 2) + 2 * (st % 2) + w;
                        const uint32_t hi = pack_bf16(v[c], v[c + 4]);
                        qf[x][gr][st][w] = kTwo && (g & 1) ? pack_bf16(v[c] - lo_f(hi), v[c + 4] - hi_f(hi)) : hi;
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);  // of column g
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float s = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * h);  // of column 2 t + h
                    start[x][gr][h] = start[x][gr][2 + h] = kTwo ? 0.0f : -136.0f * s;
                }
            }
        }
        // The lane's rows, the keys they see, maxima (in log2 units) and sums; the output's columns
        // 64 gr + 8 g + 2 j (elements 0, 1: the lane's columns) and the next (2, 3).
        auto row_of = [&](int x, int h) { return kTwo ? 4 * x + t : 8 * x + 2 * t + h; };
        int lo[NT][H], hi[NT][H];
        float m[NT][H];
        uint64_t l2[NT];
        float o[NT][G][4][4];
#pragma unroll
        for (int x = 0; x < NT; x++) {
            l2[x] = f2(0.0f, 0.0f);
#pragma unroll
            for (int h = 0; h < H; h++) {
                range(row0 + row_of(x, h), lo[x][h], hi[x][h]);
                m[x][h] = kNegInf;
            }
#pragma unroll
            for (int gr = 0; gr < G; gr++)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[x][gr][j][e] = 0.0f;
        }

#pragma unroll 1
        for (int i = 0; i < mine; i++) {
            const uint32_t fill = filled + (uint32_t)i, s = fill % kStages;
            if (!mbar_wait(smem_u32(&bars[warp][s]), (fill / kStages) & 1u)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            if (failed) {
                missing = fill;
                break;
            }
            const uint8_t* kt = ring + s * 2 * S::kTile;
            const uint8_t* vt = kt + S::kTile;
            const int key0 = (int)((int64_t)(tile0 + warp + i * kWarps) * 64 - seq.k_start);  // of the tile, in the sequence (may be < 0)
            const bool whole = key0 >= in_lo && key0 + 64 <= in_hi;

            // ---- scores, 16 keys at a time ------------------------------------------------------------
            // Rows g and g + 8 of the instruction are keys kg = g / 2 + 4 (g % 2) and kg + 8.  A pair of scores:
            // of the lane's two rows for one key, or with two terms of its one row for the two keys.
            uint64_t sc[4][NT][H];
            const int kg = (g >> 1) + 4 * (g & 1);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                float acc[NT][G][4];
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    const uint8_t* rec = kt + gr * (int)kQ4Record + (16 * c + kg) * 32 + 8 * t;
                    const uint2 w0 = *reinterpret_cast<const uint2*>(rec), w1 = *reinterpret_cast<const uint2*>(rec + 8 * 32);
#pragma unroll
                    for (int st = 0; st < 4; st++) {
                        const uint32_t u0 = st < 2 ? w0.x : w0.y, u1 = st < 2 ? w1.x : w1.y;
                        const int i0 = 2 * (st % 2);
                        uint32_t a[4];
                        if constexpr (kTwo) {
                            a[0] = dequant(u0, i0, magic), a[1] = dequant(u1, i0, magic);
                            a[2] = dequant(u0, i0 + 1, magic), a[3] = dequant(u1, i0 + 1, magic);
                        } else {
                            a[0] = biased(u0, i0, magic), a[1] = biased(u1, i0, magic);
                            a[2] = biased(u0, i0 + 1, magic), a[3] = biased(u1, i0 + 1, magic);
                        }
#pragma unroll
                        for (int x = 0; x < NT; x++) {
                            if (st == 0) mma16816_from(acc[x][gr], a, qf[x][gr][0], start[x][gr]);
                            else mma16816(acc[x][gr], a, qf[x][gr][st]);
                        }
                    }
                }
#pragma unroll
                for (int gr = 0; gr < G; gr++) {
                    const uint32_t sw = *reinterpret_cast<const uint32_t*>(kt + gr * (int)kQ4Record + kQ4Quants + (16 * c + 2 * g) * 2);
                    const float d0 = lo_f(sw), d1 = hi_f(sw);
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        const float (&y)[4] = acc[x][gr];
                        if constexpr (kTwo) {
                            const uint64_t d = f2(d0, d1), both = f2(y[0] + y[1], y[2] + y[3]);
                            if (gr == 0) sc[c][x][0] = f2mul(d, both);
                            else f2fma(sc[c][x][0], d, both);
                        } else {
                            const uint64_t first = f2(y[0], y[1]), second = f2(y[2], y[3]);
                            if (gr == 0) sc[c][x][0] = f2mul(f2(d0, d0), first), sc[c][x][H - 1] = f2mul(f2(d1, d1), second);
                            else f2fma(sc[c][x][0], f2(d0, d0), first), f2fma(sc[c][x][H - 1], f2(d1, d1), second);
                        }
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int x = 0; x < NT; x++)
#pragma unroll
                        for (int u = 0; u < H; u++) {
                            float2 v = f2split(sc[c][x][u]);
                            const int k0 = key0 + 16 * c + kg + (kTwo ? 0 : 8 * u), k1 = kTwo ? k0 + 8 : k0;
                            if (k0 < lo[x][0] || k0 >= hi[x][0]) v.x = kNegInf;
                            if (k1 < lo[x][H - 1] || k1 >= hi[x][H - 1]) v.y = kNegInf;
                            sc[c][x][u] = f2(v.x, v.y);
                        }
            }
            // ---- the rows' maxima, in log2 units; NaN stays NaN ---------------------------------------
            float mx[NT][H];
            bool move[NT][H];
            bool any = false;
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int h = 0; h < H; h++) {
                    float v[8];
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const float2 y = f2split(sc[c][x][kTwo ? 0 : u]);
                            v[2 * c + u] = kTwo ? (u ? y.y : y.x) : (h ? y.y : y.x);
                        }
                    float y = max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], v[7]));
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) {
                        const float other = __shfl_xor_sync(0xffffffffu, y, w);
                        y = max3(y, other, other);
                    }
                    y *= p.scale2;
                    mx[x][h] = y;
                    move[x][h] = y != kNegInf && !(y <= m[x][h] + kLazy);
                    any = any || move[x][h];
                }
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                for (int x = 0; x < NT; x++) {
                    float f[2];
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        f[h] = !move[x][h] ? 1.0f : m[x][h] == kNegInf ? 0.0f : ex2(m[x][h] - mx[x][h]);
                        if (move[x][h]) m[x][h] = fmaf(mx[x][h], 0.0f, mx[x][h]);  // (+inf becomes NaN)
                    }
                    if (kTwo) f[1] = f[0];
                    l2[x] = f2mul(l2[x], f2(f[0], f[1]));
#pragma unroll
                    for (int gr = 0; gr < G; gr++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[x][gr][j][e] *= f[e % 2];
                }
            }
            // ---- weights, and O^T += V^T P^T ----------------------------------------------------------------
            uint64_t ref[NT];
            const uint64_t scale = f2(p.scale2, p.scale2);
#pragma unroll
            for (int x = 0; x < NT; x++) {
                float r[2];
#pragma unroll
                for (int h = 0; h < H; h++) r[h] = m[x][h] == kNegInf ? 0.0f : -(m[x][h] + kOffset);
                if (kTwo) r[1] = r[0];
                ref[x] = f2(r[0], r[1]);
            }
            auto weigh = [&](auto all) {
                constexpr bool WHOLE = decltype(all)::value;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint64_t w[NT][H];
#pragma unroll
                    for (int x = 0; x < NT; x++)
#pragma unroll
                        for (int u = 0; u < H; u++) {
                            uint64_t y = ref[x];
                            f2fma(y, sc[c][x][u], scale);
                            const float2 z = f2split(y);
                            w[x][u] = f2(ex2(z.x), ex2(z.y));
                            l2[x] = f2add(l2[x], w[x][u]);
                        }
#pragma unroll
                    for (int gr = 0; gr < G; gr++) {
                        const uint8_t* rec = vt + gr * (int)kQ4Record;
                        const uint32_t sw = *reinterpret_cast<const uint32_t*>(rec + kQ4Quants + (16 * c + 2 * g) * 2);
                        const float d0 = lo_f(sw), d1 = hi_f(sw);
                        uint32_t b[NT][2];
#pragma unroll
                        for (int x = 0; x < NT; x++) {
                            // the weights of keys kg and kg + 8, as rows of 8 x 8 matrices whose transposes are operands
                            uint32_t k0, k1;
                            if constexpr (kTwo) {
                                float2 v = f2split(f2mul(w[x][0], f2(d0, d1)));
                                if constexpr (!WHOLE) {  // a weight of nothing keeps out whatever the row holds
                                    const float2 z = f2split(w[x][0]);
                                    if (z.x == 0.0f) v.x = 0.0f;
                                    if (z.y == 0.0f) v.y = 0.0f;
                                }
                                const uint32_t hi = pack_bf16(v.x, v.y), lo = pack_bf16(v.x - lo_f(hi), v.y - hi_f(hi));
                                k0 = __byte_perm(hi, lo, 0x5410);
                                k1 = __byte_perm(hi, lo, 0x7632);
                            } else {
                                float2 v0 = f2split(f2mul(w[x][0], f2(d0, d0))), v1 = f2split(f2mul(w[x][H - 1], f2(d1, d1)));
                                if constexpr (!WHOLE) {
                                    const float2 z0 = f2split(w[x][0]), z1 = f2split(w[x][H - 1]);
                                    if (z0.x == 0.0f) v0.x = 0.0f;
                                    if (z0.y == 0.0f) v0.y = 0.0f;
                                    if (z1.x == 0.0f) v1.x = 0.0f;
                                    if (z1.y == 0.0f) v1.y = 0.0f;
                                }
                                k0 = pack_bf16(v0.x, v0.y);
                                k1 = pack_bf16(v1.x, v1.y);
                            }
                            b[x][0] = transposed(k0);
                            b[x][1] = transposed(k1);
                        }
                        // lane g's word of a key: columns 8 g .. 8 g + 7 of the block; two keys' halves side by side
                        uint32_t v[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] = *reinterpret_cast<const uint32_t*>(rec + (16 * c + t + 4 * e) * 32 + 4 * g);
                        const uint32_t h0[2] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[0], v[1], 0x7632)};
                        const uint32_t h1[2] = {__byte_perm(v[2], v[3], 0x5410), __byte_perm(v[2], v[3], 0x7632)};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int i0 = 2 * (j % 2);
                            const uint32_t a[4] = {dequant(h0[j / 2], i0, magic), dequant(h0[j / 2], i0 + 1, magic),
                                                   dequant(h1[j / 2], i0, magic), dequant(h1[j / 2], i0 + 1, magic)};
#pragma unroll
                            for (int x = 0; x < NT; x++) mma16816(o[x][gr][j], a, b[x]);
                        }
                    }
                }
            };
            if (whole) weigh(std::true_type{});
            else weigh(std::false_type{});
            __syncwarp();  // all lanes have read the stage
            if (lane == 0 && i + kStages < mine) {
                fence_proxy_async();  // its last reads come before the copy that overwrites it
                load(i + kStages);
            }
        }
        filled += (uint32_t)mine;

        // ---- the warps' results, merged --------------------------------------------------------------------
        __syncthreads();  // the rings are free
        float* so = reinterpret_cast<float*>(smem);  // [warp][16 rows][kLd]
        float* sm = so + kWarps * 16 * S::kLd;       // [warp][16][2]: m, l
#pragma unroll
        for (int x = 0; x < NT; x++) {
            float2 sum = f2split(l2[x]);
            if (kTwo) sum.x += sum.y;
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                sum.x += __shfl_xor_sync(0xffffffffu, sum.x, w);
                sum.y += __shfl_xor_sync(0xffffffffu, sum.y, w);
            }
#pragma unroll
            for (int h = 0; h < H; h++) {
                const int r = warp * 16 + row_of(x, h);
                float* row = so + r * S::kLd;
#pragma unroll
                for (int gr = 0; gr < G; gr++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float (&y)[4] = o[x][gr][j];
                        *reinterpret_cast<float2*>(row + 64 * gr + 8 * g + 2 * j) =
                            kTwo ? make_float2(y[0] + y[1], y[2] + y[3]) : make_float2(y[h], y[2 + h]);
                    }
                if (g == 0) {
                    sm[r * 2] = m[x][h];
                    sm[r * 2 + 1] = h ? sum.y : sum.x;
                }
            }
        }
        __syncthreads();
        const bool whole_block = count == all_units;
        // This share's place among the partial results: the first of the CTA's two if it begins with the CTA's
        // own share, else the second (a share is cut at its two ends only).
        const uint64_t begin = units * blockIdx.x / grid;
        float* part = p.partial + (((uint64_t)blockIdx.x * p.a.kv_head_count + kvh) * 2 + (pos == begin ? 0 : 1)) * kPart;
        auto row_out = [&](int r) {
            return out + ((uint64_t)(seq.q_start + (uint32_t)((row0 + r) / (int)p.group)) * p.a.head_count + kvh * p.group +
                          (uint32_t)((row0 + r) % (int)p.group)) * D;
        };
        for (int e = threadIdx.x; e < R * (D / 4); e += kThreads) {
            const int r = e / (D / 4), c = 4 * (e % (D / 4));
            if (row0 + r >= rows) break;
            float mm = kNegInf;
#pragma unroll
            for (int w = 0; w < kWarps; w += 2) mm = max3(mm, sm[(w * 16 + r) * 2], sm[((w + 1) * 16 + r) * 2]);
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
            if (whole_block) {
                const float inv = mm == kNegInf ? 0.0f : 1.0f / ll;
                T* dst = row_out(r) + c;
#pragma unroll
                for (int i = 0; i < 4; i++) dst[i] = from_f32<T>(acc[i] * inv);
            } else {
                float* dst = part + r * (D + 2);
                *reinterpret_cast<float2*>(dst + c) = make_float2(acc[0], acc[1]);
                *reinterpret_cast<float2*>(dst + c + 2) = make_float2(acc[2], acc[3]);
                if (c == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mm, ll);
            }
        }
        if (!whole_block) {
            // ---- the shares of a row block, merged by the CTA that finishes last --------------------------
            const uint64_t block_end = block_begin + all_units;
            auto owner = [&](uint64_t unit) { return ((unit + 1) * grid - 1) / units; };  // the CTA a unit falls to
            const uint64_t cta0 = owner(block_begin), cta1 = owner(block_end - 1);
            const uint32_t shares = (uint32_t)(cta1 - cta0 + 1);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned* counter = p.counters + cta0 * p.a.kv_head_count + kvh;
                s_last = atomicAdd(counter, 1u) == shares - 1;
                if (s_last) *counter = 0u;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                const uint64_t next = p.a.kv_head_count * 2 * (uint64_t)kPart;
                const bool head = units * cta0 / grid == block_begin;  // the first share begins its CTA's
                const float* parts = p.partial + (cta0 * p.a.kv_head_count + kvh) * 2 * kPart;
                auto share = [&](uint32_t i) { return parts + i * next + (i == 0 && !head ? kPart : 0); };
                // Four columns of a row per thread, the shares taken in order, eight loads ahead; a running maximum
                // as in the main loop.
                for (int e = threadIdx.x; e < R * (D / 4); e += kThreads) {
                    const int r = e / (D / 4), c = 4 * (e % (D / 4));
                    if (row0 + r >= rows) break;
                    float mm = kNegInf, ll = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (uint32_t i0 = 0; i0 < shares; i0 += 8) {
                        float2 ml[8], v0[8], v1[8];
#pragma unroll
                        for (uint32_t u = 0; u < 8; u++) {
                            const float* q = share(min(i0 + u, shares - 1)) + r * (D + 2);
                            ml[u] = __ldcg(reinterpret_cast<const float2*>(q + D));
                            v0[u] = __ldcg(reinterpret_cast<const float2*>(q + c));
                            v1[u] = __ldcg(reinterpret_cast<const float2*>(q + c + 2));
                        }
#pragma unroll
                        for (uint32_t u = 0; u < 8; u++) {
                            if (i0 + u >= shares || ml[u].x == kNegInf) continue;
                            const float m_new = max3(mm, ml[u].x, ml[u].x);
                            const float f = mm == kNegInf ? 0.0f : ex2(mm - m_new), w = ex2(ml[u].x - m_new);
                            mm = m_new;
                            ll = fmaf(w, ml[u].y, ll * f);
                            y[0] = fmaf(w, v0[u].x, y[0] * f);
                            y[1] = fmaf(w, v0[u].y, y[1] * f);
                            y[2] = fmaf(w, v1[u].x, y[2] * f);
                            y[3] = fmaf(w, v1[u].y, y[3] * f);
                        }
                    }
                    const float inv = mm == kNegInf ? 0.0f : 1.0f / ll;
                    T* dst = row_out(r) + c;
#pragma unroll
                    for (int i = 0; i < 4; i++) dst[i] = from_f32<T>(y[i] * inv);
                }
            }
        }
        pos += count;
        at += count;
        __syncthreads();  // the merge's shared memory becomes rings again
    }
    if (failed) {
        // No copy is under way when the CTA leaves: one more wait for those it had asked for.
        for (int i = 0; i < kStages; i++)
            (void)mbar_wait(smem_u32(&bars[warp][(missing + i) % kStages]), ((missing + i) / kStages) & 1u);
        if (lane == 0) atomicExch(p.error, 1);
    }
}

template <typename T, int D, int NT>
mg_status launch(Device* d, const k::PackedAttentionArgs& a) {
    using S = Q4Shape<D>;
    constexpr int R = (std::is_same<T, __nv_bfloat16>::value ? 8 : 4) * NT;
    static bool configured[64] = {false};
    if (!configured[d->ordinal & 63]) {
        MG_CUDA(cudaFuncSetAttribute(attention_q4_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
                "configuring the 4-bit attention kernel");
        configured[d->ordinal & 63] = true;
    }
    Q4Params p;
    p.a = a;
    p.group = (uint32_t)(a.head_count / a.kv_head_count);
    p.scale2 = a.scale * 1.4426950408889634f;
    p.counters = d->counters;
    p.error = d->flags + 2;
    uint64_t units = 0, most = 0;  // now, and with a captured step's largest advance
    for (const SeqRow& r : a.host->rows) {
        const uint64_t blocks = ((uint64_t)r.q_count * p.group + R - 1) / R;
        auto tiles = [&](uint64_t keys) { return kBlockCost + (r.k_start + keys + 63) / 64 - r.k_start / 64; };
        units += blocks * tiles(r.k_count);
        most += blocks * tiles(r.k_count + a.max_step);
    }
    p.units = units;
    if (a.kv_head_count > 65535) return fail(MG_SHAPE_UNSUPPORTED, "attention kv_head_count exceeds the launch grid");
    // One wave of CTAs, each with kLeastShare at the least.
    const uint64_t wave = std::max<uint64_t>(1, (uint64_t)d->sm_count * (NT == 1 ? kPerSm : 2) / a.kv_head_count);
    const uint64_t shares = std::max<uint64_t>(1, std::min(wave, (most + kLeastShare - 1) / kLeastShare));
    MG_TRY(scratch(d, 9, shares * a.kv_head_count * 2 * R * (D + 2) * sizeof(float), (void**)&p.partial));
    enqueue(d, attention_q4_kernel<T, D, NT>, dim3((unsigned)shares, (unsigned)a.kv_head_count), kThreads, S::kSmem, p);
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
        // Two column tiles where a sequence has more score rows than one holds: its keys are then read and made
        // operands half as often.
        const uint64_t rows = a.host->max_queries * (a.head_count / a.kv_head_count);
        if (rows <= (std::is_same<T, __nv_bfloat16>::value ? 8 : 4)) return a.head_dim == 64 ? launch<T, 64, 1>(d, a) : launch<T, 128, 1>(d, a);
        return a.head_dim == 64 ? launch<T, 64, 2>(d, a) : launch<T, 128, 2>(d, a);
    });
}

}  // namespace k
}  // namespace mg
