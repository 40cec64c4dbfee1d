// Attention of packed sequences on the 5th-generation tensor cores: head dimensions 64 and 128, f32,
// bfloat16 and f16.
//
// A CTA serves 256 query rows of one sequence as two 128-row tiles that share every tile of keys and
// values it loads.  A row is one (token, head): where the heads that share a key/value head are a
// multiple of a power of two, that many heads of a token are neighbouring rows (grouped heads read
// each key once, and short prompts fill their tiles).  Warp 0 loads with TMA, warp 1 issues the MMAs,
// warps 2 and 3 look after the values of tiles that are not wholly visible, warps 4-7 (tile 0) and
// 8-11 (tile 1) run the softmax, one row per thread.  While one tile's softmax runs, the tensor cores
// have the other tile's products.
//
// S = Q K^T goes to tensor memory; the softmax writes its weights P as 16-bit values over the scores it
// has read, and O += P V reads P from there.  The weights are 2^(s - m - offset) with a reference m that
// moves only when a tile's maximum passes it by more than 2^kLazy; O and the sum are then rescaled.
// The offset (2^40 for weights with f32's exponent range) keeps O below the largest |v|
// however many keys are summed, so large finite values cannot overflow the sum.
//
// The tensor cores add into their accumulators by cutting digits off, not by rounding, so that every sum of 16 products
// takes an output some 2^-24 of itself towards zero: 5e-9 a key, 2e-4 after 32768 keys.  After kKeysSummed keys O is
// therefore added to sums in memory, in f32, and starts again from zero: 1024 f32 queries over 131072 keys are 1e-5 off
// instead of 8e-4, for 3 to 5 % of the time of long rows (one f32 prompt of 8192 tokens, 32 heads, 1335 -> 1399 us).
//
// f32 operands are two bfloat16 terms each, hi + lo, and three products: lo hi + hi lo + hi hi; K and V
// are split by a pass of their own into a workspace of the sequences' rows one after another, a query
// row by the thread that owns it.
//
// Masks: scores of keys a row must not see become -inf.  A weight of zero does not keep out a NaN or an
// infinity in V, though, so in tiles that some row sees only in part the value rows that no row sees
// are zeroed in shared memory, and if a remaining one is not finite the CTA's rows are computed again
// one by one at the end.
//
// Few rows over many keys: the keys are split over CTAs, whose parts a second kernel joins.
//
// The roundings to 16 bits are what the tensor cores' rate costs: weights of bfloat16 leave outputs 2.0e-3 off, of
// which their own rounding is 1.6e-3, and two terms of f32 operands 6e-6, where f32 arithmetic has 4e-7.
//
// Causal, heads of 128: ten prompts of 1 to 8192 tokens, 32 heads over 8, bfloat16, 719 to 739 us, 1.02 to 1.05
// PFLOP/s, the tensor pipe busy for 58 % (the chain scores, softmax, product of two tiles sets the pace); 4 x 2048 tokens,
// 32 heads, f32, 557 to 569 us with the split, 242 to 247 TFLOP/s, three times that on the tensor cores.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attention_packed.cuh"
#include "sm100.cuh"

namespace mg {
namespace {

using namespace sm100;

constexpr int kRows = 128;      // rows of a query tile (MMA M)
constexpr int kThreads = 384;   // 12 warps
// Registers of a thread of warps 0-3 and of warps 4-11; their sum over the block must not pass what it
// is launched with (checked before the first launch).
constexpr int kFewRegs = 80, kManyRegs = 200;
constexpr uint64_t kPartKeys = 512;  // keys that a CTA of split keys has at the least

template <typename T, int D>
struct Shape {
    static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kKeys = kTerms == 2 ? 64 : 128;   // keys of a tile
    static constexpr int kScores = 128 / kKeys;            // score buffers of a query tile
    static constexpr int kParts = kKeys / 32;              // weights of a tile are handed over 32 keys at a time
    // Keys that O sums in tensor memory before it is taken out: up to 1e-5 of it are lost, for the 16-bit types 8e-5, a
    // third of f16's own rounding (a bfloat16 prompt of 32768 tokens 7.08 -> 7.27 ms).
    static constexpr int kKeysSummed = kTerms == 2 ? 2048 : 16384;
    static constexpr int kTilesSummed = kKeysSummed / kKeys;
    static constexpr int kQAtom = kRows * 128;             // [128 rows][64 columns], 128-byte swizzle
    static constexpr int kQTerm = (D / 64) * kQAtom;
    static constexpr int kQTile = kTerms * kQTerm;
    static constexpr int kAtom = kKeys * 128;              // [keys][64 columns]
    static constexpr int kTerm = (D / 64) * kAtom;
    static constexpr int kStage = kTerms * kTerm;          // one tile of K, or of V
    static constexpr int kKStages = 2;
    static constexpr int kVStages = kTerms == 2 && D == 128 ? 1 : 2;
    static constexpr int kOffK = 2 * kQTile;
    static constexpr int kOffV = kOffK + kKStages * kStage;
    static constexpr int kSmem = kOffV + kVStages * kStage + 1024;
    static constexpr uint32_t kColO = 256;                 // tensor memory: scores of tile t at 128 t, O at 256 + D t
};

struct Params {
    k::PackedAttentionArgs a;
    uint32_t pack, pack_log2;   // heads of a token that are neighbouring rows (a power of two)
    uint32_t groups;            // sets of `pack` heads
    uint32_t tokens;            // of a CTA: 256 / pack
    float scale2;               // scores to log2 units
    int* error;
    // Keys split over several CTAs: the parts, and for CTA c (of part c % parts) and its row r the mean of the
    // part's values at means + (c * live + r) * D, the reference and the sum at stats[c * live + r], and whether
    // the CTA met a value that asks for its rows to be computed again.
    uint32_t parts, live;
    float* means;
    float2* stats;
    uint32_t* again;
    // O taken out of tensor memory (where a row has more than kKeysSummed keys): column c of the row of warp
    // 4 + w, lane l of CTA i at ((i * 8 + w) * (D + 1) + c) * 32 + l, and its reference as column D.
    float* summed;
};

// Two values as a packed pair of the 16-bit type, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// Two values as two bfloat16 terms each, packed; a finite value that would round to infinity is held at
// the largest bfloat16, so that its lo term has the rest.
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& lo) {
    constexpr float kMost = 3.3895313892515355e38f;
    const uint32_t hi = pack16<__nv_bfloat16>(fminf(fmaxf(x, -kMost), kMost), fminf(fmaxf(y, -kMost), kMost));
    lo = pack16<__nv_bfloat16>(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
    return hi;
}

// The sequences' f32 rows of K (blockIdx.y 0) and V (1), one sequence after another, as their two terms:
// ws holds K's hi terms, its lo terms, V's hi and V's lo, `stride` rows each.  Streaming, 4 bytes read and 4
// written per value; kSplitPieces pieces of 16 bytes per thread, all loaded before the first is split
// (4 x 2048 rows of 4096 of both: about 95 us, 5.7 TB/s; row by row with a division each 107).
constexpr int kSplitThreads = 256, kSplitPieces = 4;
__global__ void __launch_bounds__(kSplitThreads) split_rows_kernel(k::SeqTable t, const float* __restrict__ keys_src,
                                                                   const float* __restrict__ values_src, uint16_t* __restrict__ ws,
                                                                   uint64_t keys, uint64_t stride, uint32_t vecs) {
    pdl_enter();
    const uint32_t step = t.step ? (uint32_t)*t.step : 0;
    keys += (uint64_t)step * t.count;
    const uint64_t first = (uint64_t)blockIdx.x * (kSplitPieces * kSplitThreads) + threadIdx.x;
    if (first >= keys * vecs) return;
    const float4* src = reinterpret_cast<const float4*>(blockIdx.y ? values_src : keys_src);
    uint2* hi = reinterpret_cast<uint2*>(ws) + (blockIdx.y ? 2 * stride * vecs : 0);
    uint2* lo = hi + stride * vecs;
    Places<kSplitThreads> at(first, vecs);
    auto prefix = [&](uint32_t s) { return __ldg(t.key_prefix + s) + step * s; };
    uint32_t a = 0, from = 0, to = 0, k_start = 0;  // the sequence of a row: its packed rows [from, to)
    float4 x[kSplitPieces];
#pragma unroll
    for (int j = 0; j < kSplitPieces; j++) {
        const uint32_t g = (uint32_t)min(at.i, keys - 1);  // (past the last row: read, not written)
        if (j == 0 || g >= to) {
            a = 0;
            uint32_t b = t.count;  // the last sequence whose keys start at or before g
            while (b - a > 1) {
                const uint32_t mid = (a + b) / 2;
                if (prefix(mid) <= g) a = mid;
                else b = mid;
            }
            from = prefix(a);
            to = a + 1 < t.count ? prefix(a + 1) : (uint32_t)keys;
            k_start = __ldg(&t.rows[a].k_start);
        }
        x[j] = __ldg(src + (uint64_t)(k_start + (g - from)) * vecs + at.c);
        at.next();
    }
#pragma unroll
    for (int j = 0; j < kSplitPieces; j++) {
        const uint64_t w = first + j * kSplitThreads;
        if (w >= keys * vecs) return;
        uint2 h, l;
        h.x = split2(x[j].x, x[j].y, l.x);
        h.y = split2(x[j].z, x[j].w, l.y);
        hi[w] = h;
        lo[w] = l;
    }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Descriptor of a 16-bit operand whose rows (128 bytes, 64 consecutive values of the N dimension) are
// the contraction: 8-row groups 1024 bytes apart, the next 64 of N `next` bytes further.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr, uint32_t next) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((next >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// kind::f16 with an f32 accumulator: operand format 0 f16, 1 bfloat16; B with N along its rows.
constexpr uint32_t idesc(int format, int m, int n, bool b_mn) {
    return (1u << 4) | ((uint32_t)format << 7) | ((uint32_t)format << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// 1 in one lane of the warp.
__device__ __forceinline__ uint32_t elected() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r;
}

// The MMAs and the commit, carried out by the lane whose `lead` is 1 (all lanes of the warp call them
// with the same other arguments).
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(lead)
        : "memory");
}

// The sequence and the tokens of work item `item` (by all lanes of a warp).  Sequences with the most keys
// first, and a sequence's last (heaviest) tokens first: CTAs start in grid order, so light ones fill the last wave.
__device__ __forceinline__ void item_place(const Params& p, uint32_t item, uint32_t& seq, uint32_t& place) {
    auto tiles = [&](uint32_t n) { return (n + p.tokens - 1) / p.tokens; };
    const bool found = find_item(p.a.table, item, tiles, seq, place);
    place = found ? tiles(__ldg(&p.a.table.ordered[seq].q_count)) - 1 - place : 0;
    seq = found ? seq : 0xffffffffu;
}

template <typename T, int D>
__device__ __noinline__ void recompute_rows(const Params& p, const SeqRow& s, uint32_t tok0, uint32_t head0) {
    extern __shared__ uint8_t smem_raw[];
    float* q_shared = reinterpret_cast<float*>(smem_raw + (-smem_u32(smem_raw) & 15u));  // (all copies and MMAs are done)
    const int lane = threadIdx.x % 32;
    const uint64_t w = p.a.kv_head_count * D;
    const PlainRows<T> kr{(const T*)p.a.k, w, true}, vr{(const T*)p.a.v, w, true};
    for (uint32_t r = threadIdx.x / 32 - 4; r < 2 * kRows; r += 8) {  // (by warps 4-11)
        const uint32_t tok = tok0 + (r >> p.pack_log2);
        if (tok >= s.q_count) break;
        attention_row<T, PlainRows<T>, D / 32, 1>(p.a, kr, vr, s, s.q_start + tok, head0 + (r & (p.pack - 1)), lane,
                                               q_shared + (threadIdx.x / 32 - 4) * D);
    }
}

// SPLIT: the CTA takes one of p.parts equal parts of its rows' tiles of keys, and leaves the part's means and
// statistics to merge_parts_kernel.
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    attention_packed_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                               const __grid_constant__ CUtensorMap map_klo, const __grid_constant__ CUtensorMap map_v,
                               const __grid_constant__ CUtensorMap map_vlo, const __grid_constant__ Params p) {
    using S = Shape<T, D>;
    constexpr int KV = S::kKeys;
    constexpr bool kTwo = S::kTerms == 2;
    constexpr int kFormat = std::is_same<T, __half>::value ? 0 : 1;
    // f16 weights have no exponents to spare: they may reach 2^15, and vanish below 2^-24
    constexpr float kLazy = kFormat == 0 ? 7.0f : 8.0f;
    constexpr float kOffset = kFormat == 0 ? -8.0f : 40.0f;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[28];
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t s_seq, s_place, s_poison;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    const uint32_t b0 = smem_u32(bars);
    const uint32_t q_full = b0;
    auto k_full = [&](int s) { return b0 + 8 + 8u * (uint32_t)s; };
    auto k_empty = [&](int s) { return b0 + 24 + 8u * (uint32_t)s; };
    auto v_full = [&](int s) { return b0 + 40 + 8u * (uint32_t)s; };
    auto v_ready = [&](int s) { return b0 + 56 + 8u * (uint32_t)s; };
    auto v_empty = [&](int s) { return b0 + 72 + 8u * (uint32_t)s; };
    auto s_full = [&](int t, int b) { return b0 + 88 + 8u * (uint32_t)(2 * t + b); };
    auto pv_done = [&](int t, int b) { return b0 + 120 + 8u * (uint32_t)(2 * t + b); };
    // (kScores * kParts = 4 parts of a query tile at a time)
    auto p_full = [&](int t, int b, int part) { return b0 + 152 + 8u * (uint32_t)(4 * t + b * S::kParts + part); };
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x / 32, 0), lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 27; i++) {
            const uint32_t bar = b0 + 8u * (uint32_t)i;
            // P: the tile's four softmax warps; Q: all eight where they split it; V: its two warps
            const bool is_p = bar >= p_full(0, 0, 0), is_v = bar >= v_ready(0) && bar <= v_ready(1);
            mbar_init(bar, is_p ? 4 : is_v ? 2 : bar == q_full && kTwo ? 8 : 1);
        }
        s_poison = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    if (warp == 0) {
        // (the table was written by copies, which a launch never overtakes)
        uint32_t seq, place;
        item_place(p, (SPLIT ? blockIdx.x / p.parts : blockIdx.x) / p.groups, seq, place);
        if (lane == 0) {
            s_seq = seq;
            s_place = place;
        }
    }
    pdl_enter();  // after the TMEM allocation, as every tensor-memory kernel here does
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const bool any = s_seq != 0xffffffffu;
    const SeqRow seq = any ? seq_load(p.a.table, p.a.table.ordered, s_seq) : SeqRow{0, 0, 0, 0};
    const uint32_t tok0 = s_place * p.tokens, head0 = ((SPLIT ? blockIdx.x / p.parts : blockIdx.x) % p.groups) * p.pack;
    const int kvh = (int)(head0 / (uint32_t)(p.a.head_count / p.a.kv_head_count));
    const int m_keys = (int)seq.k_count, shift = m_keys - (int)seq.q_count;  // token i stands at shift + i
    const int window = p.a.window >= 0 && p.a.window < 0x7fffffff ? (int)p.a.window : -1;
    // first row of K and V: f32 terms lie in the workspace, packed
    int key_row0 = (int)seq.k_start;
    if (kTwo && any) {
        const uint32_t id = __ldg(p.a.table.order + s_seq);
        key_row0 = (int)(__ldg(p.a.table.key_prefix + id) + (p.a.table.step ? (uint32_t)*p.a.table.step * id : 0u));
    }
    // Keys [kv0, ...) the CTA reads, and the tiles of them each query tile reads.
    const int live_tokens = min((int)p.tokens, (int)seq.q_count - (int)tok0);
    int kv0 = window > 0 ? max(0, shift + (int)tok0 - window + 1) : 0;
    int n_t[2], hi_cta = 0, kv_end = 0x7fffffff;
    if constexpr (SPLIT) {
        const int hi = p.a.causal ? min(m_keys, shift + (int)tok0 + live_tokens) : m_keys;
        const int tiles = hi > kv0 ? (hi - kv0 + KV - 1) / KV : 0, part = (int)(blockIdx.x % p.parts);
        const int each = (tiles + (int)p.parts - 1) / (int)p.parts;
        kv_end = kv0 + min(tiles, (part + 1) * each) * KV;
        kv0 += min(tiles, part * each) * KV;
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int first = t * (int)p.tokens / 2;  // (a tile holds whole tokens: pack <= 128)
        const int last = min(live_tokens, first + (int)p.tokens / 2) - 1;
        const int hi = last < first ? 0 : min(kv_end, p.a.causal ? min(m_keys, shift + (int)tok0 + last + 1) : m_keys);
        n_t[t] = hi > kv0 ? (hi - kv0 + KV - 1) / KV : 0;
        hi_cta = max(hi_cta, hi);
    }
    const int n_kv = max(n_t[0], n_t[1]);
    // Keys every row of the CTA sees.
    const int all_lo = window > 0 ? max(0, shift + (int)tok0 + live_tokens - window) : 0;
    const int all_hi = p.a.causal ? min(m_keys, shift + (int)tok0 + 1) : m_keys;

    // The softmax threads hold a row of scores each: they take registers from the other warps.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (warp == 0) {
            // ---- TMA producer ----------------------------------------------------------------------
            if (lane == 0 && n_kv > 0) {
                if constexpr (!kTwo) {
                    mbar_arrive_expect_tx(q_full, 2 * S::kQTile);
                    for (int t = 0; t < 2; t++)
                        for (int a = 0; a < D / 64; a++)
                            tma_load_3d(base + t * S::kQTile + a * S::kQAtom, &map_q, q_full, a * 64, (int)head0,
                                        (int)(seq.q_start + tok0) + t * (int)p.tokens / 2);
                }
                auto load = [&](uint32_t slot, uint32_t bar, const CUtensorMap* hi, const CUtensorMap* lo, int j) {
                    mbar_arrive_expect_tx(bar, S::kStage);
                    for (int a = 0; a < D / 64; a++) {
                        const int x = kvh * D + a * 64, y = key_row0 + kv0 + j * KV;
                        tma_load_2d(slot + a * S::kAtom, hi, bar, x, y);
                        if constexpr (kTwo) tma_load_2d(slot + S::kTerm + a * S::kAtom, lo, bar, x, y);
                    }
                };
                auto load_k = [&](int j) -> bool {
                    const int s = j % S::kKStages;
                    if (j >= S::kKStages && !mbar_wait(k_empty(s), (uint32_t)(j / S::kKStages - 1) & 1u)) return false;
                    load(base + S::kOffK + s * S::kStage, k_full(s), &map_k, &map_klo, j);
                    return true;
                };
                bool ok = load_k(0);
                int k_loads = 1, v_loads = 0;
                for (int j = 0; j < n_kv && ok; j++) {
                    if (j + 1 < n_kv) {
                        ok = load_k(j + 1);
                        k_loads += ok;
                    }
                    const int s = j % S::kVStages;
                    if (ok && j >= S::kVStages) ok = mbar_wait(v_empty(s), (uint32_t)(j / S::kVStages - 1) & 1u);
                    if (ok) {
                        load(base + S::kOffV + s * S::kStage, v_full(s), &map_v, &map_vlo, j);
                        v_loads++;
                    }
                }
                // Whoever's wait may have run out, no copy is under way when the CTA leaves.
                if constexpr (!kTwo) ok = mbar_wait(q_full, 0) && ok;
                for (int j = max(0, k_loads - S::kKStages); j < k_loads; j++)
                    ok = mbar_wait(k_full(j % S::kKStages), (uint32_t)(j / S::kKStages) & 1u) && ok;
                for (int j = max(0, v_loads - S::kVStages); j < v_loads; j++)
                    ok = mbar_wait(v_full(j % S::kVStages), (uint32_t)(j / S::kVStages) & 1u) && ok;
                if (!ok) atomicExch(p.error, 1);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---- MMA issuer --------------------------------------------------------------------------
            // The whole warp walks the loop and one elected lane's instructions take effect: addresses and
            // descriptors are then the same for all lanes and stay in uniform registers.  (Issued from a
            // branch that one lane takes, each MMA cost some 60 cycles of moving them there.)
            if (n_kv > 0) {
                constexpr uint32_t idesc_s = idesc(kFormat, kRows, KV, false);
                constexpr uint32_t idesc_o = idesc(kFormat, kRows, D, true);
                const uint32_t lead = elected();
                const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
                const uint32_t n0 = (uint32_t)__shfl_sync(0xffffffffu, n_t[0], 0), n1 = (uint32_t)__shfl_sync(0xffffffffu, n_t[1], 0);
                const uint32_t n_all = max(n0, n1);
                const uint64_t dq0 = desc_k_sw128(base), dk0 = desc_k_sw128(base + S::kOffK);
                const uint64_t dv0 = desc_mn_sw128(base + S::kOffV, S::kAtom);
                // S_t(j) = Q_t K(j)^T into tile t's score buffer j % kScores
                auto issue_s = [&](uint32_t t, uint32_t j) {
                    const uint32_t tS = tm + 128u * t + (j % S::kScores) * KV;
                    const uint64_t dq = dq0 + (uint64_t)(t * (S::kQTile >> 4));
                    const uint64_t dk = dk0 + (uint64_t)((j % S::kKStages) * (S::kStage >> 4));
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint64_t q = dq + (uint64_t)(((kk / 4) * S::kQAtom + (kk % 4) * 32) >> 4);
                        const uint64_t k = dk + (uint64_t)(((kk / 4) * S::kAtom + (kk % 4) * 32) >> 4);
                        if constexpr (kTwo) {
                            mma_ss(lead, tS, q + (uint64_t)(S::kQTerm >> 4), k, idesc_s, kk > 0 ? 1u : 0u);
                            mma_ss(lead, tS, q, k + (uint64_t)(S::kTerm >> 4), idesc_s, 1u);
                            mma_ss(lead, tS, q, k, idesc_s, 1u);
                        } else {
                            mma_ss(lead, tS, q, k, idesc_s, kk > 0 ? 1u : 0u);
                        }
                    }
                    commit(lead, s_full((int)t, (int)(j % S::kScores)));
                };
                bool ok = mbar_wait(q_full, 0);
                for (uint32_t j = 0; j < S::kScores && j < n_all && ok; j++) {
                    ok = mbar_wait(k_full((int)j), 0);
                    if (!ok) break;
                    tc_fence_after();
                    if (j < n0) issue_s(0, j);
                    if (j < n1) issue_s(1, j);
                    commit(lead, k_empty((int)j));
                }
                for (uint32_t j = 0; j < n_all && ok; j++) {
                    const uint32_t vs = j % S::kVStages, jn = j + S::kScores, vp = (j / S::kVStages) & 1u;
                    ok = mbar_wait(v_full((int)vs), vp) && mbar_wait(v_ready((int)vs), vp);
                    if (ok && jn < n_all) ok = mbar_wait(k_full((int)(jn % S::kKStages)), (jn / S::kKStages) & 1u);
                    if (!ok) break;
#pragma unroll
                    for (uint32_t t = 0; t < 2; t++) {
                        if (j < (t ? n1 : n0)) {
                            // O_t += P_t(j) V(j): P from tensor memory, two values per column
                            const uint32_t tP = tm + 128u * t + (j % S::kScores) * KV;
                            const uint32_t tO = tm + S::kColO + D * t;
                            const uint64_t dv = dv0 + (uint64_t)(vs * (S::kStage >> 4));
#pragma unroll
                            for (int part = 0; part < S::kParts; part++) {
                                ok = ok && mbar_wait(p_full((int)t, (int)(j % S::kScores), part), (j / S::kScores) & 1u);
                                if (!ok) break;
                                tc_fence_after();
#pragma unroll
                                for (int k2 = 0; k2 < 2; k2++) {
                                    const int kk = 2 * part + k2;
                                    const uint64_t v = dv + (uint64_t)((kk * 2048) >> 4);
                                    const uint32_t pa = tP + (uint32_t)kk * 8;
                                    const uint32_t acc = (j % S::kTilesSummed > 0 || kk > 0) ? 1u : 0u;
                                    if constexpr (kTwo) {
                                        mma_ts(lead, tO, pa + KV / 2, v, idesc_o, acc);
                                        mma_ts(lead, tO, pa, v + (uint64_t)(S::kTerm >> 4), idesc_o, 1u);
                                        mma_ts(lead, tO, pa, v, idesc_o, 1u);
                                    } else {
                                        mma_ts(lead, tO, pa, v, idesc_o, acc);
                                    }
                                }
                            }
                            if (!ok) break;
                            commit(lead, pv_done((int)t, (int)(j & 1)));
                        }
                        if (t == 1) commit(lead, v_empty((int)vs));
                        // With one score buffer a tile's next scores follow its own product, so that its softmax
                        // runs beside the other tile's products.  With two they are a tile ahead, and come after
                        // both products: V's only stage is then free for longer before it is needed again.
                        if (S::kScores == 1 && jn < (t ? n1 : n0)) issue_s(t, jn);
                    }
                    if (ok && S::kScores == 2) {
                        if (jn < n0) issue_s(0, jn);
                        if (jn < n1) issue_s(1, jn);
                    }
                    if (ok && jn < n_all) commit(lead, k_empty((int)(jn % S::kKStages)));
                }
                if (!ok && lane == 0) atomicExch(p.error, 1);
            }
            __syncwarp();
        } else {
            // ---- values of tiles some row sees only in part ------------------------------------------
            const int i0 = (int)threadIdx.x - 64;
            constexpr uint32_t kExponents = kFormat == 0 ? 0x7c007c00u : 0x7f807f80u, kOne = kFormat == 0 ? 0x04000400u : 0x00800080u;
            bool failed = false;
            for (int j = 0; j < n_kv && !failed; j++) {
                const int s = j % S::kVStages;
                failed = !mbar_wait(v_full(s), (uint32_t)(j / S::kVStages) & 1u);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                const int key0 = kv0 + j * KV;
                if (key0 < all_lo || key0 + KV > all_hi) {
                    uint8_t* stage = base_ptr + S::kOffV + s * S::kStage;
                    uint32_t bad = 0;
#pragma unroll 1
                    for (int r = i0; r < KV; r += 64) {
                        const bool seen = key0 + r < hi_cta;
#pragma unroll 1
                        for (int a = 0; a < S::kTerms * (D / 64); a++) {
                            uint4* row = reinterpret_cast<uint4*>(stage + a * S::kAtom + r * 128);
                            // (neighbouring lanes start in different banks)
                            if (seen) {
                                uint4 v[8];
#pragma unroll
                                for (int c = 0; c < 8; c++) v[c] = row[(c + lane) & 7];
                                // an exponent of all ones, and only that, carries into the sign's place
#pragma unroll
                                for (int c = 0; c < 8; c++)
                                    bad |= ((v[c].x & kExponents) + kOne) | ((v[c].y & kExponents) + kOne) | ((v[c].z & kExponents) + kOne) |
                                           ((v[c].w & kExponents) + kOne);
                            } else {
#pragma unroll
                                for (int c = 0; c < 8; c++) row[(c + lane) & 7] = make_uint4(0u, 0u, 0u, 0u);
                            }
                        }
                    }
                    if (bad & 0x80008000u) s_poison = 1;
                    fence_proxy_async();  // the zeros are read by tcgen05.mma
                }
                mbar_arrive_warp(v_ready(s));
            }
            if (failed && lane == 0) atomicExch(p.error, 1);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        // ---- softmax: one query row per thread ---------------------------------------------------
        const float kNegInf = __int_as_float(0xff800000);
        const int t = (warp - 4) / 4, qq = warp % 4;
        const int r = qq * 32 + lane;
        const int tile_tok0 = (int)tok0 + t * (int)p.tokens / 2;
        const int tok = tile_tok0 + (r >> p.pack_log2);
        const bool live = tok < (int)seq.q_count;
        // element offset of row i of this warp in q and out; of the sequence's last token past its end
        auto row_at = [&](int i) {
            const int rr = qq * 32 + i;
            const uint64_t token = (uint64_t)seq.q_start + (uint64_t)min(tile_tok0 + (rr >> p.pack_log2), (int)seq.q_count - 1);
            return (token * p.a.head_count + head0 + (uint32_t)(rr & (int)(p.pack - 1))) * D;
        };
        auto row_live = [&](int i) { return tile_tok0 + ((qq * 32 + i) >> p.pack_log2) < (int)seq.q_count; };
        if constexpr (kTwo) {
            if (n_kv > 0) {
                // This warp's 32 query rows as two terms in the MMA's K-major layout: 16-byte chunk c of a row
                // at position c ^ (row % 8).  Rows past the sequence repeat its last token (their outputs go
                // nowhere), so that no load hangs on a condition: a conditional load is waited for before
                // the next one starts.  One row per load, each lane D / 32 columns, sixteen rows in flight.
                constexpr int V = D / 32;
                using Vec = typename std::conditional<V == 4, float4, float2>::type;
                const float* q = (const float*)p.a.q;
                uint8_t* qt = base_ptr + t * S::kQTile;
                const int e0 = lane * V, a = e0 / 64, c = (e0 % 64) / 8, byte = (e0 % 8) * 2;
#pragma unroll 1
                for (int i0 = 0; i0 < 32; i0 += 16) {
                    Vec xv[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        xv[i] = __ldg(reinterpret_cast<const Vec*>(q + row_at(i0 + i) + lane * V));
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int rr = qq * 32 + i0 + i;
                        const int off = a * S::kQAtom + rr * 128 + ((c ^ (rr & 7)) * 16 + byte);
                        const float* xs = reinterpret_cast<const float*>(&xv[i]);
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            uint32_t lo;
                            const uint32_t hi = split2(xs[e], xs[e + 1], lo);
                            *reinterpret_cast<uint32_t*>(qt + off + 2 * e) = hi;
                            *reinterpret_cast<uint32_t*>(qt + S::kQTerm + off + 2 * e) = lo;
                        }
                    }
                }
                fence_proxy_async();  // the generic-proxy writes are read by tcgen05.mma
                mbar_arrive_warp(q_full);
            }
        }
        // Keys [row_lo, row_hi) this row sees.
        const int pos = shift + tok;
        const int row_hi = !live ? 0 : p.a.causal ? max(0, min(m_keys, pos + 1)) : m_keys;
        const int row_lo = window > 0 ? min(max(0, pos - window + 1), row_hi) : 0;
        const float sc = p.scale2;
        const uint32_t lane_base = tmem + ((uint32_t)(qq * 32) << 16);
        const uint32_t tO = lane_base + S::kColO + (uint32_t)(D * t);
        const int n = n_t[t];
        float m = kNegInf, l = 0.0f;
        auto summed = [&]() { return p.summed + ((uint64_t)blockIdx.x * 8 + (uint32_t)(warp - 4)) * ((D + 1) * 32) + lane; };
        // 2^(their reference - now's), of the values there
        auto summed_by = [&](const float* at, float now) {
            const float then = __ldcg(at + D * 32);
            return then == now ? 1.0f : ex2(then - now);
        };
        bool failed = false;
        for (int j = 0; j < n && !failed;) {
            for (const int stop = min(n, j + S::kTilesSummed); j < stop; j++) {
                failed = !mbar_wait(s_full(t, j % S::kScores), (uint32_t)(j / S::kScores) & 1u);
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                tc_fence_after();
                const uint32_t tS = lane_base + 128u * (uint32_t)t + (uint32_t)(j % S::kScores) * KV;
                float s[KV];
                const int key0 = kv0 + j * KV;
                const bool part_seen = key0 < row_lo || key0 + KV > row_hi;
#pragma unroll
                for (int c = 0; c < KV; c += 32) tmem_ld32(tS + (uint32_t)c, s + c);
                tc_wait_ld();
                if (part_seen) {
                    const int lo = row_lo - key0, hi = row_hi - key0;
#pragma unroll
                    for (int c = 0; c < KV; c++) s[c] = c >= lo && c < hi ? s[c] : kNegInf;
                }
                // the row's maximum of the raw scores (sc > 0 keeps their order), in log2 units
                float mx[4];
#pragma unroll
                for (int g = 0; g < 4; g++) mx[g] = max3(s[g], s[g + 4], s[g + 8]);
#pragma unroll
                for (int c = 12; c + 4 < KV; c += 8)
#pragma unroll
                    for (int g = 0; g < 4; g++) mx[g] = max3(mx[g], s[c + g], s[c + 4 + g]);
#pragma unroll
                for (int g = 0; g < 4; g++) mx[g] = max3(mx[g], s[KV - 4 + g], s[KV - 4 + g]);
                const float tmax = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sc;
                // the reference moves only when this tile's maximum passes it by more than kLazy; scores that are
                // NaN or +inf make it NaN, and with it all of the row
                bool move = tmax != kNegInf && !(tmax <= m + kLazy);
                float f = 1.0f;
                if (move) {
                    f = m == kNegInf ? 0.0f : ex2(m - tmax);
                    move = m != kNegInf;  // an O that holds only zero weights needs no rescale
                    m = fmaf(tmax, 0.0f, tmax);
                    l *= f;
                }
                if (j > 0 && __any_sync(0xffffffffu, move)) {
                    // O *= f, once P V(j - 1) has completed
                    failed = !mbar_wait(pv_done(t, (j - 1) & 1), (uint32_t)((j - 1) >> 1) & 1u);
                    failed = __any_sync(0xffffffffu, failed);
                    if (failed) break;
                    tc_fence_after();
                    const float g = move ? f : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        tmem_ld16(tO + (uint32_t)c, o);
                        tc_wait_ld();
                        uint32_t u[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) u[e] = __float_as_uint(o[e] * g);
                        tmem_st16(tO + (uint32_t)c, u);
                    }
                    tc_wait_st();
                }
                // (no key seen yet: every score is -inf, and weights 2^(-inf) are 0)
                const float ref = m == kNegInf ? 0.0f : -(m + kOffset);
                const uint64_t sc2 = f2(sc, sc), ref2 = f2(ref, ref);
                uint64_t sum[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
                auto hand_over = [&](int part) {
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive_warp(p_full(t, j % S::kScores, part));
                };
#pragma unroll
                for (int part = 0; part < S::kParts; part++) {
                    // 32 weights, over the scores just read
                    uint32_t h[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int c = part * 32 + 2 * e;
                        uint64_t x = ref2;
                        f2fma(x, f2(s[c], s[c + 1]), sc2);
                        const float2 y = f2split(x);
                        s[c] = ex2(y.x);
                        s[c + 1] = ex2(y.y);
                        sum[e & 1] = f2add(sum[e & 1], f2(s[c], s[c + 1]));
                        h[e] = pack16<T>(s[c], s[c + 1]);
                    }
                    if (part > 0) hand_over(part - 1);  // (the stores before it have had this part's time)
                    tmem_st16(tS + (uint32_t)(part * 16), h);
                    if constexpr (kTwo) {
                        uint32_t lo[16];
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int c = part * 32 + 2 * e;
                            lo[e] = pack16<T>(s[c] - __uint_as_float(h[e] << 16), s[c + 1] - __uint_as_float(h[e] & 0xffff0000u));
                        }
                        tmem_st16(tS + (uint32_t)(KV / 2 + part * 16), lo);
                    }
                }
                hand_over(S::kParts - 1);
                const float2 u = f2split(f2add(sum[0], sum[1]));
                l += u.x + u.y;
            }
            if (failed || j >= n) break;
            // O to memory; the next P V starts from zero
            failed = !mbar_wait(pv_done(t, (j - 1) & 1), (uint32_t)((j - 1) >> 1) & 1u);
            failed = __any_sync(0xffffffffu, failed);
            if (failed) break;
            tc_fence_after();
            float* at = summed();
            const float by = j > S::kTilesSummed ? summed_by(at, m) : 0.0f;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32], before[32];
                // (loaded the first time too, and not used: a conditional load is waited for at once)
#pragma unroll
                for (int e = 0; e < 32; e++) before[e] = __ldcg(at + (c + e) * 32);
                tmem_ld32(tO + (uint32_t)c, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e++) __stcg(at + (c + e) * 32, j > S::kTilesSummed ? fmaf(before[e], by, o[e]) : o[e]);
            }
            __stcg(at + D * 32, m);
        }
        // ---- the output row: O / l ---------------------------------------------------------------
        auto whole = [&](int c, float* o) {  // with what was taken out
            if (n <= S::kTilesSummed) return;
            const float* at = summed();
            const float by = summed_by(at, m);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = fmaf(__ldcg(at + (c + e) * 32), by, o[e]);
        };
        bool have = false;
        if (n > 0 && !failed) {
            failed = !mbar_wait(pv_done(t, (n - 1) & 1), (uint32_t)((n - 1) >> 1) & 1u);
            failed = __any_sync(0xffffffffu, failed);
            have = !failed;
        }
        if (failed) atomicExch(p.error, 1);
        if constexpr (SPLIT) {
            const uint32_t row = (uint32_t)(t * kRows + r);
            if (live) {
                const uint64_t at = (uint64_t)blockIdx.x * p.live + row;
                p.stats[at] = make_float2(have ? m : kNegInf, have ? l : 0.0f);
            }
            if (have) tc_fence_after();
            const float inv = !have || m == kNegInf ? 0.0f : 1.0f / l;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                if (have) {
                    tmem_ld32(tO + (uint32_t)c, o);  // (by the whole warp)
                    tc_wait_ld();
                    whole(c, o);
                }
                if (live) {
                    float4* dst = reinterpret_cast<float4*>(p.means + ((uint64_t)blockIdx.x * p.live + row) * D + c);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        dst[e] = have ? make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv)
                                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
        }
        T* out = (T*)p.a.out;
        constexpr int kChunks = D * (int)sizeof(T) / 16;  // 16-byte chunks per row
        constexpr int kRowsPerStore = 32 / kChunks;       // rows one warp store covers
        constexpr int N = 16 / (int)sizeof(T);
        if (!SPLIT && have) {
            // Each thread writes its row into its warp's staging area -- this tile's queries, which no MMA
            // reads once the last P V has completed -- with chunk k of row i at position k ^ i; then the
            // warp stores whole rows, 16 bytes per lane.
            tc_fence_after();
            const float inv = m == kNegInf ? 0.0f : 1.0f / l;
            uint8_t* stage = base_ptr + t * S::kQTile + qq * (32 * D * (int)sizeof(T));
            fence_proxy_async();  // after the MMAs' reads of this area, before generic writes
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                tmem_ld32(tO + (uint32_t)c, o);
                tc_wait_ld();
                whole(c, o);
#pragma unroll
                for (int e = 0; e < 32; e += N) {
                    uint4 v;
                    if constexpr (kTwo) {
                        v = make_uint4(__float_as_uint(o[e] * inv), __float_as_uint(o[e + 1] * inv), __float_as_uint(o[e + 2] * inv),
                                       __float_as_uint(o[e + 3] * inv));
                    } else {
                        v = make_uint4(pack16<T>(o[e] * inv, o[e + 1] * inv), pack16<T>(o[e + 2] * inv, o[e + 3] * inv),
                                       pack16<T>(o[e + 4] * inv, o[e + 5] * inv), pack16<T>(o[e + 6] * inv, o[e + 7] * inv));
                    }
                    *reinterpret_cast<uint4*>(stage + lane * (D * (int)sizeof(T)) + ((((c + e) / N) ^ lane) % kChunks) * 16) = v;
                }
            }
            __syncwarp();
        }
        const uint8_t* staged = base_ptr + t * S::kQTile + qq * (32 * D * (int)sizeof(T));
        const int chunk = lane % kChunks;
#pragma unroll 1
        for (int i0 = lane / kChunks; !SPLIT && i0 < 32; i0 += 4 * kRowsPerStore) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * kRowsPerStore;
                v[u] = *reinterpret_cast<const uint4*>(staged + i * (D * (int)sizeof(T)) + ((chunk ^ i) % kChunks) * 16);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * kRowsPerStore;
                if (row_live(i)) *reinterpret_cast<uint4*>(out + row_at(i) + chunk * N) = have ? v[u] : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if constexpr (SPLIT) {
        if (threadIdx.x == 0) p.again[blockIdx.x] = s_poison;
    } else {
        if (s_poison && warp >= 4) recompute_rows<T, D>(p, seq, tok0, head0);
    }
}

// The rows of one item from its parts: each part's mean by its share of the weights, one row per warp.
constexpr int kMergeWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kMergeWarps) merge_parts_kernel(const Params p) {
    __shared__ __align__(16) float q_shared[kMergeWarps][D];
    pdl_enter();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t id, place;
    item_place(p, blockIdx.x / p.groups, id, place);
    if (id == 0xffffffffu) return;
    const SeqRow seq = seq_load(p.a.table, p.a.table.ordered, id);
    const uint32_t tok0 = place * p.tokens, head0 = (blockIdx.x % p.groups) * p.pack;
    const uint32_t rows = min(p.tokens, seq.q_count - tok0) * p.pack, cta0 = blockIdx.x * p.parts;
    uint32_t again = 0;
    for (uint32_t c = lane; c < p.parts; c += 32) again |= p.again[cta0 + c];
    again = __any_sync(0xffffffffu, again);
    const uint32_t r = blockIdx.y * kMergeWarps + warp;
    if (r >= rows) return;
    const uint64_t token = seq.q_start + tok0 + (r >> p.pack_log2), head = head0 + (r & (p.pack - 1));
    if (again) {
        const uint64_t w = p.a.kv_head_count * D;
        const PlainRows<T> kr{(const T*)p.a.k, w, true}, vr{(const T*)p.a.v, w, true};
        attention_row<T, PlainRows<T>, D / 32, 4>(p.a, kr, vr, seq, token, head, lane, q_shared[warp]);
        return;
    }
    float most = __int_as_float(0xff800000), total = 0.0f, o[D / 32] = {};
    for (uint32_t c = lane; c < p.parts; c += 32) most = fmaxf(most, p.stats[(uint64_t)(cta0 + c) * p.live + r].x);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
    // (a part of a row with a NaN or +inf score has a NaN reference, and makes the row NaN)
    auto share = [&](uint32_t c) {
        const float2 ml = p.stats[(uint64_t)(cta0 + c) * p.live + r];
        return ml.y == 0.0f ? 0.0f : ml.y * exp2f(ml.x - most);
    };
    for (uint32_t c = lane; c < p.parts; c += 32) total += share(c);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
#pragma unroll 4
    for (uint32_t c = 0; c < p.parts; c++) {
        const float w = total == 0.0f ? 0.0f : share(c) / total;
#pragma unroll
        for (int i = 0; i < D / 32; i++) o[i] = fmaf(w, p.means[((uint64_t)(cta0 + c) * p.live + r) * D + lane + 32 * i], o[i]);
    }
    T* out = (T*)p.a.out + (token * p.a.head_count + head) * D;
#pragma unroll
    for (int i = 0; i < D / 32; i++) out[lane + 32 * i] = from_f32<T>(o[i]);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// A map of 16-bit values with 128-byte swizzle: boxes of 64 columns.
mg_status map_16bit(CUtensorMap* map, mg_dtype t, const void* ptr, int rank, const uint64_t* dims, const uint64_t* strides,
                    const uint32_t* box) {
    auto fn = encode_fn();
    if (!fn) return fail(MG_DRIVER_FAILED, "the driver does not provide cuTensorMapEncodeTiled");
    cuuint64_t d[3], s[2];
    cuuint32_t b[3], e[3] = {1, 1, 1};
    for (int i = 0; i < rank; i++) {
        d[i] = dims[i];
        b[i] = box[i];
        if (i > 0) s[i - 1] = strides[i - 1];
    }
    const CUresult r = fn(map, t == MG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
                          const_cast<void*>(ptr), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MG_DRIVER_FAILED, "encoding a TMA descriptor failed (CUresult %d)", (int)r);
    return MG_OK;
}

template <typename T, int D>
mg_status launch(Device* d, const k::PackedAttentionArgs& a) {
    using S = Shape<T, D>;
    static_assert(S::kSmem <= 227 * 1024 - 512, "shared memory budget");
    static bool configured[64] = {false};
    if (!configured[d->ordinal & 63]) {
        for (auto kernel : {attention_packed_tc_kernel<T, D, false>, attention_packed_tc_kernel<T, D, true>}) {
            MG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
                    "configuring the packed attention kernel");
            cudaFuncAttributes fa;
            MG_CUDA(cudaFuncGetAttributes(&fa, kernel), "configuring the packed attention kernel");
            if (fa.numRegs * kThreads < kFewRegs * 128 + kManyRegs * 256)
                return fail(MG_EXECUTION_FAILED, "the packed attention kernel was built with %d registers, too few to share out", fa.numRegs);
        }
        configured[d->ordinal & 63] = true;
    }
    Params p;
    p.a = a;
    const uint32_t group = (uint32_t)(a.head_count / a.kv_head_count);
    p.pack = 1;
    p.pack_log2 = 0;
    while (p.pack < 64 && group % (2 * p.pack) == 0) p.pack *= 2, p.pack_log2++;
    p.groups = (uint32_t)a.head_count / p.pack;
    p.tokens = 2 * kRows / p.pack;
    p.scale2 = a.scale * 1.4426950408889634f;
    p.error = d->flags + 2;
    p.parts = p.live = 0;
    p.means = nullptr;
    p.stats = nullptr;
    p.again = nullptr;
    p.summed = nullptr;
    uint64_t items = 0;
    for (const SeqRow& r : a.host->rows) items += (r.q_count + p.tokens - 1) / p.tokens;
    if (items * p.groups > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    const uint64_t width = a.kv_head_count * D;
    CUtensorMap maps[5];
    const uint32_t kv_box[2] = {64, (uint32_t)S::kKeys};
    const uint64_t kv_stride[1] = {width * 2};
    if constexpr (S::kTerms == 2) {
        const uint64_t keys = a.host->keys + a.max_step * a.host->rows.size();
        uint16_t* ws = nullptr;
        MG_TRY(scratch(d, 8, std::max<uint64_t>(keys, 1) * width * 4 * sizeof(uint16_t), (void**)&ws));
        uint16_t* terms[4];
        for (int i = 0; i < 4; i++) terms[i] = ws + (uint64_t)i * keys * width;
        if (keys) {
            const uint32_t vecs = (uint32_t)(width / 4);
            constexpr uint64_t per_block = kSplitPieces * kSplitThreads;
            const uint64_t blocks = (keys * vecs + per_block - 1) / per_block;
            if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
            enqueue(d, split_rows_kernel, dim3((unsigned)blocks, 2), kSplitThreads, 0, a.table, (const float*)a.k, (const float*)a.v, ws,
                    a.host->keys, keys, vecs);
            MG_TRY(launched(d, "packed attention split launch"));
        }
        const uint64_t dims[2] = {width, std::max<uint64_t>(keys, 1)};
        for (int i = 0; i < 4; i++) MG_TRY(map_16bit(&maps[1 + i], MG_BF16, terms[i], 2, dims, kv_stride, kv_box));
        maps[0] = maps[1];  // queries are read by the threads that own them
    } else {
        const uint64_t q_dims[3] = {(uint64_t)D, a.head_count, a.queries}, q_strides[2] = {(uint64_t)D * 2, a.head_count * D * 2};
        const uint32_t q_box[3] = {64, p.pack, (uint32_t)kRows / p.pack};
        MG_TRY(map_16bit(&maps[0], a.dtype, a.q, 3, q_dims, q_strides, q_box));
        const uint64_t dims[2] = {width, a.kv_rows};
        MG_TRY(map_16bit(&maps[1], a.dtype, a.k, 2, dims, kv_stride, kv_box));
        MG_TRY(map_16bit(&maps[3], a.dtype, a.v, 2, dims, kv_stride, kv_box));
        maps[2] = maps[1];
        maps[4] = maps[3];
    }
    // Fewer CTAs than half of the SMs: the keys are split, and a second kernel joins the parts.  One bfloat16 query
    // over 32768 keys, 32 heads over 8: 516 -> 50 us; 16 queries over 4096: 67 -> 20; four of 64 to 3000 keys:
    // 53 -> 19.  With parts of fewer than kPartKeys the join costs more than it gives (8 heads over 500 keys:
    // 11.3 us whole, 13.3 in two parts).
    const uint64_t ctas = items * p.groups;
    uint64_t longest = 0;
    for (const SeqRow& r : a.host->rows) longest = std::max<uint64_t>(longest, r.k_count + a.max_step);
    const uint64_t parts = ctas ? std::min<uint64_t>((uint64_t)d->sm_count / ctas, longest / kPartKeys) : 0;
    // A row sees at most `span` keys, a CTA's tiles as many and its tokens' more.
    const uint64_t span = a.causal && a.window >= 0 ? std::min(longest, (uint64_t)a.window + p.tokens) : longest;
    if (span > (uint64_t)S::kKeysSummed)
        MG_TRY(scratch(d, 10, ctas * std::max<uint64_t>(1, parts) * 2 * kRows * (D + 1) * sizeof(float), (void**)&p.summed));
    if (parts < 2) {
        enqueue(d, attention_packed_tc_kernel<T, D, false>, (unsigned)ctas, kThreads, S::kSmem, maps[0], maps[1], maps[2], maps[3], maps[4], p);
        return launched(d, "packed attention launch");
    }
    p.parts = (uint32_t)parts;
    p.live = (uint32_t)std::min<uint64_t>(2 * kRows, a.host->max_queries * p.pack);
    const uint64_t rows = ctas * parts * p.live;
    MG_TRY(scratch(d, 9, rows * (D * sizeof(float) + sizeof(float2)) + ctas * parts * sizeof(uint32_t), (void**)&p.means));
    p.stats = reinterpret_cast<float2*>(p.means + rows * D);
    p.again = reinterpret_cast<uint32_t*>(p.stats + rows);
    enqueue(d, attention_packed_tc_kernel<T, D, true>, (unsigned)(ctas * parts), kThreads, S::kSmem, maps[0], maps[1], maps[2], maps[3], maps[4],
            p);
    MG_TRY(launched(d, "packed attention launch"));
    enqueue(d, merge_parts_kernel<T, D>, dim3((unsigned)ctas, (p.live + kMergeWarps - 1) / kMergeWarps), 32 * kMergeWarps, 0, p);
    return launched(d, "packed attention launch");
}

}  // namespace

namespace k {

// Head dimensions of whole 64-column atoms whose scores and output fit in tensor memory, on the 16-byte
// boundaries that TMA takes; f32 also needs its split rows to be counted in 31 bits.
bool attention_packed_tc_eligible(const PackedAttentionArgs& a) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.out);
    return a.kv_dtype == a.dtype && (at & 15) == 0 && (a.head_dim == 64 || a.head_dim == 128) && a.value_dim == a.head_dim &&
           a.kv_rows > 0 && (a.dtype != MG_F32 || a.host->keys + a.max_step * a.host->rows.size() < (1ull << 31));
}

mg_status attention_packed_tc(Device* d, const PackedAttentionArgs& a) {
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        return a.head_dim == 64 ? launch<T, 64>(d, a) : launch<T, 128>(d, a);
    });
}

}  // namespace k
}  // namespace mg
