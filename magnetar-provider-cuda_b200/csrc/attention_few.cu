// Attention of packed sequences with few queries over f32 keys and values: decode steps over plain stores, head
// dimensions 64 and 128.
//
// A step reads every key and value once against a handful of operations for each, in f32 as they lie: the tensor
// cores would want them as two 16-bit terms, which a pass of its own has to write and read again.  A CTA takes one
// query of G heads that share a key/value head (each key is loaded once for them) and one of `parts` parts of
// its keys; a warp takes every fourth 32 keys of the part.  Scores: eight lanes share a key, four dimensions
// at a time, so that a load covers whole lines; each of the eight keeps the score of one key.  Values: lanes over
// the dimensions.  The output is a weighted mean of V rows throughout, which never exceeds the largest |v|;
// warps are merged in shared memory, parts by a second kernel.  Memory bounds long stores.
// One query each, 32 heads over 8 of 128: 16 sequences of 8192 keys 229 us, 4.7 TB/s (split into 16-bit terms for
// the tensor cores: 611); four 67 us (158).
#include <algorithm>
#include <type_traits>

#include "attention_packed.cuh"

namespace mg {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kCtasPerSm = 3;
constexpr int kAhead = 2;  // keys of eight lanes whose loads are under way together
constexpr uint64_t kPartKeys = 256;  // keys that a part has at the least

struct Parts {
    uint32_t parts;
    float* means;   // [item, part, head of the item][D]
    float2* stats;  // their references and sums
};

// The mean of several by their references and sums; f(i) is the i-th value.
template <int N, class F>
__device__ __forceinline__ float weighted(const float (&share)[N], F&& f) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) x = fmaf(share[i], f(i), x);
    return x;
}

template <int D, int G>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_few_kernel(const k::PackedAttentionArgs a, const Parts p) {
    constexpr int C = D / 32;  // values of a lane in an output row; 16-byte pieces of a key in a lane
    __shared__ float means[kWarps][G][D];
    __shared__ float2 stats[kWarps][G];
    pdl_enter();
    const float kNegInf = __int_as_float(0xff800000);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, lane8 = lane % 8;
    const uint32_t group = (uint32_t)(a.head_count / a.kv_head_count), sets = group / G, per_row = (uint32_t)a.kv_head_count * sets;
    const uint32_t row = blockIdx.x / per_row, kvh = blockIdx.x % per_row / sets, head0 = kvh * group + blockIdx.x % sets * G;
    const SeqRow s = seq_load(a.table, seq_of_query(a.table, row));
    int64_t lo, hi;
    key_range(a.causal, a.window, (int64_t)s.k_count - s.q_count + (int64_t)(row - s.q_start), s.k_count, lo, hi);
    const int tiles = (int)((hi - lo + 31) / 32), each = (tiles + (int)p.parts - 1) / (int)p.parts;
    const int tile_end = min(tiles, ((int)blockIdx.y + 1) * each);
    const uint64_t ld = a.kv_head_count * D;
    const float* keys = (const float*)a.k + (s.k_start + (uint64_t)lo) * ld + kvh * D + lane8 * 4;
    const float* values = (const float*)a.v + (s.k_start + (uint64_t)lo) * ld + kvh * D + lane * C;

    float4 q[G][C];
    float o[G][C], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const float* src = (const float*)a.q + ((uint64_t)row * a.head_count + head0 + g) * D + lane8 * 4;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(src + 32 * c));
            q[g][c] = make_float4(x.x * a.scale, x.y * a.scale, x.z * a.scale, x.w * a.scale);
            o[g][c] = 0.0f;
        }
        m[g] = kNegInf;
        l[g] = 0.0f;
    }
    for (int tile = (int)blockIdx.y * each + warp; tile < tile_end; tile += kWarps) {
        const int n = (int)min((int64_t)32, hi - lo - (int64_t)tile * 32);
        const float* k0 = keys + (uint64_t)tile * 32 * ld;
        float sc[G];
        // key 4 i + (lane / 8) of the tile for the eight lanes, whose lane i keeps it
#pragma unroll
        for (int i0 = 0; i0 < 8; i0 += kAhead) {
            float4 x[kAhead][C];
#pragma unroll
            for (int i = 0; i < kAhead; i++)
#pragma unroll
                for (int c = 0; c < C; c++)
                    x[i][c] = __ldg(reinterpret_cast<const float4*>(k0 + (uint64_t)min(4 * (i0 + i) + lane / 8, n - 1) * ld + 32 * c));
#pragma unroll
            for (int i = 0; i < kAhead; i++)
#pragma unroll
                for (int g = 0; g < G; g++) {
                    float d0 = 0.0f, d1 = 0.0f;
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        d0 = fmaf(q[g][c].x, x[i][c].x, fmaf(q[g][c].z, x[i][c].z, d0));
                        d1 = fmaf(q[g][c].y, x[i][c].y, fmaf(q[g][c].w, x[i][c].w, d1));
                    }
                    d0 += d1;
#pragma unroll
                    for (int w = 1; w < 8; w <<= 1) d0 += __shfl_xor_sync(0xffffffffu, d0, w);
                    if (lane8 == i0 + i) sc[g] = d0;
                }
        }
        float weight[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const float dot = 4 * lane8 + lane / 8 < n ? sc[g] : kNegInf;
            float most = fmaxf(m[g], dot);
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
            const float alpha = m[g] == kNegInf ? 0.0f : expf(m[g] - most);
            // (a NaN score passes through here, whatever the maximum made of it)
            const float e = dot == kNegInf ? 0.0f : expf(dot - most);
            float sum = e;
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            const float total = l[g] * alpha + sum, keep = l[g] > 0.0f ? l[g] * alpha / total : 0.0f;
            weight[g] = total != 0.0f ? e / total : 0.0f;
            m[g] = most;
            l[g] = total;
#pragma unroll
            for (int c = 0; c < C; c++) o[g][c] *= keep;
        }
        const float* v0 = values + (uint64_t)tile * 32 * ld;
        auto add = [&](int j0, auto whole) {
            float v[8][C];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float* src = v0 + (uint64_t)min(j0 + j, n - 1) * ld;
                if constexpr (C == 4) *reinterpret_cast<float4*>(v[j]) = __ldg(reinterpret_cast<const float4*>(src));
                else *reinterpret_cast<float2*>(v[j]) = __ldg(reinterpret_cast<const float2*>(src));
                // (a key past the last one: its weight of nothing would not keep an infinite value out)
                if (!decltype(whole)::value && j0 + j >= n)
#pragma unroll
                    for (int c = 0; c < C; c++) v[j][c] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const float w = __shfl_sync(0xffffffffu, weight[g], (j & 3) * 8 + (j0 + j) / 4);
#pragma unroll
                    for (int c = 0; c < C; c++) o[g][c] = fmaf(w, v[j][c], o[g][c]);
                }
        };
        int j0 = 0;
#pragma unroll 1
        for (; j0 + 8 <= n; j0 += 8) add(j0, std::true_type{});
        if (j0 < n) add(j0, std::false_type{});
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
#pragma unroll
        for (int c = 0; c < C; c++) means[warp][g][lane * C + c] = o[g][c];
        if (lane == 0) stats[warp][g] = make_float2(m[g], l[g]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * D; i += kThreads) {
        const int g = i / D, c = i % D;
        float most = kNegInf, total = 0.0f, share[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; w++) most = fmaxf(most, stats[w][g].x);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            share[w] = stats[w][g].y == 0.0f ? 0.0f : stats[w][g].y * expf(stats[w][g].x - most);
            total += share[w];
        }
#pragma unroll
        for (int w = 0; w < kWarps; w++) share[w] = total == 0.0f ? 0.0f : share[w] / total;
        const float x = weighted(share, [&](int w) { return means[w][g][c]; });
        if (p.parts == 1) {
            ((float*)a.out)[((uint64_t)row * a.head_count + head0 + g) * D + c] = x;
        } else {
            const uint64_t at = ((uint64_t)blockIdx.x * p.parts + blockIdx.y) * G + g;
            p.means[at * D + c] = x;
            if (c == 0) p.stats[at] = make_float2(most, total);
        }
    }
}

// A head's parts by their shares of the weights, one (query, head) per warp.
template <int D, int G>
__global__ void __launch_bounds__(kThreads) merge_few_kernel(const k::PackedAttentionArgs a, const Parts p, uint64_t heads) {
    pdl_enter();
    const uint64_t i = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;  // (query, head): the heads of an item in order
    const int lane = threadIdx.x % 32;
    if (i >= heads) return;
    const uint64_t first = i / G * p.parts * G + i % G;  // its part c at first + c G
    float most = __int_as_float(0xff800000), total = 0.0f, o[D / 32] = {};
    for (uint32_t c = lane; c < p.parts; c += 32) most = fmaxf(most, p.stats[first + (uint64_t)c * G].x);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
    auto share = [&](uint32_t c) {
        const float2 ml = p.stats[first + (uint64_t)c * G];
        return ml.y == 0.0f ? 0.0f : ml.y * expf(ml.x - most);
    };
    for (uint32_t c = lane; c < p.parts; c += 32) total += share(c);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
#pragma unroll 4
    for (uint32_t c = 0; c < p.parts; c++) {
        const float w = total == 0.0f ? 0.0f : share(c) / total;
#pragma unroll
        for (int e = 0; e < D / 32; e++) o[e] = fmaf(w, p.means[(first + (uint64_t)c * G) * D + lane + 32 * e], o[e]);
    }
#pragma unroll
    for (int e = 0; e < D / 32; e++) ((float*)a.out)[i * D + lane + 32 * e] = o[e];
}

template <int D, int G>
mg_status launch(Device* d, const k::PackedAttentionArgs& a) {
    const uint64_t heads = a.queries * a.head_count, items = heads / G;
    if (items > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    uint64_t longest = 0;
    for (const SeqRow& r : a.host->rows) longest = std::max<uint64_t>(longest, r.k_count + a.max_step);
    // Parts that fill the SMs once: for two rounds 4 sequences of 8192 keys take 85 us instead of 67, 16 take 236
    // instead of 229.
    const uint64_t want = (uint64_t)kCtasPerSm * d->sm_count / items;
    Parts p{(uint32_t)std::max<uint64_t>(1, std::min(want, longest / kPartKeys)), nullptr, nullptr};
    if (p.parts > 1) {
        MG_TRY(scratch(d, 9, heads * p.parts * (D * sizeof(float) + sizeof(float2)), (void**)&p.means));
        p.stats = reinterpret_cast<float2*>(p.means + heads * p.parts * D);
    }
    enqueue(d, attention_few_kernel<D, G>, dim3((unsigned)items, p.parts), kThreads, 0, a, p);
    if (p.parts > 1) {
        MG_TRY(launched(d, "packed attention launch"));
        enqueue(d, merge_few_kernel<D, G>, (unsigned)((heads + kWarps - 1) / kWarps), kThreads, 0, a, p, heads);
    }
    return launched(d, "packed attention launch");
}

}  // namespace

namespace k {

bool attention_packed_tc_eligible(const PackedAttentionArgs& a);

// With more queries a sequence's keys are read so often that splitting them once is cheaper: four sequences of 2000
// keys, 16 heads over 4, take 26 us with one query each (34 on the tensor cores), 27 with two (34), 37 with
// four (34); four of 8192 with four queries 199 (161).
constexpr uint64_t kMostQueries = 2;
bool attention_few_eligible(const PackedAttentionArgs& a) {
    return a.dtype == MG_F32 && a.host->max_queries <= kMostQueries && attention_packed_tc_eligible(a);
}

mg_status attention_few(Device* d, const PackedAttentionArgs& a) {
    const uint64_t group = a.head_count / a.kv_head_count;
    auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return group % 4 == 0 ? launch<D, 4>(d, a) : group % 2 == 0 ? launch<D, 2>(d, a) : launch<D, 1>(d, a);
    };
    return a.head_dim == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{});
}

}  // namespace k
}  // namespace mg
