// Attention of packed sequences: softmax(Q K^T * scale) V, each sequence over its own keys, with
// causal / sliding-window masks and grouped heads.
//
// Query j of a sequence with n queries and m keys stands at position m - n + j; causal admits the
// keys up to and with that position, a window of w the last w of those.  A query that sees no key
// gives zeros.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "attention_packed.cuh"

namespace mg {
namespace {

// Any dimensions up to 512, any alignment, on the CUDA cores: one warp per (query, head), or SPLIT: a block for
// each, whose warps take every eighth 32 keys and are merged at the end.
// Four prompts of up to 512 tokens, 16 heads over 4 of 96, bfloat16: 0.42 ms (keys one at a time by lanes over the
// dimensions, as this kernel once did: 5.8); one query each of four over 64 to 3000 keys: 58 us (one warp each:
// 0.85 ms).  Bound by the loads' latency: a key's row is 16-byte pieces of 32 different lines.
constexpr int kRowWarps = 8, kRowThreads = 32 * kRowWarps;

template <typename T, typename R, int N, bool SPLIT>
__global__ void __launch_bounds__(kRowThreads) attention_packed_row_kernel(const k::PackedAttentionArgs a, R kr, R vr) {
    __shared__ __align__(16) float q_shared[kRowWarps][k::kPackedMaxDim];
    __shared__ float means[SPLIT ? kRowWarps : 1][32 * N];
    __shared__ float maxima[kRowWarps], sums[kRowWarps];
    constexpr int kAhead = N <= 4 ? 8 : N <= 8 ? 4 : 2;
    pdl_enter();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t item = SPLIT ? blockIdx.x : (uint64_t)blockIdx.x * kRowWarps + warp;
    if (item >= a.queries * a.head_count) return;
    const uint64_t row = item / a.head_count, head = item % a.head_count;
    const SeqRow s = seq_load(a.table, seq_of_query(a.table, (uint32_t)row));
    if constexpr (!SPLIT) {
        attention_row<T, R, N, kAhead>(a, kr, vr, s, row, head, lane, q_shared[warp]);
    } else {
        float o[N], m, l;
        attention_keys<T, R, N, kAhead>(a, kr, vr, s, row, head, lane, q_shared[warp], 32 * warp, 32 * kRowWarps, o, m, l);
#pragma unroll
        for (int i = 0; i < N; i++) means[warp][lane + 32 * i] = o[i];
        if (lane == 0) {
            maxima[warp] = m;
            sums[warp] = l;
        }
        __syncthreads();
        // the warps' means, each by its share of the weights
        float most = __int_as_float(0xff800000), total = 0.0f, share[kRowWarps];
#pragma unroll
        for (int w = 0; w < kRowWarps; w++) most = fmaxf(most, maxima[w]);
#pragma unroll
        for (int w = 0; w < kRowWarps; w++) {
            share[w] = sums[w] == 0.0f ? 0.0f : sums[w] * expf(maxima[w] - most);
            total += share[w];
        }
        T* out = (T*)a.out + (row * a.head_count + head) * a.value_dim;
        for (int i = threadIdx.x; i < (int)a.value_dim; i += kRowThreads) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowWarps; w++) x = fmaf(total != 0.0f ? share[w] / total : 0.0f, means[w][i], x);
            out[i] = from_f32<T>(x);
        }
    }
}

template <typename T, typename R>
void enqueue_rows(Device* d, const k::PackedAttentionArgs& a, unsigned blocks, bool split, const R& kr, const R& vr) {
    auto go = [&](auto n) {
        constexpr int N = decltype(n)::value;
        if (split) enqueue(d, attention_packed_row_kernel<T, R, N, true>, blocks, kRowThreads, 0, a, kr, vr);
        else enqueue(d, attention_packed_row_kernel<T, R, N, false>, blocks, kRowThreads, 0, a, kr, vr);
    };
    if (a.value_dim <= 128) go(std::integral_constant<int, 4>{});
    else if (a.value_dim <= 256) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, (int)(k::kPackedMaxDim / 32)>{});
}

mg_status attention_packed_rows(Device* d, const k::PackedAttentionArgs& a) {
    // A block for each while that leaves the SMs with fewer warps than they hold.
    const uint64_t items = a.queries * a.head_count;
    const bool split = items < (uint64_t)d->sm_count * 16;
    const uint64_t blocks = split ? items : (items + kRowWarps - 1) / kRowWarps;
    if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        const uint64_t kw = a.kv_head_count * a.head_dim, vw = a.kv_head_count * a.value_dim;
        if (a.kv_dtype == MG_Q4) {
            enqueue_rows<T>(d, a, (unsigned)blocks, split, Q4Rows{(const uint8_t*)a.k, kw / kQ4Block}, Q4Rows{(const uint8_t*)a.v, vw / kQ4Block});
        } else {
            const bool vec = reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && a.head_dim % 8 == 0;
            enqueue_rows<T>(d, a, (unsigned)blocks, split, PlainRows<T>{(const T*)a.k, kw, vec}, PlainRows<T>{(const T*)a.v, vw, false});
        }
        return launched(d, "packed attention launch");
    });
}

}  // namespace

namespace k {

bool attention_packed_tc_eligible(const PackedAttentionArgs& a);
mg_status attention_packed_tc(Device* d, const PackedAttentionArgs& a);
bool attention_few_eligible(const PackedAttentionArgs& a);
mg_status attention_few(Device* d, const PackedAttentionArgs& a);
bool attention_q4_eligible(const PackedAttentionArgs& a);
mg_status attention_q4(Device* d, const PackedAttentionArgs& a);

mg_status attention_packed(Device* d, const PackedAttentionArgs& a) {
    if (a.queries == 0) return MG_OK;
    // f32 queries take two bfloat16 terms per operand on the tensor cores (2-6e-6 of relative error against 64 bits) for
    // 20 to 30 times the rate of f32 arithmetic (2-4e-7; 4 x 2048 tokens, 32 heads: 15.6 ms against 0.5), which a caller
    // may have instead.
    static const bool f32_throughout = [] {
        const char* e = getenv("MAGNETAR_CUDA_PACKED_F32");
        return e && atoi(e) != 0;
    }();
    if (f32_throughout && a.dtype == MG_F32) return attention_packed_tc_eligible(a) ? attention_few(d, a) : attention_packed_rows(d, a);
    if (attention_few_eligible(a)) return attention_few(d, a);
    if (attention_packed_tc_eligible(a)) {
        // The two-term copies of f32 keys and values hold a row for every key of every sequence (with a captured step's
        // largest advance), 8 bytes a pair of values.  Where memory cannot hold them -- long rows that many sequences
        // share -- the keys are read as they lie.
        const mg_status s = attention_packed_tc(d, a);
        if (s != MG_OUT_OF_DEVICE_MEMORY || a.dtype != MG_F32) return s;
        clear_error();
        return attention_few(d, a);
    }
    if (attention_q4_eligible(a)) return attention_q4(d, a);
    return attention_packed_rows(d, a);
}

}  // namespace k
}  // namespace mg
