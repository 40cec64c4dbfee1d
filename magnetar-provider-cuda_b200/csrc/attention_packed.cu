// Attention of packed sequences: softmax(Q K^T * scale) V, each sequence over its own keys, with
// causal / sliding-window masks and grouped heads.
//
// Query j of a sequence with n queries and m keys stands at position m - n + j; causal admits the
// keys up to and with that position, a window of w the last w of those.  A query that sees no key
// gives zeros.
#include <algorithm>

#include "attention_packed.cuh"

namespace mg {
namespace {

// Any dimensions up to 512, any alignment: one warp per (query, head).
constexpr int kRowThreads = 256;

template <typename T, typename R>
__global__ void __launch_bounds__(kRowThreads) attention_packed_row_kernel(const k::PackedAttentionArgs a, R kr, R vr) {
    pdl_enter();
    const uint64_t warp = (uint64_t)blockIdx.x * (kRowThreads / 32) + threadIdx.x / 32;
    if (warp >= a.queries * a.head_count) return;
    const uint64_t row = warp / a.head_count, head = warp % a.head_count;
    const SeqRow s = seq_load(a.table, seq_of_query(a.table, (uint32_t)row));
    attention_row<T, R, (int)(k::kPackedMaxDim / 32)>(a, kr, vr, s, row, head, threadIdx.x % 32);
}

mg_status attention_packed_rows(Device* d, const k::PackedAttentionArgs& a) {
    const uint64_t blocks = (a.queries * a.head_count + kRowThreads / 32 - 1) / (kRowThreads / 32);
    if (blocks > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "attention launch size overflows");
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        const uint64_t kw = a.kv_head_count * a.head_dim, vw = a.kv_head_count * a.value_dim;
        if (a.kv_dtype == MG_Q4) {
            const Q4Rows kr{(const uint8_t*)a.k, kw / kQ4Block}, vr{(const uint8_t*)a.v, vw / kQ4Block};
            enqueue(d, attention_packed_row_kernel<T, Q4Rows>, (unsigned)blocks, kRowThreads, 0, a, kr, vr);
        } else {
            const PlainRows<T> kr{(const T*)a.k, kw}, vr{(const T*)a.v, vw};
            enqueue(d, attention_packed_row_kernel<T, PlainRows<T>>, (unsigned)blocks, kRowThreads, 0, a, kr, vr);
        }
        return launched(d, "packed attention launch");
    });
}

}  // namespace

namespace k {

bool attention_packed_tc_eligible(const PackedAttentionArgs& a);
mg_status attention_packed_tc(Device* d, const PackedAttentionArgs& a);
bool attention_q4_eligible(const PackedAttentionArgs& a);
mg_status attention_q4(Device* d, const PackedAttentionArgs& a);

mg_status attention_packed(Device* d, const PackedAttentionArgs& a) {
    if (a.queries == 0) return MG_OK;
    if (attention_packed_tc_eligible(a)) return attention_packed_tc(d, a);
    if (attention_q4_eligible(a)) return attention_q4(d, a);
    return attention_packed_rows(d, a);
}

}  // namespace k
}  // namespace mg
