// Log probabilities of given tokens, with entropy and top alternatives, from a row of logits.
#include <algorithm>

#include "sequences.cuh"

namespace mg {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kGroup = 4;                       // threads whose largest values are taken together
constexpr int kGroups = kThreads / kGroup;      // at least MG_LOGPROBS_MAX_TOP
constexpr int kCandidates = 1024;
static_assert(kGroups >= MG_LOGPROBS_MAX_TOP, "as many groups as top columns");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;  // stands for a maximum of nothing: finite, so that -inf less it is -inf

// A row's statistics so far: the largest logit m, and with d = scale (x - m) (scale = log2 e over the
// temperature) l = sum 2^d and t = sum d 2^d.
struct Stats {
    float m, l, t;
};

// l and t moved to the maximum m_new >= m.  d may be -inf where the maxima lie far apart: a part of no
// weight adds nothing (a NaN in l still does).
__device__ __forceinline__ void move_to(Stats& s, float m_new, float scale) {
    const float d = (s.m - m_new) * scale, w = exp2f(d);
    s.t = w > 0.0f ? w * fmaf(s.l, d, s.t) : 0.0f;
    s.l *= w;
    s.m = m_new;
}

__device__ __forceinline__ Stats merge(Stats a, Stats b, float scale) {
    const float m = fmaxf(a.m, b.m);
    move_to(a, m, scale);
    move_to(b, m, scale);
    return {m, a.l + b.l, a.t + b.t};
}

__device__ __forceinline__ Stats merge_warp(Stats s, float scale) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        s = merge(s, {__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.l, o), __shfl_xor_sync(0xffffffffu, s.t, o)},
                  scale);
    return s;
}

struct LogprobsK {
    const void* logits;
    const float* tokens;
    float* out;
    uint64_t rows;
    uint32_t vocab, top;
    float inv_temperature;
};

// Calls f(value, column) for the row's values of this thread, in 16-byte chunks where it can: the
// values before the first aligned one and after the last go to the first threads singly.
template <typename T, class Chunk, class One>
__device__ __forceinline__ void for_values(const T* x, uint32_t n, Chunk&& chunk, One&& one) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t head = min(n, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (uint32_t)sizeof(T));
    const uint32_t chunks = (n - head) / N, tail = head + chunks * N;
    for (uint32_t c = threadIdx.x; c < chunks; c += kThreads) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + head) + c);
        const T* p = reinterpret_cast<const T*>(&u);
        float v[N];
#pragma unroll
        for (uint32_t e = 0; e < N; e++) v[e] = to_f32(p[e]);
        chunk(v, head + c * N);
    }
    if (threadIdx.x < head) one(to_f32(x[threadIdx.x]), threadIdx.x);
    if (threadIdx.x < n - tail) one(to_f32(x[tail + threadIdx.x]), tail + threadIdx.x);
}

// One row per block.  A first pass over the row keeps each thread's running maximum and sums; the
// threads' maxima also bound the top columns: the top-th largest of the groups' maxima is reached by
// at least `top` values, so only the threads whose own maximum reaches it read their part of the
// row again (from the L2) and collect what reaches it.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobsK p) {
    __shared__ Stats parts[kWarps];
    __shared__ float group_max[kGroups];
    __shared__ float s_bound;
    __shared__ uint32_t s_count;
    __shared__ float cand[kCandidates];
    __shared__ uint32_t cand_col[kCandidates];
    __shared__ unsigned long long s_best[kWarps];
    pdl_enter();
    constexpr uint32_t N = 16 / sizeof(T);
    const uint64_t row = blockIdx.x;
    const T* x = (const T*)p.logits + row * p.vocab;
    float* out = p.out + row * (2 + 2 * (uint64_t)p.top);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float scale = kLog2e * p.inv_temperature;  // logits to log2 units

    Stats s{kLowest, 0.0f, 0.0f};
    auto grow = [&](float to) {
        if (to > s.m) move_to(s, to, scale);
    };
    auto add = [&](float v) {
        // an excluded logit (-inf) weighs nothing, and its distance must not be multiplied as infinite
        const float d = fmaxf((v - s.m) * scale, kLowest), w = exp2f(v != v ? v : d);
        s.l += w;
        s.t = fmaf(w, d, s.t);
    };
    for_values(x, p.vocab,
               [&](const float (&v)[N], uint32_t) {
                   float top = v[0];
#pragma unroll
                   for (uint32_t e = 1; e < N; e++) top = fmaxf(top, v[e]);
                   grow(top);
#pragma unroll
                   for (uint32_t e = 0; e < N; e++) add(v[e]);
               },
               [&](float v, uint32_t) {
                   grow(v);
                   add(v);
               });
    const float mine = s.m;
    s = merge_warp(s, scale);
    if (lane == 0) parts[warp] = s;
    if (p.top) {
        float g = mine;
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (threadIdx.x % kGroup == 0) group_max[threadIdx.x / kGroup] = g;
    }
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    s = parts[0];
#pragma unroll 1
    for (int w = 1; w < kWarps; w++) s = merge(s, parts[w], scale);
    // With log l, a log probability is (x - m) / temperature - log l, which keeps its digits where m is
    // large; NaN where there is no distribution (l is 0 without a finite logit, NaN with a NaN).
    const float nan = __int_as_float(0x7fc00000);
    const float log_l = s.l > 0.0f && s.m <= -kLowest ? logf(s.l) : nan;
    auto logprob = [&](float v) { return (v - s.m) * p.inv_temperature - log_l; };
    if (threadIdx.x == 0) {
        const float id = p.tokens ? p.tokens[row] : -1.0f;
        const bool is_column = id >= 0.0f && id < (float)p.vocab && id == floorf(id);
        out[0] = is_column ? logprob(to_f32(x[(uint32_t)id])) : nan;
        out[1] = log_l - s.t * kLn2 / s.l;  // log sum e^z - sum p z
    }
    if (!p.top) return;
    if (log_l != log_l) {
        for (uint32_t i = threadIdx.x; i < 2 * p.top; i += kThreads) out[2 + i] = nan;
        return;
    }
    // the top-th largest of the groups' maxima
    if (threadIdx.x < kGroups) {
        const float g = group_max[threadIdx.x];
        uint32_t rank = 0;
#pragma unroll 8
        for (int i = 0; i < kGroups; i++) {
            const float o = group_max[i];
            rank += o > g || (o == g && i < (int)threadIdx.x);
        }
        if (rank == p.top - 1) s_bound = g;
    }
    __syncthreads();
    // (fewer than `top` finite logits leave a bound of nothing: -inf columns fill up the rest)
    const float bound = s_bound <= kLowest ? __int_as_float(0xff800000) : s_bound;
    auto collect = [&](float v, uint32_t col) {
        if (v >= bound) {
            const uint32_t at = atomicAdd(&s_count, 1u);
            if (at < kCandidates) {
                cand[at] = v;
                cand_col[at] = col;
            }
        }
    };
    if (mine >= bound)
        for_values(x, p.vocab,
                   [&](const float (&v)[N], uint32_t col) {
                       float top = v[0];
#pragma unroll
                       for (uint32_t e = 1; e < N; e++) top = fmaxf(top, v[e]);
                       if (top >= bound)
#pragma unroll
                           for (uint32_t e = 0; e < N; e++) collect(v[e], col + e);
                   },
                   collect);
    __syncthreads();
    const uint32_t n = s_count;
    if (n <= kCandidates) {
        // each candidate's rank among them, ties by column
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float v = cand[i];
            const uint32_t col = cand_col[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < n; j++) rank += cand[j] > v || (cand[j] == v && cand_col[j] < col);
            if (rank < p.top) {
                out[2 + rank] = logprob(v);
                out[2 + p.top + rank] = (float)col;
            }
        }
        return;
    }
    // Very many equal logits: the largest (value, lowest column) below the last one taken, `top` times.
    // A key orders them: the value's bits made monotone (-0 as +0), then the column's complement.
    auto key_of = [](float v, uint32_t col) {
        const uint32_t b = __float_as_uint(v + 0.0f);
        return (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - col);
    };
    unsigned long long last = ~0ull;
    for (uint32_t r = 0; r < p.top; r++) {
        unsigned long long best = 0;
        auto consider = [&](float v, uint32_t col) {
            const unsigned long long key = key_of(v, col);
            if (key < last && key > best) best = key;
        };
        for_values(x, p.vocab,
                   [&](const float (&v)[N], uint32_t col) {
#pragma unroll
                       for (uint32_t e = 0; e < N; e++) consider(v[e], col + e);
                   },
                   consider);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; w++) best = max(best, s_best[w]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) {
            const uint32_t col = 0xffffffffu - (uint32_t)best;
            out[2 + r] = logprob(to_f32(x[col]));
            out[2 + p.top + r] = (float)col;
        }
    }
}

}  // namespace

namespace k {

mg_status token_logprobs(Device* d, const LogprobsArgs& a) {
    if (a.rows == 0) return MG_OK;
    if (a.rows > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "token log probabilities of too many rows");
    const LogprobsK p{a.logits, a.tokens, a.out, a.rows, (uint32_t)a.vocab, a.top, 1.0f / a.temperature};
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        enqueue(d, logprobs_kernel<T>, (unsigned)a.rows, kThreads, 0, p);
        return launched(d, "token log probabilities launch");
    });
}

}  // namespace k
}  // namespace mg
