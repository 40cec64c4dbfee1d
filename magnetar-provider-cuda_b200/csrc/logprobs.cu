// Log probabilities of given tokens, with entropy and top alternatives, from a row of logits.
//
// One pass over the row: with c = log2 e / temperature and a reference r near the largest c x, d = c x - r, l =
// sum 2^d and t = sum d 2^d.  The entropy is log l - ln 2 t / l, whatever the reference, and log p(x) =
// (x - max) / temperature - log l once l is about c max itself: c max - r, which is no more than the rounding
// of c max, is known exactly (one fused multiply-add), and so is every d up to the rounding of its own size.
// The row is read once from memory (the top columns look at a part of it again, in the L2): 2 or 4
// bytes a logit against one exponential and some ten other instructions.
#include <algorithm>
#include <cmath>

#include "sequences.cuh"
#include "sm100.cuh"

namespace mg {
namespace {

using namespace sm100;

// Threads of an SM, of a block (where there are more rows than SMs), and 16-byte chunks of a thread in
// flight.  8192 rows of 32000 bf16: 134 to 139 us, 3.8 to 3.9 TB/s, bound by instruction issue (62 % of the
// slots; 11.9 instructions a logit with 20 top columns).  Beside one such form of 132 us: 1280 threads an SM 136, blocks of 128
// threads 139 and of 512 172, 2 chunks 138 (the 40 registers of 1536 threads just hold 4).
constexpr int kPerSm = 1536, kBlock = 256, kBatch = 4;
constexpr int kGroups = 64;  // at the most, of threads whose largest values are taken together: 32 or 64
constexpr int kCandidates = 512;
static_assert(kGroups >= MG_LOGPROBS_MAX_TOP, "as many groups as top columns");
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMove = 16.0f;  // the reference moves when a value passes it by more than 2^16
// The pass holds where the row's maximum is at least kNear above the floor (2^-kNear is zero in an f32 of normal
// range, so it does not matter by how far logits were raised to it) and at most kFar (c x then rounds by no
// more than 4, so 2^d stays in range).  Other rows -- maxima or temperatures far from the usual -- take a second pass.
constexpr float kNear = 160.0f, kFar = 0x1p27f;

struct LogprobsK {
    const void* logits;
    const float* tokens;
    float* out;
    uint64_t rows;
    uint32_t vocab, top;
    float inv_temperature;
    float scale;  // c: logits to log2 units
    float floor;  // logits below it (excluded ones among them) are counted as it, see kNear and kFar
};

// Logits as they lie in memory: a 32-bit word of one or two, its larger and its values.
template <typename T>
struct Word;
template <>
struct Word<float> {
    static constexpr int kValues = 1;
    static constexpr uint32_t kExcluded = 0xff800000u;
    static __device__ __forceinline__ uint32_t of(float x) { return __float_as_uint(x); }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ float largest(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ float value(uint32_t a, int) { return __uint_as_float(a); }
};
template <>
struct Word<__nv_bfloat16> {
    static constexpr int kValues = 2;
    static constexpr uint32_t kExcluded = 0xff80ff80u;
    static __device__ __forceinline__ uint32_t of(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)) * 0x10001u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ float value(uint32_t a, int i) { return __uint_as_float(i ? a & 0xffff0000u : a << 16); }
    static __device__ __forceinline__ float largest(uint32_t a) { return max_nan(value(a, 0), value(a, 1)); }
};
template <>
struct Word<__half> {
    static constexpr int kValues = 2;
    static constexpr uint32_t kExcluded = 0xfc00fc00u;
    static __device__ __forceinline__ uint32_t of(float x) { return __half_as_ushort(__float2half_rn(x)) * 0x10001u; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ float value(uint32_t a, int i) {
        return __half2float(__ushort_as_half((unsigned short)(i ? a >> 16 : a & 0xffffu)));
    }
    static __device__ __forceinline__ float largest(uint32_t a) { return max_nan(value(a, 0), value(a, 1)); }
};

// A row in 16-byte chunks: the values before the first aligned one and after the last whole chunk are
// taken singly.
template <typename T>
struct Row {
    static constexpr uint32_t N = 16 / sizeof(T);  // values of a chunk
    const T* x;
    uint32_t n, head, chunks, tail;
    __device__ __forceinline__ Row(const T* row, uint32_t vocab) : x(row), n(vocab) {
        head = min(n, (uint32_t)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (uint32_t)sizeof(T));
        chunks = (n - head) / N;
        tail = head + chunks * N;
    }
    // The single value that falls to this thread (below 2 N threads), and whether there is one.
    __device__ __forceinline__ bool single(uint32_t i, uint32_t& col) const {
        col = i < head ? i : tail + (i - head);
        return i < head + (n - tail);
    }
    // f(value, column) for those that fall to this thread of the block.
    template <class F>
    __device__ __forceinline__ void for_values(F&& f) const {
        for (uint32_t c = threadIdx.x; c < chunks; c += blockDim.x) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(x + head) + c);
            const T* p = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (uint32_t e = 0; e < N; e++) f(to_f32(p[e]), head + c * N + e);
        }
        uint32_t col;
        if (single(threadIdx.x, col)) f(to_f32(x[col]), col);
    }
};

// One row per block.  The threads' maxima also bound the top columns: the top-th largest of the groups'
// maxima is reached by at least `top` values, so only the parts of the row of threads whose own maximum
// reaches it are read again (by the thread's whole warp), and what reaches it is collected.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kPerSm / kThreads) logprobs_kernel(const LogprobsK p) {
    using W = Word<T>;
    constexpr int kWarps = kThreads / 32;
    constexpr int kWords = kBatch * 4;
    __shared__ float warp_max[kWarps], warp_l[kWarps], warp_t[kWarps];
    __shared__ float lane_max[kWarps][32];
    __shared__ float group_max[kGroups];
    __shared__ float s_bound;
    __shared__ uint32_t s_count;
    __shared__ float cand[kCandidates];
    __shared__ uint32_t cand_col[kCandidates];
    __shared__ unsigned long long s_best[kWarps];
    __shared__ uint32_t s_equal[kWarps];
    pdl_enter();
    const uint64_t row = blockIdx.x;
    const Row<T> x((const T*)p.logits + row * p.vocab, p.vocab);
    float* out = p.out + row * (2 + 2 * (uint64_t)p.top);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    // ---- the row's sums -----------------------------------------------------------------------------
    const uint32_t floor = W::of(p.floor);
    const float low = W::value(floor, 0);
    float ref = low * p.scale;  // in log2 units
    uint64_t l2 = f2(0.0f, 0.0f), t2 = f2(0.0f, 0.0f);
    uint32_t most = W::kExcluded;  // of the logits as they are, NaN staying NaN
    const uint64_t scale2 = f2(p.scale, p.scale);
    // l and t moved to another reference; a part of no weight adds nothing, however far away
    auto moved = [&](float to, float& l, float& t) {
        const float d = ref - to, w = ex2(d);
        t = w > 0.0f ? w * fmaf(l, d, t) : 0.0f;
        l *= w;
    };
    // (a thread's batch holds n chunks; the rest of w is excluded logits)
    auto batch = [&](const uint32_t (&w)[kWords], int n) {
        uint32_t top[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
        for (int i = 4; i < kWords; i++) top[i % 4] = W::larger(top[i % 4], w[i]);
        const uint32_t all = W::larger(W::larger(top[0], top[1]), W::larger(top[2], top[3]));
        most = W::larger(most, all);
        if (fmaf(W::largest(all), p.scale, -ref) > kMove) {
            const float to = W::largest(all) * p.scale;
            float2 l = f2split(l2), t = f2split(t2);
            moved(to, l.x, t.x);
            moved(to, l.y, t.y);
            l2 = f2(l.x, l.y);
            t2 = f2(t.x, t.y);
            ref = to;
        }
        const uint64_t ref2 = f2(-ref, -ref);
#pragma unroll
        for (int b = 0; b < kBatch; b++) {
            if (b >= n) break;
#pragma unroll
            for (int i = 4 * b; i < 4 * b + 4; i += 3 - W::kValues) {
                const uint32_t u = W::larger(w[i], floor), v = W::kValues == 1 ? W::larger(w[(i + 1) % kWords], floor) : 0u;
                uint64_t d = ref2;
                f2fma(d, f2(W::value(u, 0), W::kValues == 2 ? W::value(u, 1) : W::value(v, 0)), scale2);
                const float2 y = f2split(d);
                const uint64_t e = f2(ex2(y.x), ex2(y.y));
                l2 = f2add(l2, e);
                f2fma(t2, e, d);
            }
        }
    };
    const uint4* chunk = reinterpret_cast<const uint4*>(x.x + x.head) + threadIdx.x;
    int left = x.chunks > threadIdx.x ? (int)((x.chunks - threadIdx.x + kThreads - 1) / kThreads) : 0;  // of this thread
    for (; left >= kBatch; left -= kBatch, chunk += kBatch * kThreads) {
        uint32_t w[kWords];
#pragma unroll
        for (int b = 0; b < kBatch; b++) {
            const uint4 u = __ldg(chunk + b * kThreads);
            w[4 * b] = u.x;
            w[4 * b + 1] = u.y;
            w[4 * b + 2] = u.z;
            w[4 * b + 3] = u.w;
        }
        batch(w, kBatch);
    }
    if (left) {
        uint32_t w[kWords];
#pragma unroll
        for (int b = 0; b < kBatch; b++) {
            // (the address is bounded, not the load: a conditional load is waited for at once)
            const uint4 u = __ldg(chunk + min(b, left - 1) * kThreads);
            w[4 * b] = b < left ? u.x : W::kExcluded;
            w[4 * b + 1] = b < left ? u.y : W::kExcluded;
            w[4 * b + 2] = b < left ? u.z : W::kExcluded;
            w[4 * b + 3] = b < left ? u.w : W::kExcluded;
        }
        batch(w, left);
    }
    uint32_t single;
    float lone = __int_as_float(0xff800000);
    const bool has_single = x.single(threadIdx.x, single);
    if (has_single) lone = to_f32(x.x[single]);
    float mine = max_nan(W::largest(most), lone);
    float2 ll = f2split(l2), tt = f2split(t2);
    float l = ll.x + ll.y, t = tt.x + tt.y;
    if (has_single) {
        const float v = max_nan(lone, low), to = v * p.scale;
        if (to > ref) {
            moved(to, l, t);
            ref = to;
        }
        const float d = fmaf(v, p.scale, -ref), w = ex2(d);
        l += w;
        t = fmaf(w, d, t);
    }
    // ---- the block's ----------------------------------------------------------------------------------
    float m = mine;
    lane_max[warp][lane] = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_max[warp] = m;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    m = warp_max[lane % kWarps];
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float to = max_nan(m, low) * p.scale;
    moved(to, l, t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) {
        warp_l[warp] = l;
        warp_t[warp] = t;
    }
    // The top-th largest of the groups' maxima.  A group is a lane of all warps, or of every other one (a short
    // row, which only the first warps read, still has all groups); the fewer groups where they are enough.
    const int groups = p.top <= 32 ? 32 : 64;
    float g = __int_as_float(0xff800000);
    if (p.top && threadIdx.x < groups) {
        for (int w = warp; w < kWarps; w += groups / 32) g = fmaxf(g, lane_max[w][lane]);
        group_max[threadIdx.x] = g;
    }
    if (groups == 64) __syncthreads();
    else __syncwarp();
    if (p.top && threadIdx.x < groups) {
        uint32_t rank = 0;
#pragma unroll 8
        for (int i = 0; i < groups; i++) {
            const float o = group_max[i];
            rank += o > g || (o == g && i < (int)threadIdx.x);
        }
        if (rank == p.top - 1) s_bound = g;
    }
    __syncthreads();
    l = warp_l[lane % kWarps];
    t = warp_t[lane % kWarps];
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    float lost = fmaf(m, p.scale, -to);  // by the rounding of c m
    const float over = (m - low) * p.scale;
    if (!(over >= kNear && over <= kFar) && m > __int_as_float(0xff800000)) {
        // The sums once more, about the largest itself.
        lost = 0.0f;
        l = t = 0.0f;
        x.for_values([&](float v, uint32_t) {
            const float d = fmaxf((v - m) * p.scale, -1e38f), w = ex2(d);
            l += w;
            t = fmaf(w, d, t);
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        __syncthreads();
        if (lane == 0) {
            warp_l[warp] = l;
            warp_t[warp] = t;
        }
        __syncthreads();
        l = t = 0.0f;
        for (int w = 0; w < kWarps; w++) {
            l += warp_l[w];
            t += warp_t[w];
        }
    }
    // A log probability is (x - m) / temperature - log l, which keeps its digits where m is large; NaN where
    // there is no distribution (no finite logit, an infinite one, a NaN).
    const float nan = __int_as_float(0x7fc00000);
    const float log_l = m > __int_as_float(0xff800000) && m < __int_as_float(0x7f800000) ? fmaf(-kLn2, lost, logf(l)) : nan;
    // (no probability is above one, and no entropy below zero, by a rounding either; NaN stays)
    auto logprob = [&](float v) {
        const float x = (v - m) * p.inv_temperature - log_l;
        return x > 0.0f ? 0.0f : x;
    };
    if (threadIdx.x == 0) {
        const float id = p.tokens ? p.tokens[row] : -1.0f;
        const bool is_column = id >= 0.0f && id < (float)p.vocab && id == floorf(id);
        out[0] = is_column ? logprob(to_f32(x.x[(uint32_t)id])) : nan;
        const float entropy = log_l - kLn2 * (t / l - lost);  // log sum e^z - sum p z
        out[1] = entropy < 0.0f ? 0.0f : entropy;
    }
    if (!p.top) return;
    if (log_l != log_l) {
        for (uint32_t i = threadIdx.x; i < 2 * p.top; i += kThreads) out[2 + i] = nan;
        return;
    }
    // ---- the top columns --------------------------------------------------------------------------------
    // (the bound is -inf where fewer than `top` groups have a finite logit)
    const float bound = s_bound;
    // Chunks of one thread at a time, or of two where a half warp covers them.  Where too many reach the bound
    // (a mask that leaves few columns, many equal logits) once more for those above it.
    const bool two = x.chunks <= 16u * kThreads;
    uint32_t n = 0;
    bool above = false;
    for (;;) {
        auto collect = [&](float v, uint32_t col) {
            if (above ? v > bound : v >= bound) {
                const uint32_t at = atomicAdd(&s_count, 1u);
                if (at < kCandidates) {
                    cand[at] = v;
                    cand_col[at] = col;
                }
            }
        };
        if (has_single) collect(lone, single);
        const float own = W::largest(most);
        for (uint32_t q = __ballot_sync(0xffffffffu, above ? own > bound : own >= bound); q; q &= q - 1) {
            uint32_t of = (uint32_t)__ffs(q) - 1, at = lane;
            if (two) {
                const uint32_t next = q & (q - 1);
                at = lane & 15;
                if (lane >= 16) of = next ? (uint32_t)__ffs(next) - 1 : 0xffffffu;
                if (next) q = next;
            }
            for (uint32_t c = threadIdx.x - lane + of + at * kThreads; c < x.chunks; c += 32 * kThreads) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(x.x + x.head) + c);
                if (!(W::largest(W::larger(W::larger(u.x, u.y), W::larger(u.z, u.w))) >= bound)) continue;
                const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
                for (uint32_t e = 0; e < x.N; e++) collect(to_f32(v[e]), x.head + c * x.N + e);
            }
        }
        __syncthreads();
        n = s_count;
        if (n <= kCandidates || above) break;
        __syncthreads();
        if (threadIdx.x == 0) s_count = 0;
        above = true;
        __syncthreads();
    }
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
        // the places that those above the bound leave: its first columns
        for (uint32_t col0 = 0; n < p.top && col0 < p.vocab; col0 += kThreads) {
            const uint32_t col = col0 + threadIdx.x;
            const bool equal = col < p.vocab && to_f32(x.x[min(col, p.vocab - 1)]) == bound;
            const uint32_t lanes = __ballot_sync(0xffffffffu, equal);
            if (lane == 0) s_equal[warp] = (uint32_t)__popc(lanes);
            __syncthreads();
            uint32_t place = n + (uint32_t)__popc(lanes & ((1u << lane) - 1));
            for (int w = 0; w < kWarps; w++) {
                if (w < warp) place += s_equal[w];
                n += s_equal[w];
            }
            if (equal && place < p.top) {
                out[2 + place] = logprob(bound);
                out[2 + p.top + place] = (float)col;
            }
            __syncthreads();
        }
        return;
    }
    // Very many logits in very few groups: the largest (value, lowest column) below the last one taken, `top` times.
    // A key orders them: the value's bits made monotone (-0 as +0), then the column's complement.
    auto key_of = [](float v, uint32_t col) {
        const uint32_t b = __float_as_uint(v + 0.0f);
        return (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - col);
    };
    unsigned long long last = ~0ull;
    for (uint32_t r = 0; r < p.top; r++) {
        unsigned long long best = 0;
        x.for_values([&](float v, uint32_t col) {
            const unsigned long long key = key_of(v, col);
            if (key < last && key > best) best = key;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; w++) best = max(best, s_best[w]);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) {
            const uint32_t col = 0xffffffffu - (uint32_t)best;
            out[2 + r] = logprob(to_f32(x.x[col]));
            out[2 + p.top + r] = (float)col;
        }
    }
}

}  // namespace

namespace k {

mg_status token_logprobs(Device* d, const LogprobsArgs& a) {
    if (a.rows == 0) return MG_OK;
    if (a.rows > 0x7fffffffull) return fail(MG_SHAPE_UNSUPPORTED, "token log probabilities of too many rows");
    LogprobsK p{a.logits, a.tokens, a.out, a.rows, (uint32_t)a.vocab, a.top, 1.0f / a.temperature, 0.0f, 0.0f};
    p.scale = 1.4426950408889634f * p.inv_temperature;
    // Half of kFar away from zero (a power of two in logits, which every type holds), or f16's lowest value, where only
    // -inf is below it.
    p.floor = -exp2f(floorf(log2f(std::min(1e38f, 0.5f * kFar / p.scale))));
    if (a.dtype == MG_F16) p.floor = std::max(p.floor, -65504.0f);
    return by_float(a.dtype, [&](auto t) {
        using T = decltype(t);
        // A block of 1024 threads where the rows leave SMs free and are long enough: 8 and 148 rows of 128 KB
        // 5.3 and 7.5 us (of 256 threads 6.4 and 10.4), of 32 KB 4.3 and 4.9 (3.9 and 4.5).
        if (a.rows <= (uint64_t)d->sm_count && a.vocab * sizeof(T) >= 49152) enqueue(d, logprobs_kernel<T, 1024>, (unsigned)a.rows, 1024, 0, p);
        else enqueue(d, logprobs_kernel<T, kBlock>, (unsigned)a.rows, kBlock, 0, p);
        return launched(d, "token log probabilities launch");
    });
}

}  // namespace k
}  // namespace mg
