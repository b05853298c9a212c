// k_logprobs.cu — log probability of a given token, entropy, and the most
// probable alternatives, from rows of logits (what the engine reads back to
// the host at chatterbox-cpp/src/t3.cpp:612-614).
//
// With R a whole number near max_j x_j log2 e, d_j = x_j log2 e - R (one FMA),
// S = sum 2^d_j and T = sum 2^d_j d_j:
//   entropy = (log2 S - T / S) ln 2,
//   logprob = x_tok - m - (log2 S - d_max) ln 2,  m the largest logit.
// No d is much above kSlack, so nothing overflows, and the entropy has no large
// terms that cancel.  One pass holds (R, S, T) per thread;
// a larger R' turns T into c (T + S (R - R')) and S into c S, c = 2^(R - R').
// R is a whole number, so that R, every R - R' and the powers are exact: the
// states of all threads refer to the same logits (log2 e max x, rounded in each
// thread, would not).  From 2^22 on, R is off m log2 e by its own rounding, which
// grows with it until 2^d is 0 or overflows; x log2 e itself overflows near the
// end of f32.  So a row whose largest logit is above 2^21 in magnitude (all of it
// masked by one large value, say) is summed again with d = (x - m) log2 e.
// Beside a smaller maximum such logits weigh nothing, whatever R their thread
// had: it leaves a state of 0, or a NaN where a sum overflowed, which sums the row
// again too.
//
// Alternatives.  Each thread keeps the largest logit of every segment of its
// elements.  The threads form 32 groups; the k-th largest of the 32 group
// maxima, tau, is at most the k-th largest logit (k groups hold one at or above
// it), so only segments whose largest reaches tau are read again, by all
// threads together, and their elements at or above tau, a few dozen, are ranked
// by counting.  The order is
// that of one 64-bit number per element (x as an ordered integer, then the
// complement of its index), so ties fall to the lowest index and no two
// elements are equal.  A row with more candidates than the list holds (a mask
// that leaves fewer than k, long runs of ties) or without a distribution takes
// its maxima one after the other instead.
//
// Bound by HBM at many rows (each logit is read once), by latency at few: NT
// threads share a row, from a warp each (no barriers; the work per row outside
// the loop is that of one warp) to a CTA of 512.
#include <type_traits>

#include "cbx_common.cuh"

namespace cbx {
namespace {

struct LogprobArgs {
    const void* x;
    int64_t stride;
    int64_t n_rows;
    int vocab;
    const int32_t* tokens;
    int top_k;
    float* logprob;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    int32_t* err;
};

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLeast = -1e4f; // 2^d = 0 far above it; keeps 0 * d from being a NaN

// x as an integer that orders like it; -0 as +0, NaN above +inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int j) {
    return (unsigned long long)ordered(x) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ float value_of(unsigned long long key) {  // of a key that is no NaN's
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) {
    return a > b ? a : b;
}

// The reference for a maximum m (any m, NaN aside): m log2 e to the nearest
// whole number, by the shift of 1.5 * 2^23, for |m| up to kWholeTo; beyond, any
// finite number near m log2 e.
constexpr float kWholeTo = 2097152.0f;  // 2^21: m log2 e is below 2^22
__device__ __forceinline__ float reference_of(float m) {
    constexpr float kShift = 12582912.0f, kMost = 1e37f;  // kMost log2 e is finite
    const float v = fminf(fmaxf(m, -kMost), kMost) * kLog2e;
    return __fsub_rn(__fadd_rn(v, kShift), kShift);
}

// The reference and the two sums relative to it, two halves each.
struct Stat {
    float r;
    float2 s, t;
    __device__ __forceinline__ void raise(float to) {
        const float d = fmaxf(r - to, kLeast), c = ex2_approx(d);
        t = __fmul2_rn(pair(c), __ffma2_rn(s, pair(d), t));
        s = __fmul2_rn(pair(c), s);
        r = to;
    }
};

// A maximum may lie this far above the reference: 2^d is far from overflow, and
// T gains no larger terms than log2 S has, so the threads of a warp seldom
// leave their common path to raise it after their first values.
constexpr float kSlack = 8.0f;

// Adds N values (N even) whose maximum is b.  NaN and +inf make s a NaN or inf.
template <int N, bool BOUNDED>
__device__ __forceinline__ void add(Stat& st, const float2 (&f)[N / 2], float b) {
    const float to = reference_of(b);
    if (to > st.r + kSlack) st.raise(to);
    const float2 ref = pair(-st.r);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 d = __ffma2_rn(f[i], pair(kLog2e), ref);
        const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        st.s = __fadd2_rn(st.s, e);
        // 0 * -inf would be NaN; 16-bit values come bounded from widen()
        if constexpr (BOUNDED) st.t = __ffma2_rn(e, d, st.t);
        else st.t = __ffma2_rn(e, make_float2(fmaxf(d.x, kLeast), fmaxf(d.y, kLeast)), st.t);
    }
}

// A row of logits: scalars up to the first 16-byte boundary, whole vectors,
// scalars behind them.  Thread tid owns scalar tid of either end and the
// vectors tid, tid + NT, ...
template <typename T>
struct Row {
    const T* x;
    int head, nv, tail, V;
    __device__ __forceinline__ Row(const LogprobArgs& a, int64_t r) {
        x = static_cast<const T*>(a.x) + r * a.stride;
        V = a.vocab;
        head = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
        if (head > V) head = V;
        nv = (V - head) / Vec<T>::n;
        tail = head + nv * Vec<T>::n;
    }
    __device__ __forceinline__ int first(int i) const { return head + i * Vec<T>::n; }
    __device__ __forceinline__ uint4 vec(int i) const {
        return __ldg(reinterpret_cast<const uint4*>(x + head) + i);
    }
};

// The least maximum whose row the sums above are right for.  f16: far enough above
// what widen() raises -inf to that this weighs nothing.
template <typename T>
__device__ __forceinline__ float least_max() {
    return __is_same(T, __half) ? -65000.0f : -kWholeTo;
}

// What widen() raises lower 16-bit logits to: the lowest finite value (f16), -2^100
// (bf16; its product with log2 e is exact, so its difference from its own
// reference is 0).
template <typename T>
__device__ __forceinline__ float lowest() {
    return __is_same(T, __half) ? -65504.0f : -0x1p100f;
}

// Elements of a vector as f32.  With BOUNDED, 16-bit ones are raised to lowest(),
// two in one instruction: no weight beside a maximum of least_max or more, but a
// finite x log2 e.  NaN stays.
template <typename T, bool BOUNDED>
__device__ __forceinline__ void widen(uint4 w, float2 (&f)[Vec<T>::n / 2]) {
    if constexpr (BOUNDED && sizeof(T) == 2) {
        constexpr bool bf16 = __is_same(T, __nv_bfloat16);
        using T2 = std::conditional_t<bf16, __nv_bfloat162, __half2>;
        const float low[2] = {lowest<T>(), lowest<T>()};
        const uint32_t b = pack32(low, T{});
        auto raise = [&](uint32_t v) {
            const T2 r = __hmax2_nan(*reinterpret_cast<const T2*>(&v), *reinterpret_cast<const T2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&r);
        };
        w = make_uint4(raise(w.x), raise(w.y), raise(w.z), raise(w.w));
    }
    float g[Vec<T>::n];
    constexpr int k = 4 / (int)sizeof(T);
    unpack32(w.x, g, T{});
    unpack32(w.y, g + k, T{});
    unpack32(w.z, g + 2 * k, T{});
    unpack32(w.w, g + 3 * k, T{});
#pragma unroll
    for (int i = 0; i < Vec<T>::n / 2; ++i) f[i] = make_float2(g[2 * i], g[2 * i + 1]);
}

// Largest of the elements of N words: 16-bit pairs compared as they are.
// NaN is passed over, as by fmaxf.
template <int N>
__device__ __forceinline__ float max_of(const uint4 (&w)[N], float) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i)
        m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(w[i].x), __uint_as_float(w[i].y)),
                           fmaxf(__uint_as_float(w[i].z), __uint_as_float(w[i].w))));
    return m;
}
template <int N, typename T, typename T2>
__device__ __forceinline__ float max_of_pairs(const uint4 (&w)[N]) {
    auto p = [](const uint32_t& v) { return *reinterpret_cast<const T2*>(&v); };
    T2 m = __hmax2(__hmax2(p(w[0].x), p(w[0].y)), __hmax2(p(w[0].z), p(w[0].w)));
#pragma unroll
    for (int i = 1; i < N; ++i)
        m = __hmax2(m, __hmax2(__hmax2(p(w[i].x), p(w[i].y)), __hmax2(p(w[i].z), p(w[i].w))));
    return fmaxf(fmaxf(to_f(m.x), to_f(m.y)), -INFINITY);  // all NaN: -inf
}
template <int N>
__device__ __forceinline__ float max_of(const uint4 (&w)[N], __nv_bfloat16) {
    return max_of_pairs<N, __nv_bfloat16, __nv_bfloat162>(w);
}
template <int N>
__device__ __forceinline__ float max_of(const uint4 (&w)[N], __half) {
    return max_of_pairs<N, __half, __half2>(w);
}
// A vector of -inf, which adds nothing.
template <typename T>
__device__ __forceinline__ uint4 nothing() {
    constexpr float kInf[2] = {-INFINITY, -INFINITY};
    const uint32_t v = pack32(kInf, T{});
    return make_uint4(v, v, v, v);
}

// The threads of one row: a warp, or the CTA.
template <int NT>
struct Team {
    static constexpr int kWarps = NT / 32;
    // Vectors that a thread sums at a time, and as many again on their way: two
    // where a team has little for each thread and latency counts.
    static constexpr int kUnroll = NT >= 256 ? 2 : 4;
    static constexpr int kCap = NT == 32 ? 128 : 512;   // candidates
    static constexpr int kWork = NT == 32 ? 128 : 256;  // segments to read again
    static constexpr int kSegs = 16;                    // segments of a thread's elements
    struct Shared {
        float seg[kSegs * NT];
        unsigned long long list[kCap];
        float group[32];
        float s[kWarps], t[kWarps];
        unsigned long long key[kWarps];
        int work[kWork];
        int count, n_work;
    };
    static __device__ __forceinline__ void sync() {
        if constexpr (NT == 32) __syncwarp();
        else __syncthreads();
    }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The lanes' values in falling order over the lanes (bitonic).
__device__ __forceinline__ float sort_falling(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int o = k >> 1; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, v, o);
            const bool larger = ((lane & o) == 0) == ((lane & k) == 0);
            v = larger ? fmaxf(v, w) : fminf(v, w);
        }
    return v;
}

// The top_k largest one after the other: each thread's largest, the team's
// largest, and its owner looks for its next one below it.
template <typename T, int NT>
__device__ __noinline__ void top_by_rounds(Row<T> row, int top_k, int32_t* ids, int tid,
                                           typename Team<NT>::Shared& sh) {
    constexpr int EV = Vec<T>::n;
    unsigned long long below = ~0ull, best = 0;
    for (int k = 0; k < top_k; ++k) {
        if (k == 0 || best == below) {
            best = 0;
            auto look = [&](int j) {
                const unsigned long long c = key_of(to_f(row.x[j]), j);
                if (k == 0 || c < below) best = max_key(best, c);
            };
            if (tid < row.head) look(tid);
            for (int i = tid; i < row.nv; i += NT)
                for (int e = 0; e < EV; ++e) look(row.first(i) + e);
            if (tid < row.V - row.tail) look(row.tail + tid);
        }
        unsigned long long b = best;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) b = max_key(b, __shfl_xor_sync(0xffffffffu, b, o));
        if constexpr (NT > 32) {
            if ((tid & 31) == 0) sh.key[tid >> 5] = b;
            __syncthreads();
            for (int w = 0; w < NT / 32; ++w) b = max_key(b, sh.key[w]);
            __syncthreads();
        }
        below = b;
        if (tid == 0) ids[k] = (int)~(uint32_t)b;
    }
}

// S and T with d = (x - m) log2 e, for the rows that have no whole reference.
template <typename T, int NT>
__device__ __noinline__ void sums_from_differences(Row<T> row, int tid, float m,
                                                   typename Team<NT>::Shared& sh, float* s_out, float* t_out) {
    float s = 0.0f, t = 0.0f;
    for (int j = tid; j < row.V; j += NT) {
        const float d = (to_f(row.x[j]) - m) * kLog2e, e = ex2_approx(d);
        s += e;
        t = fmaf(e, fmaxf(d, kLeast), t);
    }
    s = warp_sum(s);
    t = warp_sum(t);
    if constexpr (NT > 32) {
        __syncthreads();  // the first sums have been read
        if ((tid & 31) == 0) {
            sh.s[tid >> 5] = s;
            sh.t[tid >> 5] = t;
        }
        __syncthreads();
        s = t = 0.0f;
        for (int w = 0; w < NT / 32; ++w) {
            s += sh.s[w];
            t += sh.t[w];
        }
    }
    *s_out = s;
    *t_out = t;
}

template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT < 128 ? 128 : NT, NT <= 128 ? 7 : NT == 256 ? 5 : 1)
k_token_logprobs(LogprobArgs a) {
    using Tm = Team<NT>;
    constexpr int EV = Vec<T>::n;
    constexpr int kTeams = NT < 128 ? 128 / NT : 1;  // rows at a time
    __shared__ typename Tm::Shared shared[kTeams];
    const int tid = threadIdx.x % NT, lane = tid & 31, warp = tid >> 5;
    typename Tm::Shared& sh = shared[threadIdx.x / NT];
    grid_dep_wait();
    grid_dep_launch();
    const int64_t stride = (int64_t)gridDim.x * kTeams;
    const int64_t r0 = (int64_t)blockIdx.x * kTeams + threadIdx.x / NT;
    constexpr int kUnroll = Tm::kUnroll;
    constexpr bool kBounded = sizeof(T) == 2;
    constexpr int kBatch = NT * kUnroll;  // vectors that the team takes at a time
    // A row's b-th batch; behind the row: nothing.
    auto fetch = [&](const Row<T>& row, int b, uint4 (&w)[kUnroll]) {
        const uint4* p = reinterpret_cast<const uint4*>(row.x + row.head) + b * kBatch + tid;
        if ((b + 1) * kBatch <= row.nv) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) w[u] = __ldg(p + u * NT);
        } else {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                w[u] = nothing<T>();
                if (b * kBatch + u * NT + tid < row.nv) w[u] = __ldg(p + u * NT);
            }
        }
    };
    // The next batch is on its way while one is summed, the next row's first
    // batch and token while a row is finished: a row's sums, joins and
    // alternatives are a chain of latencies that would otherwise follow its loads.
    uint4 ahead[kUnroll];
    int tok_ahead = -1;
    if (r0 < a.n_rows) {
        if (tid == 0 && a.logprob) tok_ahead = __ldg(a.tokens + r0);
        fetch(Row<T>(a, r0), 0, ahead);
    }
    for (int64_t r = r0; r < a.n_rows; r += stride) {
        const Row<T> row(a, r);
        Stat st = {reference_of(-INFINITY), {0.0f, 0.0f}, {0.0f, 0.0f}};
        float top = -INFINITY;  // the thread's largest
        // The ends: at most one scalar of each per thread.  The given token's logit.
        T end_head = from_f<T>(-INFINITY), end_tail = end_head, x_tok = from_f<T>(NAN);
        if (tid < row.head) end_head = row.x[tid];
        if (tid < row.V - row.tail) end_tail = row.x[row.tail + tid];
        const int tok = tok_ahead;
        if (tok >= 0 && tok < row.V) x_tok = row.x[tok];

        const int batches = row.nv > kBatch ? (row.nv + kBatch - 1) / kBatch : 1;
        const int per = (batches + Tm::kSegs - 1) / Tm::kSegs;  // batches of a segment
        int n_segs = 0;
        float seg = -INFINITY;
        for (int b = 0, in_seg = 0; b < batches; ++b) {
            uint4 w[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) w[u] = ahead[u];
            if (b + 1 < batches) {
                fetch(row, b + 1, ahead);
            } else if (r + stride < a.n_rows) {
                if (tid == 0 && a.logprob) tok_ahead = __ldg(a.tokens + r + stride);
                fetch(Row<T>(a, r + stride), 0, ahead);
            }
            const float m = max_of(w, T{});
            // The largest of the values summed: a thread with nothing but -inf so far must
            // not take that as its reference, or its sums overflow.
            const float most = kBounded ? fmaxf(m, lowest<T>()) : m;
            if ((b + 1) * kBatch <= row.nv) {
                float2 f[kUnroll * EV / 2];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    widen<T, kBounded>(w[u], *reinterpret_cast<float2(*)[EV / 2]>(f + u * EV / 2));
                add<kUnroll * EV, kBounded>(st, f, most);
            } else {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    if (b * kBatch + u * NT < row.nv) {
                        float2 f[EV / 2];
                        widen<T, kBounded>(w[u], f);
                        add<EV, kBounded>(st, f, most);
                    }
            }
            if (TOP) {
                seg = fmaxf(seg, m);
                if (++in_seg == per || b + 1 == batches) {
                    sh.seg[n_segs++ * NT + tid] = seg;
                    seg = -INFINITY;
                    in_seg = 0;
                }
            }
            top = fmaxf(top, m);
        }
        float2 ends[1] = {{to_f(end_head), to_f(end_tail)}};
        if (tid < row.head || tid < row.V - row.tail) {
            const float m = fmaxf(ends[0].x, ends[0].y);
            add<2, false>(st, ends, m);
            top = fmaxf(top, m);
        }

        // Maximum of the row, and of the 32 groups.
        float m = warp_max(top), group = top;
        if (TOP && tid == 0) sh.count = sh.n_work = 0;
        if constexpr (NT > 32) {
#pragma unroll
            for (int o = 1; o < NT / 32; o <<= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
            if (tid % (NT / 32) == 0) sh.group[tid / (NT / 32)] = group;
            __syncthreads();
            group = sh.group[lane];
            m = warp_max(group);
        } else if (TOP) {
            __syncwarp();
        }
        // The sums relative to the row's reference.
        const float ref = reference_of(m);
        st.raise(ref);
        float s = warp_sum(st.s.x + st.s.y), t = warp_sum(st.t.x + st.t.y);
        if (NT > 32 && lane == 0) {
            sh.s[warp] = s;
            sh.t[warp] = t;
        }
        if constexpr (TOP) {
            float tau = m;
            if (a.top_k > 1) tau = __shfl_sync(0xffffffffu, sort_falling(group, lane), a.top_k - 1);
            auto put = [&](int at, float v, int j) {
                if (at < Tm::kCap) sh.list[at] = key_of(v, j);
            };
            if (top >= tau && (tau != -INFINITY || row.V <= Tm::kCap)) {
                if (tid < row.head && ends[0].x >= tau) put(atomicAdd(&sh.count, 1), ends[0].x, tid);
                if (tid < row.V - row.tail && ends[0].y >= tau) put(atomicAdd(&sh.count, 1), ends[0].y, row.tail + tid);
                uint32_t todo = 0;
                for (int q = 0; q < n_segs; ++q) todo |= (sh.seg[q * NT + tid] >= tau ? 1u : 0u) << q;
                if (todo) {
                    int at = atomicAdd(&sh.n_work, __popc(todo));
                    for (; todo && at < Tm::kWork; todo &= todo - 1, ++at)
                        sh.work[at] = (__ffs(todo) - 1) * NT + tid;
                }
            }
            Tm::sync();
            // The vectors of the listed segments, one for each thread: their owners
            // alone would walk them one by one, their warps waiting.
            const int n_work = sh.n_work, span = per * kUnroll;
            if (n_work <= Tm::kWork)
                for (int i = tid; i < n_work * span; i += NT) {
                    const int item = i / span, of = sh.work[item];
                    const int v = of % NT + (of / NT * span + (i - item * span)) * NT;
                    if (v >= row.nv) continue;
                    const uint4 w[1] = {row.vec(v)};
                    if (max_of(w, T{}) < tau) continue;
                    float2 f[EV / 2];
                    widen<T, false>(w[0], f);
                    int n = 0;
#pragma unroll
                    for (int e = 0; e < EV / 2; ++e) n += (f[e].x >= tau) + (f[e].y >= tau);
                    if (!n) continue;  // all NaN
                    int at = atomicAdd(&sh.count, n);
                    const int j = row.first(v);
#pragma unroll
                    for (int e = 0; e < EV / 2; ++e) {
                        if (f[e].x >= tau) put(at++, f[e].x, j + 2 * e);
                        if (f[e].y >= tau) put(at++, f[e].y, j + 2 * e + 1);
                    }
                }
        }
        if (NT > 32 || TOP) Tm::sync();
        if constexpr (NT > 32) {
            s = t = 0.0f;
#pragma unroll
            for (int w = 0; w < Tm::kWarps; ++w) {
                s += sh.s[w];
                t += sh.t[w];
            }
        }
        bool bad = false, huge = false;
        if (!(m >= least_max<T>() && m <= kWholeTo && s <= 3e38f && t == t)) {  // rare: no distribution, or very large logits
            huge = true;
            sums_from_differences<T, NT>(row, tid, m, sh, &s, &t);
            bad = fabsf(m) == INFINITY || s != s;
        }
        const float log_s = log2f(s);
        // ln sum e^(x - m): the sums refer to ref, which m log2 e is below by the FMA's value.
        const float ln_s = (log_s - (huge ? 0.0f : fmaf(m, kLog2e, -ref))) * kLn2;
        // The sum's rounding may put a value that is 0 but for it 2^-24 on the wrong side of 0.
        auto log_prob = [&](float x) {
            const float v = (x - m) - ln_s;
            return bad ? (float)NAN : v > 0.0f ? 0.0f : v;  // NaN (no token) stays
        };
        if (tid == 0) {
            const float h = (log_s - t / s) * kLn2;
            if (a.entropy) a.entropy[r] = bad ? (float)NAN : h < 0.0f ? 0.0f : h;
            if (a.logprob) {
                if (tok < -1 || tok >= row.V) atomicOr(a.err, CBX_EFLAG_TOKEN_OOB);
                a.logprob[r] = log_prob(to_f(x_tok));  // NaN without a token
            }
        }
        if constexpr (TOP) {
            const int n = sh.count;
            if (!bad && sh.n_work <= Tm::kWork && n >= a.top_k && n <= Tm::kCap) {
                for (int i = tid; i < n; i += NT) {
                    const unsigned long long key = sh.list[i];
                    int rank = 0;
                    for (int j = 0; j < n; ++j) rank += sh.list[j] > key;
                    if (rank < a.top_k) {
                        a.top_ids[r * a.top_k + rank] = (int)~(uint32_t)key;
                        a.top_logprobs[r * a.top_k + rank] = log_prob(value_of(key));
                    }
                }
            } else {
                int32_t* ids = a.top_ids + r * a.top_k;
                top_by_rounds<T, NT>(row, a.top_k, ids, tid, sh);
                if (tid == 0)
                    for (int k = 0; k < a.top_k; ++k)
                        a.top_logprobs[r * a.top_k + k] = log_prob(to_f(row.x[ids[k]]));
            }
        }
        Tm::sync();  // the next row uses the shared arrays again
    }
}

template <typename T, int NT>
int run_team(const LogprobArgs& a, cudaStream_t st) {
    constexpr int kCta = NT < 128 ? 128 : NT;
    auto kern = a.top_k > 0 ? k_token_logprobs<T, NT, true> : k_token_logprobs<T, NT, false>;
    // The fewest CTAs that give each the same number of rows within one: no last
    // round of rows on a part of the resident warps.
    const int64_t ctas = (a.n_rows + kCta / NT - 1) / (kCta / NT);
    const int64_t most = (int64_t)num_sms() * occupancy(kern, kCta);
    const int64_t rounds = (ctas + most - 1) / most;
    const unsigned grid = (unsigned)((ctas + rounds - 1) / rounds);
    return launch_status(launch(kern, dim3(grid), dim3(kCta), 0, st, a),
                         "cbx_token_logprobs");
}

// Threads of a row.  A warp costs least per row, but needs many rows to fill
// the GPU and is slow on a long one; a whole CTA is quickest on a single long
// row.  Measured in us (B200; 32 / 128 / 256 / 512 threads a row):
//   1 x 6563 f32, top 5          6.9 / 4.5 / 4.5 / 4.5
//   1 x 50276 f32, top 5        29.8 / 10.3 / 9.3 / 7.6
//   256 x 6563 f32, top 8        7.9 / 5.2 / 5.5 / 8.2
//   1000 x 500 f16, top 8        5.2 / 6.5 / 13.7 / 67.3
//   1100 x 6563 f16, top 8       8.2 / 12.4 / 13.7 / 28.7
//   1100 x 50276 f16, top 8     41.8 / 40.9 / 37.3 / 61.6
//   2048 x 50276 f16, top 20    67.6 / 45.5 / 57.5 / 110.4
//   4200 x 20000 bf16, top 5    58.1 / 50.9 / 59.3 / 138.5
//   8192 x 6563 bf16, top 1     27.7 / 42.7 / 68.4 / 170.6 (107.7 MB: 3.9 TB/s)
// A row with less than a vector for each thread would leave groups without a
// maximum and so without a bound for its alternatives: it takes fewer threads.
// The warp's list holds the candidates of up to 24 alternatives (about 32 ln(1 /
// (1 - k / 32)) of them, 44 for 24).
template <typename T>
int run_logprobs(const LogprobArgs& a, cudaStream_t st) {
    const int64_t rows = a.n_rows, sms = num_sms(), vecs = a.vocab / Vec<T>::n;
    const bool warp = a.top_k <= 24;
    if (warp && (vecs < 128 || (rows >= 7 * sms && vecs <= 2048))) return run_team<T, 32>(a, st);
    if (rows <= sms && vecs >= 2048) return run_team<T, 512>(a, st);
    if (rows >= 10 * sms || vecs < 2048) return run_team<T, 128>(a, st);
    return run_team<T, 256>(a, st);
}

}  // namespace
}  // namespace cbx

extern "C" CBX_API int cbx_token_logprobs(const void* logits, int type, int64_t row_stride,
                                          int64_t n_rows, int64_t vocab, const int32_t* tokens,
                                          int64_t top_k, float* logprob, float* entropy,
                                          int32_t* top_ids, float* top_logprobs,
                                          int32_t* err_word, cbx_stream_t stream) {
    using namespace cbx;
    const char* name = "cbx_token_logprobs";
    if (n_rows < 0 || vocab <= 0 || vocab > (1 << 30))
        return fail(CBX_ERR_INVALID_ARG, "%s: n_rows %lld vocab %lld", name, (long long)n_rows,
                    (long long)vocab);
    if (row_stride == 0) row_stride = vocab;
    if (row_stride < vocab)
        return fail(CBX_ERR_INVALID_ARG, "%s: row_stride %lld < vocab", name, (long long)row_stride);
    if (!valid_type(type)) return fail(CBX_ERR_UNSUPPORTED_DTYPE, "%s: type %d", name, type);
    if (top_k < 0 || top_k > vocab || top_k > CBX_LOGPROBS_MAX_TOP)
        return fail(CBX_ERR_INVALID_ARG, "%s: top_k %lld outside [0, min(vocab, %d)]", name,
                    (long long)top_k, CBX_LOGPROBS_MAX_TOP);
    if (n_rows == 0) return ok();
    if (!logits || (tokens != nullptr) != (logprob != nullptr) || (tokens && !err_word) ||
        (top_k > 0 && (!top_ids || !top_logprobs)))
        return fail(CBX_ERR_INVALID_ARG, "%s: NULL argument", name);
    if (!aligned_to(logits, type_size(type)) || !aligned_to(tokens, 4) || !aligned_to(logprob, 4) ||
        !aligned_to(entropy, 4) || !aligned_to(top_ids, 4) || !aligned_to(top_logprobs, 4) ||
        !aligned_to(err_word, 4))
        return fail(CBX_ERR_INVALID_ARG, "%s: an argument is not aligned to its type", name);
    LogprobArgs a{logits, row_stride, n_rows, (int)vocab, tokens, (int)top_k, logprob, entropy,
                  top_ids, top_logprobs, err_word};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (type) {
        case CBX_TYPE_F32: return run_logprobs<float>(a, st);
        case CBX_TYPE_BF16: return run_logprobs<__nv_bfloat16>(a, st);
        default: return run_logprobs<__half>(a, st);
    }
}
