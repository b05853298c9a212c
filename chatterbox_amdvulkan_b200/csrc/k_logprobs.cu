// k_logprobs.cu — log probability of a given token, entropy, and the most
// probable alternatives, from rows of logits (what the engine reads back to
// the host at chatterbox-cpp/src/t3.cpp:612-614).
//
// With d_j = x_j - m, e_j = e^d_j, S = sum e_j, T = sum e_j d_j:
//   logprob = d_tok - ln S,   entropy = ln S - T / S.
// d is at most 0, so nothing overflows, and the entropy has no large terms that
// cancel.  One pass holds (m, S, T) per thread; a larger maximum m' turns T
// into c (T + S (m - m')) and S into c S, c = e^(m - m').  Two such states join
// by the same rule.  d is formed by a subtraction, not as x log2 e - m log2 e in
// one FMA: the rounding of m log2 e would differ from thread to thread, and
// logits at the type's lowest value would overflow.
//
// The order of the alternatives is that of one 64-bit number per element,
// (x as an ordered integer, then the complement of j), so ties fall to the
// lowest index and no two elements are equal.
//
// Bound by HBM at many rows (each logit is read once); by latency at one row.
#include "cbx_common.cuh"

namespace cbx {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

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

struct Stat {
    float m, s, t;  // maximum; sums relative to it
};

// Differences below this give e = 0; the bound keeps 0 * d from being a NaN.
constexpr float kLeast = -1e4f;

__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    // a state that has seen nothing above -inf has s = t = 0
    const float da = a.m == -INFINITY ? 0.0f : fmaxf(a.m - m, kLeast);
    const float db = b.m == -INFINITY ? 0.0f : fmaxf(b.m - m, kLeast);
    const float ca = ex2_approx(da * kLog2e), cb = ex2_approx(db * kLog2e);
    return {m, ca * a.s + cb * b.s, ca * fmaf(a.s, da, a.t) + cb * fmaf(b.s, db, b.t)};
}

// Adds N elements.  +inf and NaN make s a NaN.
template <int N>
__device__ __forceinline__ void add(Stat& st, const float (&f)[N]) {
    float b = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) b = fmaxf(b, f[i]);
    if (b > st.m) {
        const float d = st.m == -INFINITY ? 0.0f : fmaxf(st.m - b, kLeast);
        const float c = ex2_approx(d * kLog2e);
        st.t = c * fmaf(st.s, d, st.t);
        st.s *= c;
        st.m = b;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float d = f[i] - ref;
        const float e = ex2_approx(d * kLog2e);
        st.s += e;
        st.t = fmaf(e, fmaxf(d, kLeast), st.t);
    }
}

// x as an integer that orders like it; -0 as +0, NaN above +inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int j) {
    return (unsigned long long)ordered(x) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) {
    return a > b ? a : b;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_token_logprobs(LogprobArgs a) {
    constexpr int EV = Vec<T>::n;
    __shared__ Stat s_stat[kWarps];
    __shared__ unsigned long long s_key[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = a.vocab;
    grid_dep_wait();
    grid_dep_launch();
    for (int64_t r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.stride;
        // elements before the first 16-byte boundary, whole vectors, the rest
        int head = (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T);
        if (head > V) head = V;
        const int nv = (V - head) / EV, tail = head + nv * EV;
        Stat st = {-INFINITY, 0.0f, 0.0f};
        unsigned long long best = 0;
        auto one = [&](int j) {
            const float f[1] = {to_f(x[j])};
            add(st, f);
            best = max_key(best, key_of(f[0], j));
        };
        if (tid < head) one(tid);
        for (int i = tid; i < nv; i += kThreads) {
            float f[EV];
            ldv<T, EV>(x + head + (int64_t)i * EV, f);
            add(st, f);
#pragma unroll
            for (int e = 0; e < EV; ++e) best = max_key(best, key_of(f[e], head + i * EV + e));
        }
        if (tid < V - tail) one(tail + tid);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Stat b = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                      __shfl_xor_sync(0xffffffffu, st.t, o)};
            st = lane & o ? join(b, st) : join(st, b);
        }
        if (lane == 0) s_stat[warp] = st;
        __syncthreads();
        st = s_stat[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) st = join(st, s_stat[w]);
        const float log_s = logf(st.s);
        const bool bad = st.m == -INFINITY || st.s != st.s;
        if (tid == 0) {
            if (a.entropy) a.entropy[r] = bad ? NAN : log_s - st.t / st.s;
            if (a.logprob) {
                const int tok = a.tokens[r];
                float lp = NAN;
                if (tok >= 0 && tok < V) {
                    if (!bad) lp = (to_f(x[tok]) - st.m) - log_s;
                } else if (tok != -1) {
                    atomicOr(a.err, CBX_EFLAG_TOKEN_OOB);
                }
                a.logprob[r] = lp;
            }
        }
        // The largest, then the largest below it, ...
        for (int k = 0; k < a.top_k; ++k) {
            unsigned long long b = best;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) b = max_key(b, __shfl_xor_sync(0xffffffffu, b, o));
            if (lane == 0) s_key[warp] = b;
            __syncthreads();
            b = s_key[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) b = max_key(b, s_key[w]);
            const int j = (int)~(uint32_t)b;
            if (tid == 0) {
                a.top_ids[r * a.top_k + k] = j;
                a.top_logprobs[r * a.top_k + k] = bad ? NAN : (to_f(x[j]) - st.m) - log_s;
            }
            if (best == b && k + 1 < a.top_k) {  // its owner looks for its next one
                best = 0;
                auto next = [&](int i) {
                    const unsigned long long c = key_of(to_f(x[i]), i);
                    if (c < b) best = max_key(best, c);
                };
                if (tid < head) next(tid);
                for (int i = tid; i < nv; i += kThreads) {
                    float f[EV];
                    ldv<T, EV>(x + head + (int64_t)i * EV, f);
#pragma unroll
                    for (int e = 0; e < EV; ++e) {
                        const unsigned long long c = key_of(f[e], head + i * EV + e);
                        if (c < b) best = max_key(best, c);
                    }
                }
                if (tid < V - tail) next(tail + tid);
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

template <typename T>
int run_logprobs(const LogprobArgs& a, cudaStream_t st) {
    const int64_t most = (int64_t)num_sms() * occupancy(k_token_logprobs<T>, kThreads);
    const unsigned grid = (unsigned)(a.n_rows < most ? a.n_rows : most);
    return launch_status(launch(k_token_logprobs<T>, dim3(grid), dim3(kThreads), 0, st, a),
                         "cbx_token_logprobs");
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
    if (reinterpret_cast<uintptr_t>(logits) % (unsigned)type_size(type))
        return fail(CBX_ERR_INVALID_ARG, "%s: logits are not aligned to their type", name);
    LogprobArgs a{logits, row_stride, n_rows, (int)vocab, tokens, (int)top_k, logprob, entropy,
                  top_ids, top_logprobs, err_word};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (type) {
        case CBX_TYPE_F32: return run_logprobs<float>(a, st);
        case CBX_TYPE_BF16: return run_logprobs<__nv_bfloat16>(a, st);
        default: return run_logprobs<__half>(a, st);
    }
}
