// k_paged_attention.cu — attention of one new token per row over a paged
// key-value cache (one query of the engine's attention, between
// chatterbox-cpp/src/t3.cpp:489 and :528).
//
// For a row and a head, over the keys j below the row's length:
//   s_j = scale q.k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).
// One pass over the keys holds (m, l = sum e^(s - m), acc = sum e^(s - m) v) in
// f32 registers; a larger maximum rescales l and acc by e^(m_old - m_new).
// Two such states over disjoint keys join into one by the same rescaling, so
// the keys are split over lanes, warps and CTAs and the states joined at the
// end.  Exponentials are base 2 (scale log2 e is folded into q).
//
// Bound by HBM: each key and value is read once and takes 2 FMAs per query
// head.  A key row of one kv head is VL 16-byte vectors, one per lane, so a
// warp reads 32 / VL keys per load instruction and holds U loads of keys and
// U of values in flight: no shared memory between HBM and the FMAs.
#include "cbx_common.cuh"

namespace cbx {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxSplits = 64;
constexpr int kMinKeys = 256;  // keys of a split at the least

struct AttnArgs {
    const void* q;
    int q_type;
    int64_t q_stride;
    const void* ck;
    const void* cv;
    int n_pages, page_size;
    int page_rows;  // page_stride in rows of kv_dim
    int64_t kv_dim;
    const int32_t* table;
    int n_reqs, max_blocks;
    const int32_t* row_reqs;
    const int32_t* seq_lens;
    int n_heads, n_kv, group, head_dim;
    int chunks;  // chunks of G query heads per kv head
    float scale_log2;
    void* out;
    float* lse;
    float* part;  // [rows][heads][splits][2 + head_dim rounded up to 4]: m, l, -, -, acc
    int splits;
    int32_t* err;
};

__device__ __forceinline__ float load_elem(const void* p, int type, int64_t i) {
    if (type == CBX_TYPE_F32) return static_cast<const float*>(p)[i];
    if (type == CBX_TYPE_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_f(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int type, int64_t i, float v) {
    if (type == CBX_TYPE_F32) static_cast<float*>(p)[i] = v;
    else if (type == CBX_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v);
    else static_cast<__half*>(p)[i] = from_f<__half>(v);
}

// 2^(a - b) for the rescaling of a state with maximum a to maximum b >= a; a
// state without keys has a = -inf, l = 0, acc = 0 and weighs nothing.
__device__ __forceinline__ float rescale(float a, float b) {
    return a == -INFINITY ? 0.0f : ex2_approx(a - b);
}

// One state (m, l, acc) of a row and head.
constexpr int kStateHead = 4;  // floats before acc: m, l, two unused
__host__ __device__ inline int state_floats(int head_dim) { return kStateHead + head_dim; }

template <typename TC, int VL, int VPL, int G>
__global__ void __launch_bounds__(kThreads) k_paged_attention(AttnArgs a) {
    constexpr int EV = Vec<TC>::n;        // elements per 16-byte vector
    constexpr int EL = EV * VPL;          // elements of the head per lane
    constexpr int U = VL < 8 ? VL : 8;    // loads in flight
    constexpr int KPL = 32 / VL;          // keys per load
    constexpr int TILE = KPL * U;         // keys per warp and step
    extern __shared__ float smem[];       // [kWarps][G][state]
    const int split = blockIdx.x, hc = blockIdx.y, row = blockIdx.z;
    const int kvh = hc / a.chunks, chunk = hc % a.chunks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int vl = lane % VL, kg = lane / VL;
    const int hd = a.head_dim;
    const int head0 = kvh * a.group + chunk * G;
    const int heads = a.group - chunk * G < G ? a.group - chunk * G : G;
    grid_dep_wait();
    grid_dep_launch();

    int flags = 0;
    int req = a.row_reqs ? a.row_reqs[row] : row;
    int len = a.seq_lens[row];
    const int64_t cap = (int64_t)a.max_blocks * a.page_size;
    if (len < 0 || len > cap) {
        flags |= CBX_EFLAG_LENGTH;
        len = len < 0 ? 0 : (int)cap;
    }
    if (req < 0 || req >= a.n_reqs) {
        flags |= CBX_EFLAG_PAGE_OOB;
        req = 0;
        len = 0;
    }
    const int32_t* table = a.table + (int64_t)req * a.max_blocks;
    // This split's keys: whole tiles of the CTA, evenly over the splits.
    const int64_t step = (int64_t)TILE * kWarps;
    const int64_t tiles = (len + step - 1) / step;
    const int64_t lo = tiles * split / a.splits * step;
    int64_t hi64 = tiles * (split + 1) / a.splits * step;
    const int hi = hi64 < len ? (int)hi64 : len;

    // The query, scaled, this lane's elements.
    float q[G][EL], acc[G][EL], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int e = 0; e < EV; ++e) {
                const int i = (v * VL + vl) * EV + e;
                q[g][v * EV + e] = g < heads && i < hd
                    ? load_elem(a.q, a.q_type, (int64_t)row * a.q_stride + (int64_t)(head0 + g) * hd + i) * a.scale_log2
                    : 0.0f;
                acc[g][v * EV + e] = 0.0f;
            }
    }
    const bool live = vl * EV < hd;  // VPL > 1 only where every vector of every lane is tested below
    const char* kbase = static_cast<const char*>(a.ck) + ((int64_t)kvh * hd + vl * EV) * sizeof(TC);
    const char* vbase = static_cast<const char*>(a.cv) + ((int64_t)kvh * hd + vl * EV) * sizeof(TC);
    const int64_t row_bytes = a.kv_dim * (int64_t)sizeof(TC);

    // Of a tile's keys j * KPL + kg, the lane scores the one whose load index j
    // has its low bits reversed: the order the exchange below leaves.
    constexpr int kBits = U == 8 ? 3 : U == 4 ? 2 : U == 2 ? 1 : 0;
    int my_j = 0;
#pragma unroll
    for (int b = 0; b < kBits; ++b) my_j |= ((vl >> b) & 1) << (kBits - 1 - b);
    auto lane_of = [&](int j) {  // the lane of this key group that scores load j
        int r = 0;
#pragma unroll
        for (int b = 0; b < kBits; ++b) r |= ((j >> b) & 1) << (kBits - 1 - b);
        return kg * VL + r;
    };
    // Cache row of the key this lane scores in the tile at t0; -1: none.
    auto find = [&](int64_t t0) {
        const int64_t key = t0 + my_j * KPL + kg;
        if (key >= hi) return -1;
        const int blk = (int)key / a.page_size;
        const int page = __ldg(table + blk);
        if (page < 0 || page >= a.n_pages) {
            flags |= CBX_EFLAG_PAGE_OOB;
            return -1;
        }
        return page * a.page_rows + (int)key % a.page_size;
    };

    int64_t t0 = lo + (int64_t)warp * TILE;
    int slot = t0 < hi ? find(t0) : -1;
    for (; t0 < hi; t0 += step) {
        uint4 kr[U][VPL], vr[U][VPL];
        int s_of[U];
#pragma unroll
        for (int j = 0; j < U; ++j) s_of[j] = __shfl_sync(0xffffffffu, slot, lane_of(j));
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                kr[j][v] = make_uint4(0, 0, 0, 0);
                if (s_of[j] >= 0 && (VPL == 1 ? live : (v * VL + vl) * EV < hd))
                    kr[j][v] = __ldg(reinterpret_cast<const uint4*>(kbase + s_of[j] * row_bytes + v * VL * 16));
            }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                vr[j][v] = make_uint4(0, 0, 0, 0);
                if (s_of[j] >= 0 && (VPL == 1 ? live : (v * VL + vl) * EV < hd))
                    vr[j][v] = __ldg(reinterpret_cast<const uint4*>(vbase + s_of[j] * row_bytes + v * VL * 16));
            }
        const bool there = slot >= 0;
        if (t0 + step < hi) slot = find(t0 + step);
        float p[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float d[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                d[j] = 0.0f;
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    constexpr int kPer32 = 4 / (int)sizeof(TC);
                    float f[EV];
                    unpack32(kr[j][v].x, f, TC{});
                    unpack32(kr[j][v].y, f + kPer32, TC{});
                    unpack32(kr[j][v].z, f + 2 * kPer32, TC{});
                    unpack32(kr[j][v].w, f + 3 * kPer32, TC{});
#pragma unroll
                    for (int e = 0; e < EV; ++e) d[j] = fmaf(q[g][v * EV + e], f[e], d[j]);
                }
            }
            // Sum each d[j] over the VL lanes of its key: the lanes exchange
            // halves of the values until one is left, then add up.
            int n = U;
#pragma unroll
            for (int b = 0; b < kBits; ++b) {
                n >>= 1;
                const bool up = (lane >> b) & 1;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const float give = up ? d[i] : d[i + n], keep = up ? d[i + n] : d[i];
                    d[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1 << b);
                }
            }
#pragma unroll
            for (int o = U; o < VL; o <<= 1) d[0] += __shfl_xor_sync(0xffffffffu, d[0], o);
            const float s = there ? d[0] : -INFINITY;
            if (__any_sync(0xffffffffu, s > m[g])) {
                float t = fmaxf(s, m[g]);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
                const float c = rescale(m[g], t);
                m[g] = t;
                l[g] *= c;
#pragma unroll
                for (int e = 0; e < EL; ++e) acc[g][e] *= c;
            }
            p[g] = there ? ex2_approx(s - m[g]) : 0.0f;
            l[g] += p[g];
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float f[VPL][EV];
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                constexpr int kPer32 = 4 / (int)sizeof(TC);
                unpack32(vr[j][v].x, f[v], TC{});
                unpack32(vr[j][v].y, f[v] + kPer32, TC{});
                unpack32(vr[j][v].z, f[v] + 2 * kPer32, TC{});
                unpack32(vr[j][v].w, f[v] + 3 * kPer32, TC{});
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float w = __shfl_sync(0xffffffffu, p[g], lane_of(j));
#pragma unroll
                for (int v = 0; v < VPL; ++v)
#pragma unroll
                    for (int e = 0; e < EV; ++e) acc[g][v * EV + e] = fmaf(w, f[v][e], acc[g][v * EV + e]);
            }
        }
    }
    if (flags) atomicOr(a.err, flags);

    // Join the warp's key groups, then the CTA's warps.
    const int sf = state_floats(hd);
#pragma unroll
    for (int g = 0; g < G; ++g) {
        // each key's p is held by VL / U lanes: count one of them
        float t = vl < U ? l[g] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        l[g] = t;
#pragma unroll
        for (int e = 0; e < EL; ++e)
#pragma unroll
            for (int o = VL; o < 32; o <<= 1) acc[g][e] += __shfl_xor_sync(0xffffffffu, acc[g][e], o);
        float* st = smem + (warp * G + g) * sf;
        if (lane == 0) {
            st[0] = m[g];
            st[1] = l[g];
        }
        if (kg == 0) {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int e = 0; e < EV; ++e) {
                    const int i = (v * VL + vl) * EV + e;
                    if (i < hd) st[kStateHead + i] = acc[g][v * EV + e];
                }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * hd; i += kThreads) {
        const int g = i / hd, e = i % hd;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, smem[(w * G + g) * sf]);
        float ll = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* st = smem + (w * G + g) * sf;
            const float c = rescale(st[0], mm);
            ll += c * st[1];
            o += c * st[kStateHead + e];
        }
        const int64_t rh = (int64_t)row * a.n_heads + head0 + g;
        if (a.splits > 1) {
            float* st = a.part + (rh * a.splits + split) * sf;
            if (e == 0) {
                st[0] = mm;
                st[1] = ll;
            }
            st[kStateHead + e] = o;
        } else {
            store_elem(a.out, a.q_type, rh * hd + e, len > 0 && ll != 0.0f ? o / ll : 0.0f);
            if (a.lse && e == 0)
                a.lse[rh] = ll != 0.0f ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
        }
    }
}

// Joins the splits' states of one row and head.
__global__ void __launch_bounds__(128) k_paged_attention_join(AttnArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const int64_t rh = blockIdx.x;
    const int sf = state_floats(a.head_dim);
    const float* st = a.part + rh * a.splits * sf;
    float mm = -INFINITY;
    for (int s = 0; s < a.splits; ++s) mm = fmaxf(mm, st[s * sf]);
    float ll = 0.0f;
    for (int s = 0; s < a.splits; ++s) ll += rescale(st[s * sf], mm) * st[s * sf + 1];
    for (int e = threadIdx.x; e < a.head_dim; e += 128) {
        float o = 0.0f;
        for (int s = 0; s < a.splits; ++s) o += rescale(st[s * sf], mm) * st[s * sf + kStateHead + e];
        store_elem(a.out, a.q_type, rh * a.head_dim + e, ll != 0.0f ? o / ll : 0.0f);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[rh] = ll != 0.0f ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
}

int group_chunk(int group) { return group >= 3 ? 4 : group; }

int choose_splits(int64_t n_rows, int64_t n_kv, int group, int64_t max_keys) {
    const int gc = group_chunk(group);
    const int64_t ctas = n_rows * n_kv * ((group + gc - 1) / gc);
    int64_t s = (2 * num_sms() + ctas - 1) / ctas;
    const int64_t most = max_keys / kMinKeys;
    if (s > most) s = most;
    if (s > kMaxSplits) s = kMaxSplits;
    return s < 1 ? 1 : (int)s;
}

template <typename TC, int VL, int VPL, int G>
int run_attention(const AttnArgs& a, int64_t n_rows, cudaStream_t st) {
    const size_t smem = sizeof(float) * kWarps * G * state_floats(a.head_dim);
    auto kern = k_paged_attention<TC, VL, VPL, G>;
    const dim3 grid((unsigned)a.splits, (unsigned)(a.n_kv * a.chunks), (unsigned)n_rows);
    cudaError_t e = launch(kern, grid, dim3(kThreads), smem, st, a);
    if (e == cudaSuccess && a.splits > 1)
        e = launch(k_paged_attention_join, dim3((unsigned)(n_rows * a.n_heads)), dim3(128), 0, st, a);
    return launch_status(e, "cbx_paged_decode_attention");
}

template <typename TC, int VL, int VPL>
int run_group(const AttnArgs& a, int64_t n_rows, cudaStream_t st) {
    switch (group_chunk(a.group)) {
        case 1: return run_attention<TC, VL, VPL, 1>(a, n_rows, st);
        case 2: return run_attention<TC, VL, VPL, 2>(a, n_rows, st);
        default: return run_attention<TC, VL, VPL, 4>(a, n_rows, st);
    }
}

template <typename TC>
int run_head(const AttnArgs& a, int64_t n_rows, cudaStream_t st) {
    const int vecs = (a.head_dim + Vec<TC>::n - 1) / Vec<TC>::n;
    if (vecs <= 4) return run_group<TC, 4, 1>(a, n_rows, st);
    if (vecs <= 8) return run_group<TC, 8, 1>(a, n_rows, st);
    if (vecs <= 16) return run_group<TC, 16, 1>(a, n_rows, st);
    if (vecs <= 32) return run_group<TC, 32, 1>(a, n_rows, st);
    if constexpr (Vec<TC>::n == 4) return run_group<TC, 32, 2>(a, n_rows, st);
    return fail(CBX_ERR_INVALID_ARG, "cbx_paged_decode_attention: head_dim %d", a.head_dim);
}

// Sizes that the workspace query and the call check alike.
int check_sizes(const char* name, int64_t n_rows, int64_t n_heads, int64_t n_kv_heads,
                int64_t head_dim, int64_t max_blocks, int64_t page_size, int cache_type) {
    constexpr int64_t kInt = 2147483647;
    if (n_rows < 0 || n_rows > 65535)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_rows %lld outside [0, 65535]", name, (long long)n_rows);
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads > 65535 || n_heads % n_kv_heads)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_heads %lld is not a multiple of n_kv_heads %lld",
                    name, (long long)n_heads, (long long)n_kv_heads);
    if (head_dim < 8 || head_dim > 256 || head_dim % 8)
        return fail(CBX_ERR_INVALID_ARG, "%s: head_dim %lld is not a multiple of 8 up to 256", name,
                    (long long)head_dim);
    if (max_blocks <= 0 || page_size <= 0 || max_blocks > kInt || page_size > kInt)
        return fail(CBX_ERR_INVALID_ARG, "%s: max_blocks %lld page_size %lld", name,
                    (long long)max_blocks, (long long)page_size);
    if (!valid_type(cache_type))
        return fail(CBX_ERR_UNSUPPORTED_DTYPE, "%s: cache_type %d", name, cache_type);
    return CBX_OK;
}

int64_t workspace_bytes_of(int64_t n_rows, int64_t n_heads, int64_t head_dim, int splits) {
    return splits > 1 ? n_rows * n_heads * splits * state_floats((int)head_dim) * (int64_t)sizeof(float) : 0;
}

}  // namespace
}  // namespace cbx

extern "C" CBX_API int64_t cbx_paged_decode_attention_workspace(int64_t n_rows, int64_t n_heads,
                                                                int64_t n_kv_heads, int64_t head_dim,
                                                                int64_t max_blocks, int64_t page_size,
                                                                int cache_type) {
    using namespace cbx;
    const char* name = "cbx_paged_decode_attention_workspace";
    const int rc = check_sizes(name, n_rows, n_heads, n_kv_heads, head_dim, max_blocks, page_size, cache_type);
    if (rc != CBX_OK) return rc;
    ok();
    if (n_rows == 0) return 0;
    const int splits = choose_splits(n_rows, n_kv_heads, (int)(n_heads / n_kv_heads), max_blocks * page_size);
    return workspace_bytes_of(n_rows, n_heads, head_dim, splits);
}

extern "C" CBX_API int cbx_paged_decode_attention(
    const void* q, int q_type, int64_t q_row_stride, const void* cache_k, const void* cache_v,
    int cache_type, int64_t n_pages, int64_t page_size, int64_t page_stride, const int32_t* table,
    int64_t n_reqs, int64_t max_blocks, const int32_t* row_reqs, const int32_t* seq_lens,
    int64_t n_rows, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, float scale, void* out,
    float* lse, void* workspace, int64_t workspace_bytes, int32_t* err_word, cbx_stream_t stream) {
    using namespace cbx;
    const char* name = "cbx_paged_decode_attention";
    constexpr int64_t kInt = 2147483647;
    const int rc = check_sizes(name, n_rows, n_heads, n_kv_heads, head_dim, max_blocks, page_size, cache_type);
    if (rc != CBX_OK) return rc;
    if (!valid_type(q_type)) return fail(CBX_ERR_UNSUPPORTED_DTYPE, "%s: q_type %d", name, q_type);
    const int64_t kv_dim = n_kv_heads * head_dim;
    if (n_pages <= 0 || n_pages > kInt / page_size)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_pages %lld page_size %lld", name, (long long)n_pages,
                    (long long)page_size);
    if (page_stride == 0) page_stride = page_size * kv_dim;
    if (page_stride < page_size * kv_dim || page_stride % kv_dim)
        return fail(CBX_ERR_INVALID_ARG,
                    "%s: page_stride %lld is not a multiple of kv_dim %lld of at least page_size of them",
                    name, (long long)page_stride, (long long)kv_dim);
    if (page_stride / kv_dim > kInt / n_pages)
        return fail(CBX_ERR_INVALID_ARG, "%s: the cache has more than 2^31 - 1 rows", name);
    if (q_row_stride == 0) q_row_stride = n_heads * head_dim;
    if (q_row_stride < n_heads * head_dim)
        return fail(CBX_ERR_INVALID_ARG, "%s: q_row_stride %lld < n_heads * head_dim", name,
                    (long long)q_row_stride);
    if (n_reqs < 0 || n_reqs > kInt || (!row_reqs && n_reqs < n_rows))
        return fail(CBX_ERR_INVALID_ARG, "%s: n_reqs %lld for %lld rows", name, (long long)n_reqs,
                    (long long)n_rows);
    if (n_rows == 0) return ok();
    if (!q || !cache_k || !cache_v || !table || !seq_lens || !out || !err_word)
        return fail(CBX_ERR_INVALID_ARG, "%s: NULL argument", name);
    if (!aligned16(cache_k) || !aligned16(cache_v) ||
        (page_stride * type_size(cache_type)) % 16)
        return fail(CBX_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", name);
    const int group = (int)(n_heads / n_kv_heads);
    const int splits = choose_splits(n_rows, n_kv_heads, group, max_blocks * page_size);
    const int64_t need = workspace_bytes_of(n_rows, n_heads, head_dim, splits);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(CBX_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)",
                    name, (long long)(workspace ? workspace_bytes : 0), (long long)need);
    const int gc = group_chunk(group);
    AttnArgs a{q, q_type, q_row_stride, cache_k, cache_v, (int)n_pages, (int)page_size,
               (int)(page_stride / kv_dim), kv_dim, table, (int)n_reqs, (int)max_blocks, row_reqs,
               seq_lens, (int)n_heads, (int)n_kv_heads, group, (int)head_dim, (group + gc - 1) / gc,
               scale * kLog2e, out, lse, static_cast<float*>(workspace), splits, err_word};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (cache_type) {
        case CBX_TYPE_F32: return run_head<float>(a, n_rows, st);
        case CBX_TYPE_BF16: return run_head<__nv_bfloat16>(a, n_rows, st);
        default: return run_head<__half>(a, n_rows, st);
    }
}
