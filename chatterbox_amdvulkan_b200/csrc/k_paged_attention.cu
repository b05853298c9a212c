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
// head.  Three kernels, all with whole tiles of keys and values in flight per
// warp and no CTA barrier in the loop:
//  - k_attend_fma: one query head per kv head, two with an f32 cache, or heads
//    of more than 128 elements.  A key row of one kv head is VL 16-byte vectors,
//    one per lane, so a warp reads 32 / VL keys per load instruction.  f32 FMAs.
//  - k_attend_mma (16-bit caches) and k_attend_mma_f32: more query heads per kv
//    head, where the FMAs and the conversions to f32 would bound it.  mma.sync of
//    16 rows: the up to 8 query heads of a kv head, twice.
//
// The keys of a row are split over the CTAs of a cluster (up to 8), which join
// their states through distributed shared memory, or, where even that leaves
// SMs idle, over more CTAs with partial states in the workspace and a second
// launch that joins them.
#include "cbx_common.cuh"

namespace cbx {
namespace {

constexpr int kMaxCluster = 8;
constexpr int kMaxSplits = 64;

struct AttnArgs {
    const void* q;
    int q_type;
    int64_t q_stride;
    const void* ck;
    const void* cv;
    int n_pages, page_size, page_shift;  // page_shift: log2(page_size), -1 where it is none
    int page_rows;  // page_stride in rows of kv_dim
    int64_t kv_dim;
    const int32_t* table;
    int n_reqs, max_blocks;
    const int32_t* row_reqs;
    const int32_t* seq_lens;
    int n_heads, n_kv, group, head_dim;
    int chunks;  // chunks of query heads per kv head
    float scale_log2;
    void* out;
    float* lse;
    float* part;  // [rows][heads][splits][state]
    int splits;
    bool cluster;  // the splits are a cluster
    int32_t* err;
};

// Calls f with the query as a pointer of its type: the branch on the type is
// taken once, not between the loads, which then travel together.
template <typename F>
__device__ __forceinline__ void with_type(const void* p, int type, F f) {
    if (type == CBX_TYPE_F32) f(static_cast<const float*>(p));
    else if (type == CBX_TYPE_BF16) f(static_cast<const __nv_bfloat16*>(p));
    else f(static_cast<const __half*>(p));
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

// Natural logarithm of the sum that (m, l) stand for; -inf without keys.
__device__ __forceinline__ float lse_of(float m, float l) {
    return l != 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// Shared memory of the cluster's CTA `rank` at this CTA's address `p`.
__device__ __forceinline__ uint32_t peer_smem(uint32_t p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_peer(uint32_t p) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(p));
    return v;
}

// One state (m, l, acc) of a row and head.
constexpr int kStateHead = 4;  // floats before acc: m, l, two unused
__host__ __device__ inline int state_floats(int head_dim) { return kStateHead + head_dim; }

// What a CTA works on: a row, one kv head with up to G of its query heads, and
// one split's keys [lo, hi), whole steps of the CTA.  Splits lie side by side in
// the grid (a cluster), then the heads of a row, which read the same lines.
struct Work {
    int row, split, kvh, head0, heads, lo, hi;
    const int32_t* table;
    int flags;
    __device__ __forceinline__ Work(const AttnArgs& a, int chunk_heads, int step) {
        const int cta = blockIdx.x / a.splits, per_row = a.n_kv * a.chunks;
        split = blockIdx.x - cta * a.splits;
        row = cta / per_row;
        const int hc = cta - row * per_row;
        kvh = hc / a.chunks;
        const int first = (hc - kvh * a.chunks) * chunk_heads;
        head0 = kvh * a.group + first;
        heads = a.group - first < chunk_heads ? a.group - first : chunk_heads;
        flags = 0;
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
        table = a.table + (int64_t)req * a.max_blocks;
        const int64_t steps = ((int64_t)len + step - 1) / step;
        const int64_t from = steps * split / a.splits * step;
        const int64_t to = steps * (split + 1) / a.splits * step;
        lo = from < len ? (int)from : len;
        hi = to < len ? (int)to : len;
    }
    // Block of a key, and its table entry (0 behind the split's last key).
    __device__ __forceinline__ int block_of(const AttnArgs& a, int64_t key) const {
        return a.page_shift >= 0 ? (int)key >> a.page_shift : (int)key / a.page_size;
    }
    __device__ __forceinline__ int entry(const AttnArgs& a, int64_t key) const {
        return key < hi ? __ldg(table + block_of(a, key)) : 0;
    }
    // Cache row of a key, from its entry; -1 behind the split's last and on a bad page.
    __device__ __forceinline__ int row_of(const AttnArgs& a, int page, int64_t key) {
        if (key >= hi) return -1;
        if (page < 0 || page >= a.n_pages) {
            flags |= CBX_EFLAG_PAGE_OOB;
            return -1;
        }
        return page * a.page_rows + ((int)key - block_of(a, key) * a.page_size);
    }
    __device__ __forceinline__ int find(const AttnArgs& a, int64_t key) { return row_of(a, entry(a, key), key); }
};

// Joins the states [W][G][state] of the CTA's warps (in shared memory, written
// by all of them) and the CTAs of the row, and stores the result.
template <int W, int G>
__device__ __forceinline__ void finish(const AttnArgs& a, const Work& w, float* states) {
    const int hd = a.head_dim, sf = state_floats(hd);
    float* own = states + W * G * sf;  // [G][state] of this CTA
    __syncthreads();
    for (int i = threadIdx.x; i < w.heads * hd; i += W * 32) {
        const int g = i / hd, e = i % hd;
        float mm = -INFINITY;
#pragma unroll
        for (int k = 0; k < W; ++k) mm = fmaxf(mm, states[(k * G + g) * sf]);
        float ll = 0.0f, o = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float* st = states + (k * G + g) * sf;
            const float c = rescale(st[0], mm);
            ll += c * st[1];
            o += c * st[kStateHead + e];
        }
        const int64_t rh = (int64_t)w.row * a.n_heads + w.head0 + g;
        if (a.splits > 1) {
            float* st = a.cluster ? own + g * sf : a.part + (rh * a.splits + w.split) * sf;
            if (e == 0) {
                st[0] = mm;
                st[1] = ll;
            }
            st[kStateHead + e] = o;
        } else {
            store_elem(a.out, a.q_type, rh * hd + e, ll != 0.0f ? o / ll : 0.0f);
            if (a.lse && e == 0) a.lse[rh] = lse_of(mm, ll);
        }
    }
    if (!a.cluster) return;
    cluster_sync();
    // Each CTA of the cluster joins its share of the values.
    for (int i = w.split * (W * 32) + threadIdx.x; i < w.heads * hd; i += a.splits * (W * 32)) {
        const int g = i / hd, e = i % hd;
        const uint32_t st = smem_addr(own + g * sf);
        float m[kMaxCluster], l[kMaxCluster], v[kMaxCluster];
        float mm = -INFINITY;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k < a.splits) {
                const uint32_t peer = peer_smem(st, k);
                m[k] = ld_peer(peer);
                l[k] = ld_peer(peer + 4);
                v[k] = ld_peer(peer + 4 * (kStateHead + e));
                mm = fmaxf(mm, m[k]);
            }
        }
        float ll = 0.0f, o = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            if (k < a.splits) {
                const float c = rescale(m[k], mm);
                ll += c * l[k];
                o += c * v[k];
            }
        }
        const int64_t rh = (int64_t)w.row * a.n_heads + w.head0 + g;
        store_elem(a.out, a.q_type, rh * hd + e, ll != 0.0f ? o / ll : 0.0f);
        if (a.lse && e == 0) a.lse[rh] = lse_of(mm, ll);
    }
    cluster_sync();  // no CTA leaves while another reads its states
}

// 16 bytes to shared memory, zeros where !there.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t p) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t lds32(uint32_t p) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t p) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
    return v;
}

// The elements of a 16-byte vector as pairs of f32, for the packed FMAs.
template <typename TC, int N>
__device__ __forceinline__ void pairs_of(uint4 w, float2 (&f)[N], TC) {
    constexpr int k = 4 / (int)sizeof(TC);
    float g[2 * N];
    unpack32(w.x, g, TC{});
    unpack32(w.y, g + k, TC{});
    unpack32(w.z, g + 2 * k, TC{});
    unpack32(w.w, g + 3 * k, TC{});
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = make_float2(g[2 * i], g[2 * i + 1]);
}

// Shape of the FMA kernel.  With one or two query heads, a tile of keys and one
// of values wait in registers (8 loads each).  With more, the registers belong
// to the heads, so the loads go through a ring in shared memory, two tiles
// ahead: each lane copies and reads its own 16-byte cells, so no barrier is
// needed.
template <int VL, int VPL, bool RING>
struct Fma {
    static constexpr int kWarps = RING ? 4 : 8;
    static constexpr int kLoads = RING ? 4 : VL < 8 ? VL : 8;  // of keys, and of values, per tile
    static constexpr int kKeysPerLoad = 32 / VL;
    static constexpr int kTile = kKeysPerLoad * kLoads;        // keys per warp and step
    static constexpr int kStep = kTile * kWarps;
    static constexpr int kStages = 3;
    static constexpr int kRingBytes = RING ? kStages * 2 * kLoads * VPL * 512 : 0;  // of a warp
};
constexpr int kRingStep = 16;  // keys of a step with the ring, which takes head_dim above 128 only

template <typename TC, int VL, int VPL, int G, bool RING>
__global__ void __launch_bounds__(Fma<VL, VPL, RING>::kWarps * 32) k_attend_fma(AttnArgs a) {
    using Shape = Fma<VL, VPL, RING>;
    constexpr int EV = Vec<TC>::n;        // elements per 16-byte vector
    constexpr int EL = EV * VPL;          // elements of the head per lane
    constexpr int U = Shape::kLoads, KPL = Shape::kKeysPerLoad, TILE = Shape::kTile, step = Shape::kStep;
    static_assert(!RING || step == kRingStep, "choose_splits counts the ring's steps");
    extern __shared__ __align__(128) float smem[];  // rings, then states
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int vl = lane % VL, kg = lane / VL;
    const int hd = a.head_dim;
    grid_dep_wait();
    grid_dep_launch();
    Work w(a, G, step);
    const int hi = w.hi;

    const char* kbase = static_cast<const char*>(a.ck) + ((int64_t)w.kvh * hd + vl * EV) * sizeof(TC);
    const char* vbase = static_cast<const char*>(a.cv) + ((int64_t)w.kvh * hd + vl * EV) * sizeof(TC);
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
    const int my_key = my_j * KPL + kg;  // of a tile, the key this lane scores

    const uint32_t ring = smem_addr(smem) + warp * Shape::kRingBytes + lane * 16;
    auto cell = [&](int stage, int kv, int j, int v) { return ring + (((stage * 2 + kv) * U + j) * VPL + v) * 512; };
    // Sends the tile whose keys' rows the lanes hold on its way to a stage.
    auto fetch = [&](int stage, int rows) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = __shfl_sync(0xffffffffu, rows, lane_of(j));
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                const bool in = s >= 0 && (v * VL + vl) * EV < hd;
                const int64_t off = in ? s * row_bytes + v * VL * 16 : 0;
                copy16(cell(stage, 0, j, v), in ? kbase + off : static_cast<const char*>(a.ck), in);
                copy16(cell(stage, 1, j, v), in ? vbase + off : static_cast<const char*>(a.cv), in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // The first table entries and the query are on their way together; with the
    // ring, the first tiles too.
    int64_t t0 = w.lo + (int64_t)warp * TILE;
    const int entry0 = w.entry(a, t0 + my_key);
    int slot = -1, slot1 = -1, slot2 = -1, stage = 0;  // cache rows of this tile and the next two
    if constexpr (RING) {
        const int entry1 = w.entry(a, t0 + step + my_key), entry2 = w.entry(a, t0 + 2 * step + my_key);
        slot = w.row_of(a, entry0, t0 + my_key);
        slot1 = w.row_of(a, entry1, t0 + step + my_key);
        slot2 = w.row_of(a, entry2, t0 + 2 * step + my_key);
        fetch(0, slot);
        fetch(1, slot1);
    }
    // The query, scaled, this lane's elements.
    float2 q[G][EL / 2], acc[G][EL / 2];
    float m[G], l[G];
    with_type(a.q, a.q_type, [&](auto* p) {
        p += (int64_t)w.row * a.q_stride + (int64_t)w.head0 * hd;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int v = 0; v < VPL; ++v)
#pragma unroll
                for (int e = 0; e < EV; e += 2) {
                    const int i = (v * VL + vl) * EV + e;  // head_dim is even: both or neither
                    const bool in = g < w.heads && i < hd;
                    q[g][(v * EV + e) / 2] = make_float2(in ? to_f(p[g * hd + i]) : 0.0f, in ? to_f(p[g * hd + i + 1]) : 0.0f);
                }
    });
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < EL / 2; ++e) {
            q[g][e] = __fmul2_rn(q[g][e], pair(a.scale_log2));
            acc[g][e] = pair(0.0f);
        }
    }
    if constexpr (!RING) slot = w.row_of(a, entry0, t0 + my_key);

    for (; t0 < hi; t0 += step) {
        uint4 kr[U][VPL], vr[U][VPL];
        const bool there = slot >= 0;
        auto landed = [&](int kv, int j, int v) { return lds16(cell(stage, kv, j, v)); };
        if constexpr (RING) {
            fetch(stage == 0 ? 2 : stage - 1, slot2);
            asm volatile("cp.async.wait_group 2;" ::: "memory");
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int v = 0; v < VPL; ++v) kr[j][v] = landed(0, j, v);
            slot = slot1;
            slot1 = slot2;
            slot2 = w.find(a, t0 + 3 * step + my_key);
        } else {
            int s_of[U];
#pragma unroll
            for (int j = 0; j < U; ++j) s_of[j] = __shfl_sync(0xffffffffu, slot, lane_of(j));
            auto load = [&](const char* base, int j, int v) {
                const bool in = (v * VL + vl) * EV < hd;
                return s_of[j] >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(base + s_of[j] * row_bytes + v * VL * 16))
                                          : make_uint4(0, 0, 0, 0);
            };
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int v = 0; v < VPL; ++v) kr[j][v] = load(kbase, j, v);
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int v = 0; v < VPL; ++v) vr[j][v] = load(vbase, j, v);
            if (t0 + step < hi) slot = w.find(a, t0 + step + my_key);
        }
        float p[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float d[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float2 sum = pair(0.0f);
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    float2 f[EV / 2];
                    pairs_of(kr[j][v], f, TC{});
#pragma unroll
                    for (int e = 0; e < EV / 2; ++e) sum = __ffma2_rn(q[g][v * EV / 2 + e], f[e], sum);
                }
                d[j] = sum.x + sum.y;
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
                for (int e = 0; e < EL / 2; ++e) acc[g][e] = __fmul2_rn(acc[g][e], pair(c));
            }
            p[g] = s == -INFINITY ? 0.0f : ex2_approx(s - m[g]);  // whatever m is: it may be -inf too
            l[g] += p[g];
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float2 f[VPL][EV / 2];
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                if constexpr (RING) vr[j][v] = landed(1, j, v);
                pairs_of(vr[j][v], f[v], TC{});
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float w = __shfl_sync(0xffffffffu, p[g], lane_of(j));
#pragma unroll
                for (int v = 0; v < VPL; ++v)
#pragma unroll
                    for (int e = 0; e < EV / 2; ++e)
                        acc[g][v * EV / 2 + e] = __ffma2_rn(pair(w), f[v][e], acc[g][v * EV / 2 + e]);
            }
        }
        if (RING) stage = stage == 2 ? 0 : stage + 1;
    }
    if (w.flags) atomicOr(a.err, w.flags);
    if constexpr (RING) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // Join the warp's key groups, then the CTA's warps.
    const int sf = state_floats(hd);
    float* states = smem + Shape::kRingBytes / 4 * Shape::kWarps;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        // each key's p is held by VL / U lanes: count one of them
        float t = vl < U ? l[g] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        l[g] = t;
#pragma unroll
        for (int e = 0; e < EL / 2; ++e)
#pragma unroll
            for (int o = VL; o < 32; o <<= 1) {
                acc[g][e].x += __shfl_xor_sync(0xffffffffu, acc[g][e].x, o);
                acc[g][e].y += __shfl_xor_sync(0xffffffffu, acc[g][e].y, o);
            }
        float* st = states + (warp * G + g) * sf;
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
                    if (i < hd) st[kStateHead + i] = e & 1 ? acc[g][(v * EV + e) / 2].y : acc[g][(v * EV + e) / 2].x;
                }
        }
    }
    finish<Shape::kWarps, G>(a, w, states);
}

// ---------------------------------------------------------- tensor cores --

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Splits (x, y) into N terms of T, each the rounded rest of those before.
template <typename T, int N>
__device__ __forceinline__ void terms_of(float x, float y, uint32_t (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float f[2] = {x, y};
        t[i] = pack32(f, T{});
        float r[2];
        unpack32(t[i], r, T{});
        x -= r[0];
        y -= r[1];
    }
}

// P as the products take it: terms of p, of p times kScale for f16, whose second
// term is times kSecond more.
template <typename T, int N>
struct Terms {
    static constexpr bool f16 = __is_same(T, __half);
    static_assert(!f16 || N == 2, "P in f16 is two terms");
    static constexpr float kScale = f16 ? 32768.0f : 1.0f, kSecond = f16 ? 4096.0f : 1.0f;
    static __device__ __forceinline__ void of(float x, float y, uint32_t (&t)[N]) {
        if constexpr (f16) {
            const float f[2] = {x * kScale, y * kScale};
            t[0] = pack32(f, T{});
            float r[2];
            unpack32(t[0], r, T{});
            const float s[2] = {(f[0] - r[0]) * kSecond, (f[1] - r[1]) * kSecond};
            t[1] = pack32(s, T{});
        } else {
            terms_of<T, N>(x, y, t);
        }
    }
    // The value that the sums of the first (and third) and of the second terms stand for.
    static __device__ __forceinline__ float sum(float first, float second) {
        return (first + second * (1.0f / kSecond)) * (1.0f / kScale);
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p) : "memory");
}

constexpr int kMmaWarps = 4;
constexpr int kMmaHeads = 8;   // query heads of a CTA
constexpr int kMmaTile = 16;   // keys per warp and step
constexpr int kMmaStages = 3;  // tiles of a warp in shared memory

template <int HD>
__host__ __device__ constexpr int mma_ring_bytes() {  // of a warp: K and V tiles
    return kMmaStages * 2 * kMmaTile * HD * 2;
}
// CTAs per SM, by registers (f32 queries take 3 terms on bf16 caches) and shared memory.
__host__ __device__ constexpr int mma_per_sm(int head_dim, bool f16) {
    return head_dim > 64 ? 2 : f16 ? 4 : 3;
}

// S = Q K^T and O = P V by m16n8k16 products, for heads of up to W elements; the
// rows of the rings are HD elements long.  Rows 0-7 of the first operand
// are the first 16-bit term of the 8 heads' values, rows 8-15 the second: Q and
// P are f32 values written as sums of 16-bit ones, so that the products are as
// exact as f32 ones where the result is.
//   QT terms of q: 1 where q has the cache's type; otherwise 3 of bf16 (24 bits)
//     or 2 of f16 (22 bits; q is brought to [2^10, 2^11) by a power of two, so
//     that the second term of all but tiny elements is a normal number).
//   PT terms of p: 2 for a 16-bit result (16 or 22 bits), 3 of bf16 for f32.  f16
//     holds p times 2^15 and the second term times 2^12 more, as p is at most 1 and
//     f16 has no exponents below 2^-24: 22 bits down to p = 2^-29, 2^-51 of the row's
//     largest below.  Unscaled, probabilities below 2^-25 would be lost.
// A third term is a second product on the same accumulators.
// Each warp streams its own tiles through a ring in shared memory (cp.async, 16
// bytes a lane, consecutive lanes on consecutive bytes of a key's row), so no
// CTA barrier stands in the loop, and two tiles are on their way while one is
// worked on.  Loading the operands' layouts straight from global memory moved
// the same bytes in 4 times the requests (quarter lines of V): 122 us for one
// row of 65,537 keys, 32 heads over 8 of 128 in bf16, against 57 us with the
// ring (both with the first form of the join; 50 us, 5.4 TB/s, now).  f32 FMAs
// with 4 heads a CTA took 107 us there.  The 16-byte vectors of a row are permuted by the
// row's number, which keeps ldmatrix free of bank conflicts.
template <typename T, int HD, int W, int QT, int PT>
__global__ void __launch_bounds__(kMmaWarps * 32, mma_per_sm(HD, __is_same(T, __half))) k_attend_mma(AttnArgs a) {
    constexpr int KS = W / 16;    // products over the head
    constexpr int VECS = W / 8;   // 16-byte vectors of a row
    constexpr int step = kMmaTile * kMmaWarps;
    extern __shared__ __align__(128) float smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hd = a.head_dim, vecs = hd / 8;
    grid_dep_wait();
    grid_dep_launch();
    Work w(a, kMmaHeads, step);

    float o[VECS][4] = {};
    float m = -INFINITY, l = 0.0f;  // head g
    const char* kbase = static_cast<const char*>(a.ck) + (int64_t)w.kvh * hd * 2;
    const char* vbase = static_cast<const char*>(a.cv) + (int64_t)w.kvh * hd * 2;
    const int64_t row_bytes = a.kv_dim * 2;
    constexpr uint32_t kTileBytes = kMmaTile * HD * 2;
    const uint32_t ring = smem_addr(smem) + warp * mma_ring_bytes<HD>();

    // Puts the tile at t0 in a stage; returns which of its keys are there.
    auto fetch = [&](int64_t t0, int stage, int slot) {
        const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0) & 0xffffu;
        if (t0 < w.hi) {
            constexpr int kCells = HD / 8, kRows = 32 / kCells;  // rows per instruction
            const int r0 = lane / kCells, c = lane % kCells;
            const uint32_t dst = ring + stage * 2 * kTileBytes;
#pragma unroll
            for (int i = 0; i < kMmaTile / kRows; ++i) {
                const int r = i * kRows + r0;
                const int s = __shfl_sync(0xffffffffu, slot, r);
                const bool in = s >= 0 && c < vecs;
                const int64_t off = in ? s * row_bytes + c * 16 : 0;
                const uint32_t at = dst + r * (HD * 2) + ((c ^ (r & 7)) << 4);
                copy16(at, kbase + off, in);
                copy16(at + kTileBytes, vbase + off, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return there;
    };

    const int64_t first = w.lo + (int64_t)warp * kMmaTile;
    uint64_t there = 0;  // 16 bits for each tile on its way, the oldest on top
    int entries[kMmaStages], slot = -1;
#pragma unroll
    for (int s = 0; s < kMmaStages; ++s) entries[s] = w.entry(a, first + (int64_t)s * step + (lane & 15));
#pragma unroll
    for (int s = 0; s < kMmaStages; ++s) {
        slot = w.row_of(a, entries[s], first + (int64_t)s * step + (lane & 15));
        if (s < kMmaStages - 1) there = there << 16 | fetch(first + (int64_t)s * step, s, slot);
    }
    // The first operand of S: head g.
    uint32_t qf[QT][KS][2];
    float scale = a.scale_log2;
    {
        float x[KS][4], most = 0.0f;
        with_type(a.q, a.q_type, [&](auto* p) {
            p += (int64_t)w.row * a.q_stride + (int64_t)(w.head0 + g) * hd;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 16 * s + (e >> 1) * 8 + 2 * t + (e & 1);
                    x[s][e] = g < w.heads && i < hd ? to_f(p[i]) : 0.0f;
                }
        });
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[s][e]));
        if constexpr (QT == 2) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            if (most > 0.0f && most < INFINITY) {
                int e = 264 - (int)(__float_as_uint(most) >> 23);  // biased exponent of the power
                if (e > 253) e = 253;
                const float up = __uint_as_float((uint32_t)e << 23);
                scale *= __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[s][i] *= up;
            }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t f[QT];
                terms_of<T, QT>(x[s][2 * e], x[s][2 * e + 1], f);
#pragma unroll
                for (int k = 0; k < QT; ++k) qf[k][s][e] = f[k];
            }
    }
    int stage = 0;
    for (int64_t t0 = first; t0 < w.hi; t0 += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kMmaStages - 2) : "memory");
        __syncwarp();  // all lanes' copies have landed, and all have left the stage that is filled next
        int next = stage + kMmaStages - 1;
        if (next >= kMmaStages) next -= kMmaStages;
        there = there << 16 | fetch(t0 + (int64_t)(kMmaStages - 1) * step, next, slot);
        slot = w.find(a, t0 + (int64_t)kMmaStages * step + (lane & 15));
        const uint32_t keys = (uint32_t)(there >> (16 * (kMmaStages - 1))) & 0xffffu;
        const uint32_t kt = ring + stage * 2 * kTileBytes, vt = kt + kTileBytes;
        if (++stage == kMmaStages) stage = 0;

        // Scores of head g: keys 2t, 2t + 1 of the first 8, and of the second.
        float s[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float c[2][4] = {};
#pragma unroll
            for (int q = 0; q < KS; q += 2) {
                uint32_t b[4];
                ldmatrix4(b, kt + (n * 8 + (lane & 7)) * (HD * 2) + (((2 * q + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma16816(c[h], qf[0][q + h][0], QT > 1 ? qf[QT > 1][q + h][0] : 0u, qf[0][q + h][1],
                             QT > 1 ? qf[QT > 1][q + h][1] : 0u, b[2 * h], b[2 * h + 1], T{});
                    if constexpr (QT > 2) mma16816(c[h], qf[2][q + h][0], 0u, qf[2][q + h][1], 0u, b[2 * h], b[2 * h + 1], T{});
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float v = c[0][k] + c[1][k];
                s[2 * n + k] = QT > 1 ? v + (c[0][k + 2] + c[1][k + 2]) : v;
            }
        }
        float best = m;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = keys >> (2 * t + (i & 1) + (i >> 1) * 8) & 1;
            s[i] = in ? s[i] * scale : -INFINITY;
            best = fmaxf(best, s[i]);
            if (QT > 1) odd |= s[i] != s[i];
        }
        if (__any_sync(0xffffffffu, best > m || odd)) {
            // An infinite key times a term of q that is 0 is a NaN, and so is the sum with
            // one of the other sign: such a tile is scored again by f32 FMAs.
            if (QT > 1 && __any_sync(0xffffffffu, odd)) {
                with_type(a.q, a.q_type, [&](auto* p) {
                    p += (int64_t)w.row * a.q_stride + (int64_t)(w.head0 + g) * hd;
                    for (int n = 0; n < 4; ++n) {
                        const int r = (n >> 1) * 8 + 2 * t + (n & 1);
                        float sum = 0.0f;
                        for (int i = 0; i < hd && g < w.heads; i += 2) {
                            float k[2];
                            unpack32(lds32(kt + r * (HD * 2) + (((i >> 3) ^ (r & 7)) << 4) + (i & 7) * 2), k, T{});
                            sum = fmaf(to_f(p[i + 1]), k[1], fmaf(to_f(p[i]), k[0], sum));
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k == n) s[k] = keys >> r & 1 ? sum * a.scale_log2 : -INFINITY;
                    }
                });
#pragma unroll
                for (int i = 0; i < 4; ++i) best = fmaxf(best, s[i]);
            }
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
            const float c = rescale(m, best);
            m = best;
            l *= c;
#pragma unroll
            for (int j = 0; j < VECS; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][k] *= c;
        }
        uint32_t pf[2][PT];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float p0 = s[2 * n] == -INFINITY ? 0.0f : ex2_approx(s[2 * n] - m);
            const float p1 = s[2 * n + 1] == -INFINITY ? 0.0f : ex2_approx(s[2 * n + 1] - m);
            l += p0 + p1;
            Terms<T, PT>::of(p0, p1, pf[n]);
        }
#pragma unroll
        for (int j = 0; j < VECS; j += 2) {
            uint32_t b[4];
            ldmatrix4_trans(b, vt + (lane & 15) * (HD * 2) + (((j + (lane >> 4)) ^ (lane & 7)) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // The products truncate what they add up: the first terms' sums start
                // anew each tile and are added with rounding (-3 to 6 % of the time; one
                // CTA over 65,536 keys: off by less than 1e-5, not 1.1e-4).
                float d[4] = {0.0f, 0.0f, o[j + h][2], o[j + h][3]};
                mma16816(d, pf[0][0], pf[0][1], pf[1][0], pf[1][1], b[2 * h], b[2 * h + 1], T{});
                if constexpr (PT > 2) mma16816(d, pf[0][2], 0u, pf[1][2], 0u, b[2 * h], b[2 * h + 1], T{});
                o[j + h][0] += d[0];
                o[j + h][1] += d[1];
                o[j + h][2] = d[2];
                o[j + h][3] = d[3];
            }
        }
    }
    if (w.flags) atomicOr(a.err, w.flags);

    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the states take the rings' place
    float* st = smem + (warp * kMmaHeads + g) * state_floats(hd);
    if (t == 0) {
        st[0] = m;
        st[1] = l;
    }
#pragma unroll
    for (int j = 0; j < VECS; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = 8 * j + 2 * t + k;
            if (e < hd) st[kStateHead + e] = Terms<T, PT>::sum(o[j][k], o[j][k + 2]);
        }
    finish<kMmaWarps, kMmaHeads>(a, w, smem);
}

__device__ __forceinline__ void mma1688(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two tf32 terms of f32 values.  By truncation (2.5 instructions a value): 11
// bits each, so less than 2^-21 of the value is lost, and nothing overflows.
// Rounded: at most 2^-24 is lost, but cvt takes several instructions (with it for
// all values the first two cases below took 57.9 and 157 us): for the query, split
// once, and P, of which a tile has few.
__device__ __forceinline__ void tf32_rounded(float x, uint32_t* t) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(t[0]) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(t[1]) : "f"(x - __uint_as_float(t[0])));
}
__device__ __forceinline__ void tf32_terms(float x, float y, uint32_t (&t)[2][2]) {
    t[0][0] = __float_as_uint(x) & 0xffffe000u;
    t[1][0] = __float_as_uint(y) & 0xffffe000u;
    const float2 r = __ffma2_rn(make_float2(__uint_as_float(t[0][0]), __uint_as_float(t[1][0])), pair(-1.0f), make_float2(x, y));
    t[0][1] = __float_as_uint(r.x) & 0xffffe000u;
    t[1][1] = __float_as_uint(r.y) & 0xffffe000u;
}

// Shape of the f32 form: KEYS per warp and step (16 of up to 64 elements, 8 of
// more), two tiles of a warp in shared memory, and CTAs per SM, by registers.
// In us (B200), with 2 / 3 / 4 CTAs per SM:
//   94 rows of 2511 keys, 16 heads over 2 of 64     61.6 / 49.8 / 61.3 (241 MB: 4.8 TB/s)
//   40 rows of 4000 keys, 32 heads over 4 of 128    141 / 158 / 233 (655 MB: 4.7 TB/s)
//   64 rows of 2000 keys, 16 heads over 4 of 32     34.3 / 34.3 / 30.6
// Three tiles, or 8 keys of 64 elements or 16 of 128, were no faster.
template <int HD>
struct MmaF32 {
    static constexpr int kKeys = HD <= 64 ? 16 : 8;
    static constexpr int kStages = 2;
    static constexpr int kPerSM = HD <= 32 ? 4 : HD <= 64 ? 3 : 2;
    static constexpr int kTileBytes = kKeys * HD * 4;            // of K, and of V
    static constexpr int kRingBytes = kStages * 2 * kTileBytes;  // of a warp
    static constexpr int kStep = kKeys * kMmaWarps;
};

// The same for f32 caches, by m16n8k8 products of tf32: every value is the sum of
// two tf32 terms, rows 0-7 of the first operand are the heads' first terms, rows
// 8-15 their second ones, and the second operand's terms take a product each.
// Lanes read 16 bytes at a time and split them in registers:
//   K: elements 4t .. 4t + 3 of 16 are k = t and t + 4 of two products (the query's
//     elements are taken in the same order);
//   V: keys 2t and 2t + 1 of 8 are k = t and t + 4, as the scores lie, and elements
//     4g .. 4g + 3 of 32 are column g of four products.
// The vectors of a row are permuted so that the 8 lanes of a shared-memory
// access meet no bank twice.  The terms of an infinite key are NaN: a tile with a
// NaN score is scored again by f32 FMAs.
// Against f32 FMAs with four heads a CTA, in us (B200): 94 rows of 2511 keys, 16
// heads over 2 of 64, 50 / 99, 8 heads over 2, 48 / 82; 40 rows of 4000 keys, 32 heads
// over 4 of 128, 141 / 281; 300 rows of 500 keys, 64 heads over 4 of 64, 110 / 207.
// With two heads the FMAs are faster: 40 rows, 8 over 4 of 128, 128 / 105; and with
// a few keys, as the long code has to be fetched: 6 rows of 13 keys, 16 over 2 of
// 128, 6.9 / 4.8 (the host knows the tables' size only, not the lengths).  Three
// bf16 terms a value, which lose nothing, take 11 instructions a pair: 55.6 and 175
// us for the first and third.  What bounds it is latency: of the splits and of
// products that wait for one another, at 12 warps an SM (issue slots 47 % busy,
// tensor pipe 32 %); the registers leave no room for more.
template <int HD, int W>
__global__ void __launch_bounds__(kMmaWarps * 32, MmaF32<HD>::kPerSM) k_attend_mma_f32(AttnArgs a) {
    using Shape = MmaF32<HD>;
    constexpr int KS = W / 16, KEYS = Shape::kKeys, NT = KEYS / 8, STAGES = Shape::kStages;
    constexpr int step = Shape::kStep;
    extern __shared__ __align__(128) float smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hd = a.head_dim, vecs = hd / 4;
    grid_dep_wait();
    grid_dep_launch();
    Work w(a, kMmaHeads, step);

    float o[W / 8][4] = {};  // [4 b + c]: elements 32 b + 4 n + c, n = 2t and 2t + 1
    float m = -INFINITY, l = 0.0f;  // head g
    const char* kbase = static_cast<const char*>(a.ck) + (int64_t)w.kvh * hd * 4;
    const char* vbase = static_cast<const char*>(a.cv) + (int64_t)w.kvh * hd * 4;
    const int64_t row_bytes = a.kv_dim * 4;
    constexpr uint32_t kTileBytes = Shape::kTileBytes;
    const uint32_t ring = smem_addr(smem) + warp * Shape::kRingBytes;
    auto k_cell = [](int r, int c) { return (uint32_t)(r * HD * 4 + ((c ^ ((r & 1) << 2)) << 4)); };
    auto v_cell = [](int r, int c) { return (uint32_t)(r * HD * 4 + ((c ^ (r & 7)) << 4)); };

    // Puts the tile at t0 in a stage; returns which of its keys are there.
    auto fetch = [&](int64_t t0, int stage, int slot) {
        const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0) & ((1u << KEYS) - 1);
        if (t0 < w.hi) {
            constexpr int kCells = HD / 4, kRows = 32 / kCells;  // rows per instruction
            const int r0 = lane / kCells, c = lane % kCells;
            const uint32_t dst = ring + stage * 2 * kTileBytes;
#pragma unroll
            for (int i = 0; i < KEYS / kRows; ++i) {
                const int r = i * kRows + r0;
                const int s = __shfl_sync(0xffffffffu, slot, r);
                const bool in = s >= 0 && c < vecs;
                const int64_t off = in ? s * row_bytes + c * 16 : 0;
                copy16(dst + k_cell(r, c), kbase + off, in);
                copy16(dst + kTileBytes + v_cell(r, c), vbase + off, in);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return there;
    };

    const int64_t first = w.lo + (int64_t)warp * KEYS;
    const int my_key = lane & (KEYS - 1);
    uint64_t there = 0;  // 16 bits for each tile on its way, the oldest on top
    int entries[STAGES], slot = -1;
#pragma unroll
    for (int s = 0; s < STAGES; ++s) entries[s] = w.entry(a, first + (int64_t)s * step + my_key);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
        slot = w.row_of(a, entries[s], first + (int64_t)s * step + my_key);
        if (s < STAGES - 1) there = there << 16 | fetch(first + (int64_t)s * step, s, slot);
    }
    // Head g's query.
    uint32_t qf[KS][2][4];
    with_type(a.q, a.q_type, [&](auto* p) {
        p += (int64_t)w.row * a.q_stride + (int64_t)(w.head0 + g) * hd;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 16 * s + 4 * t + 2 * h;  // head_dim is even: both or neither
                const bool in = g < w.heads && i < hd;
                tf32_rounded(in ? to_f(p[i]) : 0.0f, qf[s][h]);
                tf32_rounded(in ? to_f(p[i + 1]) : 0.0f, qf[s][h] + 2);
            }
    });
    int stage = 0;
    for (int64_t t0 = first; t0 < w.hi; t0 += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();  // all lanes' copies have landed, and all have left the stage that is filled next
        int next = stage + STAGES - 1;
        if (next >= STAGES) next -= STAGES;
        there = there << 16 | fetch(t0 + (int64_t)(STAGES - 1) * step, next, slot);
        slot = w.find(a, t0 + (int64_t)STAGES * step + my_key);
        const uint32_t keys = (uint32_t)(there >> (16 * (STAGES - 1))) & 0xffffu;
        const uint32_t kt = ring + stage * 2 * kTileBytes, vt = kt + kTileBytes;
        if (++stage == STAGES) stage = 0;

        // Scores of head g: keys 8n + 2t, 8n + 2t + 1.
        float s[NT][2];
        bool odd = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float c[2][4] = {};  // the large products, the small ones
#pragma unroll
            for (int q = 0; q < KS; ++q) {
                const uint4 x = lds16(kt + k_cell(n * 8 + g, 4 * q + t));
                uint32_t b[2][2][2];
                tf32_terms(__uint_as_float(x.x), __uint_as_float(x.y), b[0]);
                tf32_terms(__uint_as_float(x.z), __uint_as_float(x.w), b[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k) mma1688(c[k], qf[q][h], b[h][0][k], b[h][1][k]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                s[n][k] = (c[0][k] + c[0][k + 2]) + (c[1][k] + c[1][k + 2]);
                odd |= s[n][k] != s[n][k];
            }
        }
        if (__any_sync(0xffffffffu, odd)) {
            with_type(a.q, a.q_type, [&](auto* p) {
                p += (int64_t)w.row * a.q_stride + (int64_t)(w.head0 + g) * hd;
                for (int n = 0; n < 2 * NT; ++n) {
                    const int r = (n >> 1) * 8 + 2 * t + (n & 1);
                    float sum = 0.0f;
                    for (int i = 0; i < hd && g < w.heads; ++i)
                        sum = fmaf(to_f(p[i]), lds_f32(kt + k_cell(r, i >> 2) + (i & 3) * 4), sum);
#pragma unroll
                    for (int k = 0; k < 2 * NT; ++k)
                        if (k == n) s[k >> 1][k & 1] = sum;
                }
            });
        }
        float best = m;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const bool in = keys >> (8 * n + 2 * t + k) & 1;
                s[n][k] = in ? s[n][k] * a.scale_log2 : -INFINITY;
                best = fmaxf(best, s[n][k]);
            }
        if (__any_sync(0xffffffffu, best > m)) {
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
            const float c = rescale(m, best);
            m = best;
            l *= c;
#pragma unroll
            for (int j = 0; j < W / 8; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][k] *= c;
        }
        uint32_t pf[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float p0 = s[n][0] == -INFINITY ? 0.0f : ex2_approx(s[n][0] - m);
            const float p1 = s[n][1] == -INFINITY ? 0.0f : ex2_approx(s[n][1] - m);
            l += p0 + p1;
            tf32_rounded(p0, pf[n]);
            tf32_rounded(p1, pf[n] + 2);
        }
#pragma unroll
        for (int b = 0; b < W / 32; ++b) {
            // The products truncate what they add up: the first terms' sums start
            // anew each tile and are added with rounding (2.5 % of the time; 12 rows
            // of 4693 keys, 80 heads over 16 of 72: off by 1.1e-6, not 6.4e-6).
            float d[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                d[c][0] = d[c][1] = 0.0f;
                d[c][2] = o[4 * b + c][2];
                d[c][3] = o[4 * b + c][3];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 x = lds16(vt + v_cell(8 * n + 2 * t, 8 * b + g)), y = lds16(vt + v_cell(8 * n + 2 * t + 1, 8 * b + g));
                const uint32_t v[4][2] = {{x.x, y.x}, {x.y, y.y}, {x.z, y.z}, {x.w, y.w}};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t f[2][2];
                    tf32_terms(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]), f);
#pragma unroll
                    for (int k = 0; k < 2; ++k) mma1688(d[c], pf[n], f[0][k], f[1][k]);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                o[4 * b + c][0] += d[c][0];
                o[4 * b + c][1] += d[c][1];
                o[4 * b + c][2] = d[c][2];
                o[4 * b + c][3] = d[c][3];
            }
        }
    }
    if (w.flags) atomicOr(a.err, w.flags);

    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the states take the rings' place
    float* st = smem + (warp * kMmaHeads + g) * state_floats(hd);
    if (t == 0) {
        st[0] = m;
        st[1] = l;
    }
#pragma unroll
    for (int j = 0; j < W / 8; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = 32 * (j >> 2) + 4 * (2 * t + k) + (j & 3);
            if (e < hd) st[kStateHead + e] = o[j][k] + o[j][k + 2];
        }
    finish<kMmaWarps, kMmaHeads>(a, w, smem);
}

// Joins the splits' states of one row and head: first the weight of each split,
// then the values, 16 bytes a load, the splits shared by the threads so that a
// thread's few loads travel together (one thread for all splits of an element
// took 11 us for 36 splits, 32 us for 60).
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) k_attend_join(AttnArgs a) {
    __shared__ float weight[kMaxSplits];
    __shared__ float4 sums[kJoinThreads];
    grid_dep_wait();
    grid_dep_launch();
    const int64_t rh = blockIdx.x;
    const int sf = state_floats(a.head_dim), lane = threadIdx.x & 31;
    const int vecs = a.head_dim / 4, parts = kJoinThreads / vecs;  // head_dim is 8 .. 256
    const int v = threadIdx.x % vecs, part = threadIdx.x / vecs;
    const float* st = a.part + rh * a.splits * sf;
    // every warp for itself: kMaxSplits / 32 splits a lane
    float m[kMaxSplits / 32], l[kMaxSplits / 32], mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
        const int s = i * 32 + lane;
        m[i] = s < a.splits ? st[s * sf] : -INFINITY;
        l[i] = s < a.splits ? st[s * sf + 1] : 0.0f;
        mm = fmaxf(mm, m[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; ++i) {
        const float c = rescale(m[i], mm);
        ll += c * l[i];
        if (threadIdx.x < 32) weight[i * 32 + lane] = c;
    }
    ll = warp_sum(ll);
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (part < parts) {
#pragma unroll 4
        for (int s = part; s < a.splits; s += parts) {
            const float4 x = *reinterpret_cast<const float4*>(st + s * sf + kStateHead + 4 * v);
            const float c = weight[s];
            o = make_float4(fmaf(c, x.x, o.x), fmaf(c, x.y, o.y), fmaf(c, x.z, o.z), fmaf(c, x.w, o.w));
        }
        sums[threadIdx.x] = o;
    }
    __syncthreads();
    if (part == 0) {
        for (int p = 1; p < parts; ++p) {
            const float4 x = sums[p * vecs + v];
            o = make_float4(o.x + x.x, o.y + x.y, o.z + x.z, o.w + x.w);
        }
        const float r = ll != 0.0f ? 1.0f / ll : 0.0f;
        const int64_t at = rh * a.head_dim + 4 * v;
        store_elem(a.out, a.q_type, at, o.x * r);
        store_elem(a.out, a.q_type, at + 1, o.y * r);
        store_elem(a.out, a.q_type, at + 2, o.z * r);
        store_elem(a.out, a.q_type, at + 3, o.w * r);
    }
    if (a.lse && threadIdx.x == 0) a.lse[rh] = lse_of(mm, ll);
}

// Shared memory of the FMA kernel for G heads.
template <typename Shape>
size_t fma_smem(int G, int64_t head_dim) {
    return sizeof(float) * (Shape::kWarps + 1) * G * state_floats((int)head_dim) + (size_t)Shape::kRingBytes * Shape::kWarps;
}
// Whether an SM holds two CTAs of the ring with four heads (heads of more than 128
// elements; each CTA takes 1 KB of the 228 more).
bool two_rings(int cache_type, int64_t head_dim) {
    const size_t smem = cache_type == CBX_TYPE_F32 ? fma_smem<Fma<32, 2, true>>(4, head_dim) : fma_smem<Fma<32, 1, true>>(4, head_dim);
    return 2 * (smem + 1024) <= 228 * 1024;
}

// Query heads of a CTA.
int group_chunk(int group) { return group >= 3 ? 4 : group; }
bool use_mma(int cache_type, int group, int head_dim) {
    return head_dim <= 128 && group >= (cache_type == CBX_TYPE_F32 ? 3 : 2);
}

struct Splits {
    int n;
    bool cluster;
};
// CTAs over the keys of a row.  The host knows only the longest length the block
// table can hold, so the cost is that of rows of that length, in keys: waves of
// resident CTAs, each its whole steps and about 512 keys' time of start and end;
// joining in a cluster costs little, over the workspace a second launch.
// Measured in us (B200), splits 1 / 4 / 8 in a cluster, 16 / 32 / 48 over the
// workspace:
//   1 row, 1000 keys, 16 kv heads of 64, f32     9.7 / 5.5 / 5.2, 7.0 / 10.1 / 12.0
//   1 row, 65,537 keys, 8 kv heads of 128, bf16  711 / 187 / 97, 55 / 48 / 62
//   64 rows up to 2048, 16 kv heads of 64, f16   56 / 101 / 175
//   27 rows, 577 keys, 16 heads over 4 of 64, f32 q, bf16   splits 1 2 3 4: 11.3 9.6 9.4 14.0
//   5 rows, 7035 keys, 16 heads of 64, bf16                 splits 1 2 3 4: 49 36 29 39
// (A cluster of 16 took 65 us for the second.)
Splits choose_splits(int64_t n_rows, int64_t n_kv, int group, int64_t head_dim, int cache_type,
                     int64_t max_keys) {
    const bool mma = use_mma(cache_type, group, (int)head_dim);
    const int gc = mma ? kMmaHeads : group_chunk(group);
    const int64_t vecs = head_dim * type_size(cache_type) / 16;
    const bool f32 = cache_type == CBX_TYPE_F32;
    int64_t step, per_sm;  // CTAs per SM by registers and shared memory
    if (mma && f32) {
        step = head_dim <= 32 ? MmaF32<32>::kStep : head_dim <= 64 ? MmaF32<64>::kStep : MmaF32<128>::kStep;
        per_sm = head_dim <= 32 ? MmaF32<32>::kPerSM : head_dim <= 64 ? MmaF32<64>::kPerSM : MmaF32<128>::kPerSM;
    } else if (mma) {
        step = kMmaTile * kMmaWarps;
        per_sm = mma_per_sm((int)head_dim, cache_type == CBX_TYPE_F16);
    } else {
        const bool ring = group > 2 && two_rings(cache_type, head_dim);
        step = ring ? kRingStep : 8 * (vecs <= 8 ? 32 : vecs <= 16 ? 16 : 8);
        per_sm = group > 2 && !ring ? 1 : 2;  // four heads of 216 and more f32 elements: 253 registers
    }
    const int64_t resident = num_sms() * per_sm;
    const int64_t ctas = n_rows * n_kv * ((group + gc - 1) / gc);
    if (ctas >= 8 * resident) return {1, false};
    const int64_t steps = (max_keys + step - 1) / step;
    int64_t least = 0, best = 1;
    for (int64_t n = 1; n <= (max_keys >= 8192 ? kMaxSplits : kMaxCluster) && n <= steps; ++n) {
        // a cluster must fit into one GPC: not quite all places can be taken
        const int64_t places = n > 1 && n <= kMaxCluster ? resident * 97 / 100 : resident;
        const int64_t waves = (ctas * n + places - 1) / places;
        const int64_t cost = waves * ((steps + n - 1) / n * step + 512) +
                             (n == 1 ? 0 : n <= kMaxCluster ? 256 : 320 + 16 * n);
        if (n == 1 || cost < least) {
            least = cost;
            best = n;
        }
    }
    return {(int)best, best > 1 && best <= kMaxCluster};
}

cudaError_t launch_attend(void (*kern)(AttnArgs), int warps, size_t smem, const AttnArgs& a,
                          int64_t n_rows, cudaStream_t st) {
    const dim3 grid((unsigned)(n_rows * a.n_kv * a.chunks * a.splits));  // below 2^31: n_rows * n_heads is
    if (a.cluster) return launch_cluster(kern, grid, dim3(warps * 32), smem, (unsigned)a.splits, st, a);
    cudaError_t e = launch(kern, grid, dim3(warps * 32), smem, st, a);
    if (e == cudaSuccess && a.splits > 1)
        e = launch(k_attend_join, dim3((unsigned)(n_rows * a.n_heads)), dim3(kJoinThreads), 0, st, a);
    return e;
}

template <typename TC, int VL, int VPL, int G, bool RING>
cudaError_t run_fma_heads(AttnArgs a, int64_t n_rows, cudaStream_t st) {
    using Shape = Fma<VL, VPL, RING>;
    a.chunks = (a.group + G - 1) / G;
    const size_t smem = fma_smem<Shape>(G, a.head_dim);
    auto kern = k_attend_fma<TC, VL, VPL, G, RING>;
    if (smem > 48 * 1024 && !smem_opt_in(kern, smem)) return cudaErrorInvalidValue;
    return launch_attend(kern, Shape::kWarps, smem, a, n_rows, st);
}

// Heads of more than 128 elements, four at a time, take the ring where an SM holds
// two of its CTAs (f32: up to 208 elements), others the registers.  Ring / registers
// / registers with two at a time, in us (B200):
//   40 rows of 4000 keys, 32 heads over 4 of 160, f32      426 / 439 / 688
//   64 rows of 1000 keys, 16 heads over 4 of 200, f32      85 / 102
//   30 rows of 2511 keys, 8 heads over 2 of 160, f32       58 / 63
//   94 rows of 2511 keys, 16 heads over 2 of 256, bf16     242 / 323 / 429
//   30 rows of 2511 keys, 8 heads over 2 of 256, bf16      67 / 63
//   300 rows of 500 keys, 12 heads over 4 of 192, bf16     150 / 230
//   94 rows of 2511 keys, 16 heads over 2 of 256, f32      489 / 328
//   40 rows of 4000 keys, 32 heads over 4 of 256, f32      667 / 450
//   12 rows of 9000 keys, 8 heads over 1 of 224, f32       113 / 84
//   30 rows of 2511 keys, 8 heads over 2 of 256, f32       91 / 67 / 108
//   128 rows up to 8196 keys, 16 heads of 64, bf16         326 / 296 (1.98 GB: 6.7 TB/s)
template <typename TC, int VL, int VPL>
cudaError_t run_fma(const AttnArgs& a, int64_t n_rows, cudaStream_t st) {
    constexpr bool wide = VL * VPL * Vec<TC>::n > 128;  // heads that the tensor-core kernels do not take
    if constexpr (wide) {
        constexpr int type = sizeof(TC) == 4 ? CBX_TYPE_F32 : CBX_TYPE_F16;  // of this size
        if (a.group > 2 && two_rings(type, a.head_dim)) return run_fma_heads<TC, VL, VPL, 4, true>(a, n_rows, st);
        if constexpr (sizeof(TC) == 4)
            if (a.group > 2) return run_fma_heads<TC, VL, VPL, 4, false>(a, n_rows, st);
    }
    if constexpr (wide || sizeof(TC) == 4)
        if (a.group == 2) return run_fma_heads<TC, VL, VPL, 2, false>(a, n_rows, st);
    return run_fma_heads<TC, VL, VPL, 1, false>(a, n_rows, st);
}

template <typename T, int HD, int W>
cudaError_t run_mma(AttnArgs a, int64_t n_rows, bool same_type, cudaStream_t st) {
    constexpr bool bf16 = __is_same(T, __nv_bfloat16);
    a.chunks = (a.group + kMmaHeads - 1) / kMmaHeads;
    const size_t states = sizeof(float) * (kMmaWarps + 1) * kMmaHeads * state_floats(a.head_dim);
    const size_t rings = (size_t)kMmaWarps * mma_ring_bytes<HD>();
    const size_t smem = states > rings ? states : rings;
    void (*kern)(AttnArgs) = same_type ? k_attend_mma<T, HD, W, 1, 2> : k_attend_mma<T, HD, W, bf16 ? 3 : 2, bf16 ? 3 : 2>;
    if (smem > 48 * 1024 && !smem_opt_in(kern, smem)) return cudaErrorInvalidValue;
    return launch_attend(kern, kMmaWarps, smem, a, n_rows, st);
}

template <int HD, int W>
cudaError_t run_mma_f32(AttnArgs a, int64_t n_rows, cudaStream_t st) {
    a.chunks = (a.group + kMmaHeads - 1) / kMmaHeads;
    const size_t states = sizeof(float) * (kMmaWarps + 1) * kMmaHeads * state_floats(a.head_dim);
    const size_t rings = (size_t)kMmaWarps * MmaF32<HD>::kRingBytes;
    const size_t smem = states > rings ? states : rings;
    auto kern = k_attend_mma_f32<HD, W>;
    if (!smem_opt_in(kern, smem)) return cudaErrorInvalidValue;
    return launch_attend(kern, kMmaWarps, smem, a, n_rows, st);
}

template <typename TC>
cudaError_t run_head(const AttnArgs& a, int cache_type, int64_t n_rows, cudaStream_t st) {
    // Heads of up to 96 elements in rings made for 128: 100 rows of 2000 keys, 32
    // heads over 8 of 80, f32, 239 us (275 as 128); 3000 keys, f16, 143 (152).
    if constexpr (sizeof(TC) == 2) {
        const bool same = a.q_type == cache_type;
        if (use_mma(cache_type, a.group, a.head_dim))
            return a.head_dim <= 64   ? run_mma<TC, 64, 64>(a, n_rows, same, st)
                   : a.head_dim <= 96 ? run_mma<TC, 128, 96>(a, n_rows, same, st)
                                      : run_mma<TC, 128, 128>(a, n_rows, same, st);
    }
    if constexpr (sizeof(TC) == 4) {
        if (use_mma(cache_type, a.group, a.head_dim))
            return a.head_dim <= 32   ? run_mma_f32<32, 32>(a, n_rows, st)
                   : a.head_dim <= 64 ? run_mma_f32<64, 64>(a, n_rows, st)
                   : a.head_dim <= 96 ? run_mma_f32<128, 96>(a, n_rows, st)
                                      : run_mma_f32<128, 128>(a, n_rows, st);
    }
    const int vecs = (a.head_dim + Vec<TC>::n - 1) / Vec<TC>::n;
    if (vecs <= 4) return run_fma<TC, 4, 1>(a, n_rows, st);
    if (vecs <= 8) return run_fma<TC, 8, 1>(a, n_rows, st);
    if (vecs <= 16) return run_fma<TC, 16, 1>(a, n_rows, st);
    if constexpr (sizeof(TC) == 4)
        if (vecs > 32) return run_fma<TC, 32, 2>(a, n_rows, st);
    return run_fma<TC, 32, 1>(a, n_rows, st);
}

// Sizes that the workspace query and the call check alike.
int check_sizes(const char* name, int64_t n_rows, int64_t n_heads, int64_t n_kv_heads,
                int64_t head_dim, int64_t max_blocks, int64_t page_size, int cache_type) {
    constexpr int64_t kInt = 2147483647;
    if (n_rows < 0 || n_rows > kInt)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_rows %lld", name, (long long)n_rows);
    if (n_kv_heads <= 0 || n_heads <= 0 || n_heads > 65535 || n_heads % n_kv_heads)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_heads %lld is not a multiple of n_kv_heads %lld",
                    name, (long long)n_heads, (long long)n_kv_heads);
    if (n_rows > kInt / n_heads)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_rows * n_heads is 2^31 or more", name);
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

int64_t workspace_bytes_of(int64_t n_rows, int64_t n_heads, int64_t head_dim, Splits s) {
    if (s.n == 1 || s.cluster) return 0;
    return n_rows * n_heads * s.n * state_floats((int)head_dim) * (int64_t)sizeof(float);
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
    const Splits splits = choose_splits(n_rows, n_kv_heads, (int)(n_heads / n_kv_heads),
                                        head_dim, cache_type, max_blocks * page_size);
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
    const int qs = type_size(q_type);
    if (!aligned_to(q, qs) || !aligned_to(out, qs) || !aligned_to(table, 4) || !aligned_to(row_reqs, 4) ||
        !aligned_to(seq_lens, 4) || !aligned_to(lse, 4) || !aligned_to(err_word, 4))
        return fail(CBX_ERR_INVALID_ARG, "%s: an argument is not aligned to its type", name);
    if (meets_rows(out, n_rows * n_heads * head_dim * qs, q, n_rows, q_row_stride * qs, n_heads * head_dim * qs) ||
        meets_rows(lse, n_rows * n_heads * 4, q, n_rows, q_row_stride * qs, n_heads * head_dim * qs))
        return fail(CBX_ERR_INVALID_ARG, "%s: an output overlaps q", name);
    if (!aligned16(cache_k) || !aligned16(cache_v) ||
        (page_stride * type_size(cache_type)) % 16)
        return fail(CBX_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", name);
    const int group = (int)(n_heads / n_kv_heads);
    const Splits splits = choose_splits(n_rows, n_kv_heads, group, head_dim, cache_type,
                                        max_blocks * page_size);
    const int64_t need = workspace_bytes_of(n_rows, n_heads, head_dim, splits);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(CBX_ERR_INVALID_ARG, "%s: workspace of %lld bytes, %lld needed (16-byte aligned)",
                    name, (long long)(workspace ? workspace_bytes : 0), (long long)need);
    int shift = -1;
    if ((page_size & (page_size - 1)) == 0)
        for (shift = 0; (int64_t)1 << shift < page_size;) ++shift;
    AttnArgs a{q, q_type, q_row_stride, cache_k, cache_v, (int)n_pages, (int)page_size, shift,
               (int)(page_stride / kv_dim), kv_dim, table, (int)n_reqs, (int)max_blocks, row_reqs,
               seq_lens, (int)n_heads, (int)n_kv_heads, group, (int)head_dim, 1, scale * kLog2e, out,
               lse, static_cast<float*>(workspace), splits.n, splits.cluster, err_word};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    switch (cache_type) {
        case CBX_TYPE_F32: e = run_head<float>(a, cache_type, n_rows, st); break;
        case CBX_TYPE_BF16: e = run_head<__nv_bfloat16>(a, cache_type, n_rows, st); break;
        default: e = run_head<__half>(a, cache_type, n_rows, st);
    }
    return launch_status(e, name);
}
