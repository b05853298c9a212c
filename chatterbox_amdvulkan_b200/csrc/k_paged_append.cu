// k_paged_append.cu — the T3 attention prologue after the QKV GEMM
// (chatterbox-cpp/src/t3.cpp:465-489), with K and V written into the pages of
// a paged cache: per row, q = qkv[0, QD) + b, K[slot] = qkv[QD, QD + KD) + b,
// V[slot] = qkv[QD + KD, QD + 2 KD) + b, one f32 add and one rounding each.
//
// A copy with a scattered destination, bound by HBM: the GEMM's row is read
// once and its parts are written once.  A thread keeps one column group of 8
// elements (its bias stays in registers) and walks rows; rows narrower than the
// CTA lie side by side in it.  Measured (B200): 65,536 rows of 1024 + 2 x 1024
// f32 into bf16 pages 193 us (1.34 GB, 6.9 TB/s: above the copy rate, as part of
// what is written stays in L2); 54,170 rows of 256 + 2 x 64 f16 14.7 us (83 MB,
// 5.7 TB/s; 21.5 us with one row abreast); one row 1.5 us.
#include "cbx_common.cuh"

namespace cbx {
namespace {

constexpr int kThreads = 128;
constexpr int kCols = 8;  // elements of a column group

struct PagedAppendArgs {
    const void* qkv;
    int64_t qkv_stride;
    const float* bias;
    int64_t n_rows;
    int qd, kd;
    const int32_t* slots;
    void* ck;
    void* cv;
    int64_t page_stride;
    int page_size;
    int n_slots;
    bool dense;  // page_stride == page_size * kd: a slot is a row of the cache
    int cols;  // column groups of a CTA (vector kernel)
    void* q;
    int32_t* err;
};

__device__ __forceinline__ int64_t slot_offset(const PagedAppendArgs& a, int slot) {
    if (a.dense) return (int64_t)slot * a.kd;
    const int page = slot / a.page_size;
    return (int64_t)page * a.page_stride + (int64_t)(slot - page * a.page_size) * a.kd;
}

// Rows in flight per thread, waiting in registers as they are in memory: 4 of 16
// bits, 2 of f32.  52,428 rows of 1280 + 2 x 320 bf16, in us, 1 / 2 / 3 / 4 rows:
// 132 / 74 / 65 / 63; the f32 rows above 270 / 193 / 195 / 195.  Widened on
// arrival, 4 rows took 72 registers, and the bf16 ones 99 us.
template <typename TI>
constexpr int rows_in_flight() {
    return sizeof(TI) == 2 ? 4 : 2;
}

// qd, kd, row strides multiples of 8; all rows 16-byte aligned.
template <typename TI, typename TC>
__global__ void __launch_bounds__(kThreads) k_paged_append_vec(PagedAppendArgs a) {
    constexpr int kRows = rows_in_flight<TI>();
    constexpr int kVecs = kCols * sizeof(TI) / 16;
    grid_dep_wait();
    grid_dep_launch();
    const int side = threadIdx.x / a.cols;  // of the rows side by side
    const int abreast = kThreads / a.cols;
    const int g = blockIdx.x * a.cols + threadIdx.x % a.cols;
    if (side >= abreast || g >= (a.qd + 2 * a.kd) / kCols) return;
    const int col = g * kCols;
    const int part = col < a.qd ? 0 : col < a.qd + a.kd ? 1 : 2;
    const int in_part = part == 0 ? col : part == 1 ? col - a.qd : col - a.qd - a.kd;
    TC* cache = static_cast<TC*>(part == 1 ? a.ck : a.cv);
    float b[kCols] = {};
    if (a.bias) ldv<float, kCols>(a.bias + col, b);
    const TI* src = static_cast<const TI*>(a.qkv) + col;
    const int64_t stride = (int64_t)gridDim.y * abreast * kRows;
    for (int64_t r0 = ((int64_t)blockIdx.y * abreast + side) * kRows; r0 < a.n_rows; r0 += stride) {
        uint4 raw[kRows][kVecs];
        int slot[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            slot[i] = -1;
            if (r0 + i < a.n_rows) {
                slot[i] = __ldg(a.slots + r0 + i);
#pragma unroll
                for (int v = 0; v < kVecs; ++v)
                    raw[i][v] = __ldg(reinterpret_cast<const uint4*>(src + (r0 + i) * a.qkv_stride) + v);
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (slot[i] == -1) continue;
            float x[kCols];
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                constexpr int k = 4 / (int)sizeof(TI);
                unpack32(raw[i][v].x, x + (4 * v) * k, TI{});
                unpack32(raw[i][v].y, x + (4 * v + 1) * k, TI{});
                unpack32(raw[i][v].z, x + (4 * v + 2) * k, TI{});
                unpack32(raw[i][v].w, x + (4 * v + 3) * k, TI{});
            }
#pragma unroll
            for (int j = 0; j < kCols; ++j) x[j] = __fadd_rn(x[j], b[j]);
            const bool good = slot[i] >= 0 && slot[i] < a.n_slots;
            if (!good && col == 0) atomicOr(a.err, CBX_EFLAG_PAGE_OOB);
            if (part == 0) {
                if (a.q) stv<TI, kCols>(static_cast<TI*>(a.q) + (r0 + i) * a.qd + in_part, x);
            } else if (good) {
                stv<TC, kCols>(cache + slot_offset(a, slot[i]) + in_part, x);
            }
        }
    }
}

// Any dims and alignment: one element per thread.
template <typename TI, typename TC>
__global__ void __launch_bounds__(kThreads) k_paged_append_scalar(PagedAppendArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const int col = blockIdx.x * kThreads + threadIdx.x;
    if (col >= a.qd + 2 * a.kd) return;
    const int part = col < a.qd ? 0 : col < a.qd + a.kd ? 1 : 2;
    const int in_part = part == 0 ? col : part == 1 ? col - a.qd : col - a.qd - a.kd;
    TC* cache = static_cast<TC*>(part == 1 ? a.ck : a.cv);
    const float b = a.bias ? __ldg(a.bias + col) : 0.0f;
    const TI* src = static_cast<const TI*>(a.qkv) + col;
    for (int64_t r = blockIdx.y; r < a.n_rows; r += gridDim.y) {
        const int slot = __ldg(a.slots + r);
        if (slot == -1) continue;
        const float x = __fadd_rn(to_f(src[r * a.qkv_stride]), b);
        const bool good = slot >= 0 && slot < a.n_slots;
        if (!good && col == 0) atomicOr(a.err, CBX_EFLAG_PAGE_OOB);
        if (part == 0) {
            if (a.q) static_cast<TI*>(a.q)[r * a.qd + in_part] = from_f<TI>(x);
        } else if (good) {
            cache[slot_offset(a, slot) + in_part] = from_f<TC>(x);
        }
    }
}

template <typename TI, typename TC>
int run_append(PagedAppendArgs a, cudaStream_t st) {
    auto rows16 = [](const void* p, int64_t stride, size_t size) {
        return aligned16(p) && (stride * (int64_t)size) % 16 == 0;
    };
    const bool vec = a.qd % kCols == 0 && a.kd % kCols == 0 &&
                     rows16(a.qkv, a.qkv_stride, sizeof(TI)) && (!a.bias || aligned16(a.bias)) &&
                     (!a.q || aligned16(a.q)) && rows16(a.ck, a.page_stride, sizeof(TC)) &&
                     rows16(a.cv, a.page_stride, sizeof(TC));
    const int64_t units = vec ? (a.qd + 2LL * a.kd) / kCols : a.qd + 2LL * a.kd;
    a.cols = vec && units < kThreads ? (int)units : kThreads;
    const unsigned gx = (unsigned)((units + a.cols - 1) / a.cols);
    const int64_t per_cta = vec ? rows_in_flight<TI>() * (kThreads / a.cols) : 1;
    const int64_t want = (a.n_rows + per_cta - 1) / per_cta;
    const unsigned gy = (unsigned)(want < 65535 ? want : 65535);
    cudaError_t e = vec ? launch(k_paged_append_vec<TI, TC>, dim3(gx, gy), dim3(kThreads), 0, st, a)
                        : launch(k_paged_append_scalar<TI, TC>, dim3(gx, gy), dim3(kThreads), 0, st, a);
    return launch_status(e, "cbx_qkv_kv_append_paged");
}

template <typename TI>
int run_cache(const PagedAppendArgs& a, int cache_type, cudaStream_t st) {
    switch (cache_type) {
        case CBX_TYPE_F32: return run_append<TI, float>(a, st);
        case CBX_TYPE_BF16: return run_append<TI, __nv_bfloat16>(a, st);
        default: return run_append<TI, __half>(a, st);
    }
}

}  // namespace
}  // namespace cbx

extern "C" CBX_API int cbx_qkv_kv_append_paged(const void* qkv, int qkv_type,
                                               int64_t qkv_row_stride, const float* qkv_bias,
                                               int64_t n_rows, int64_t q_dim, int64_t kv_dim,
                                               const int32_t* slots, void* cache_k, void* cache_v,
                                               int cache_type, int64_t n_pages, int64_t page_size,
                                               int64_t page_stride, void* q_out,
                                               int32_t* err_word, cbx_stream_t stream) {
    using namespace cbx;
    const char* name = "cbx_qkv_kv_append_paged";
    constexpr int64_t kInt = 2147483647;
    if (n_rows < 0 || q_dim < 0 || kv_dim <= 0 || q_dim > (1 << 24) || kv_dim > (1 << 24))
        return fail(CBX_ERR_INVALID_ARG, "%s: n_rows %lld q_dim %lld kv_dim %lld", name,
                    (long long)n_rows, (long long)q_dim, (long long)kv_dim);
    if (qkv_row_stride == 0) qkv_row_stride = q_dim + 2 * kv_dim;
    if (qkv_row_stride < q_dim + 2 * kv_dim)
        return fail(CBX_ERR_INVALID_ARG, "%s: qkv_row_stride %lld < q_dim + 2 kv_dim", name,
                    (long long)qkv_row_stride);
    if (page_size <= 0 || page_size > kInt || n_pages <= 0 || n_pages > kInt / page_size)
        return fail(CBX_ERR_INVALID_ARG, "%s: page_size %lld n_pages %lld", name,
                    (long long)page_size, (long long)n_pages);
    if (page_stride == 0) page_stride = page_size * kv_dim;
    if (page_stride < page_size * kv_dim)
        return fail(CBX_ERR_INVALID_ARG, "%s: page_stride %lld < page_size * kv_dim: pages overlap",
                    name, (long long)page_stride);
    if (!valid_type(qkv_type) || !valid_type(cache_type))
        return fail(CBX_ERR_UNSUPPORTED_DTYPE, "%s: qkv_type %d cache_type %d", name, qkv_type,
                    cache_type);
    if (n_rows == 0) return ok();
    if (!qkv || !slots || !cache_k || !cache_v || !err_word)
        return fail(CBX_ERR_INVALID_ARG, "%s: NULL qkv, slots, cache or err_word", name);
    const int si = type_size(qkv_type), sc = type_size(cache_type);
    if (!aligned_to(qkv, si) || !aligned_to(q_out, si) || !aligned_to(cache_k, sc) || !aligned_to(cache_v, sc) ||
        !aligned_to(qkv_bias, 4) || !aligned_to(slots, 4) || !aligned_to(err_word, 4))
        return fail(CBX_ERR_INVALID_ARG, "%s: an argument is not aligned to its type", name);
    if (meets_rows(q_out, n_rows * q_dim * si, qkv, n_rows, qkv_row_stride * si, (q_dim + 2 * kv_dim) * si))
        return fail(CBX_ERR_INVALID_ARG, "%s: q_out overlaps qkv", name);
    PagedAppendArgs a{qkv, qkv_row_stride, qkv_bias, n_rows, (int)q_dim, (int)kv_dim, slots,
                      cache_k, cache_v, page_stride, (int)page_size, (int)(n_pages * page_size),
                      page_stride == page_size * kv_dim, 0, q_out, err_word};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (qkv_type) {
        case CBX_TYPE_F32: return run_cache<float>(a, cache_type, st);
        case CBX_TYPE_BF16: return run_cache<__nv_bfloat16>(a, cache_type, st);
        default: return run_cache<__half>(a, cache_type, st);
    }
}
