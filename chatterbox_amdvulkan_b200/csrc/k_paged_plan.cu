// k_paged_plan.cu — block tables, slot maps and row positions of one step of
// paged T3 serving, built on the device from the requests' lengths.
//
// The free pages are a stack.  With need[b] = ceil(len[b] / page_size) and
// have[b] = n_blocks[b]:
//   released pages: entries [need, have) of each row, in the order of (b, j);
//     the i-th goes to free[n_free + i];
//   top = n_free + (number released);
//   missing pages: entries [have, need) of each row, in the order of (b, j);
//     the i-th is free[top - 1 - i];
//   row t of the step belongs to the request b with cu[b] <= t < cu[b + 1],
//     cu the exclusive sum of n_new, at position len[b] - n_new[b] + t - cu[b].
// Three exclusive sums over the requests give every index, so all entries and
// rows are written independently, and the result does not depend on timing.
//
// Latency and the copy of the state bound it.  Every CTA forms the same three
// sums in its shared memory, then all threads share the entries and rows.
//  - New outputs (no output is its own input): nothing that is read is written,
//    released pages included (the i-th is found by a search in the sums), so the
//    CTAs need no order and the grid covers the GPU.
//  - In place: one cluster of 8 CTAs (co-scheduled by the hardware, so its
//    barrier cannot wait for a CTA that is not running) pushes the released
//    pages, then the cluster barrier makes them visible and ends all reads of
//    what is overwritten.
// Measured: 512 requests of 513 blocks, 262,656 pages, one token each: 5.1 us
// with new outputs (20.3 us with the cluster), 8.2 us in place (1.0 of it the check
// of the pages that stay); 64 requests, 65,536 rows: 4.1 us (11.7) and 11.1 us; 64
// requests, one token each, in place: 4.8 us.  (Four rows to a thread, with 16-byte stores, was slower: 8.2 and 6.5
// us with new outputs.)
#include "cbx_common.cuh"

namespace cbx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

struct PlanArgs {
    const int32_t* seq_lens;
    const int32_t* n_new;
    int n_reqs, max_blocks, page_size, n_pages, max_rows;
    const int32_t* table_in;
    const int32_t* n_blocks_in;
    const int32_t* free_in;
    const int32_t* n_free_in;
    int32_t* table;
    int32_t* n_blocks;
    int32_t* free_list;
    int32_t* n_free;
    int32_t* slots;
    int32_t* positions;
    int32_t* row_reqs;
    int32_t* row_lens;
    int32_t* row_start;
    int32_t* err;
};

// Exclusive sums of three values per thread over the CTA, in place; totals in
// `tot`.  The row count is summed in 64 bits: clamped lengths of many requests
// can pass 2^31 (pages cannot: n_reqs * max_blocks is below 2^31).
struct Sums {
    int released, missing;
    long long rows;
};

__device__ __forceinline__ Sums block_exclusive(Sums v, Sums* warp_tot, Sums* tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    Sums s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s.released, o);
        const int b = __shfl_up_sync(0xffffffffu, s.missing, o);
        const long long c = __shfl_up_sync(0xffffffffu, s.rows, o);
        if (lane >= o) {
            s.released += a;
            s.missing += b;
            s.rows += c;
        }
    }
    if (lane == 31) warp_tot[w] = s;
    __syncthreads();
    if (w == 0) {
        Sums t = warp_tot[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, t.released, o);
            const int b = __shfl_up_sync(0xffffffffu, t.missing, o);
            const long long c = __shfl_up_sync(0xffffffffu, t.rows, o);
            if (lane >= o) {
                t.released += a;
                t.missing += b;
                t.rows += c;
            }
        }
        warp_tot[lane] = t;
    }
    __syncthreads();
    *tot = warp_tot[kPlanWarps - 1];
    Sums base = {0, 0, 0};
    if (w > 0) base = warp_tot[w - 1];
    return {base.released + s.released - v.released, base.missing + s.missing - v.missing,
            base.rows + s.rows - v.rows};
}

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

template <bool IN_PLACE>
__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(PlanArgs a) {
    extern __shared__ int smem[];
    __shared__ Sums warp_tot[kPlanWarps];
    const int B = a.n_reqs, S = a.page_size;
    int* s_need = smem;              // [B]
    int* s_have = s_need + B;        // [B]
    int* s_pop = s_have + B;         // [B] missing pages of the requests before
    int* s_push = s_pop + B;         // [B] released pages of the requests before
    int* s_first = s_push + B;       // [B] position of the request's first new token
    int* s_cu = s_first + B;         // [B + 1] first row
    const int tid = threadIdx.x;
    grid_dep_wait();
    grid_dep_launch();

    // The requests, `per` of them in a row for each thread.
    const int per = (B + kPlanThreads - 1) / kPlanThreads;
    const int b0 = tid * per < B ? tid * per : B, b1 = b0 + per < B ? b0 + per : B;
    int flags = 0;
    Sums mine = {0, 0, 0};
    const long long cap = (long long)a.max_blocks * S;
    for (int b = b0; b < b1; ++b) {
        int len = a.seq_lens[b];
        if (len < 0 || len > cap) {
            flags |= CBX_EFLAG_LENGTH;
            len = len < 0 ? 0 : (int)cap;  // cap < len <= INT_MAX here
        }
        int fresh = a.n_new ? a.n_new[b] : (len > 0 ? 1 : 0);
        if (fresh < 0 || fresh > len) {
            flags |= CBX_EFLAG_LENGTH;
            fresh = clamp_int(fresh, 0, len);
        }
        int have = a.n_blocks_in[b];
        if (have < 0 || have > a.max_blocks) {
            flags |= CBX_EFLAG_LENGTH;
            have = clamp_int(have, 0, a.max_blocks);
        }
        const int need = len / S + (len % S != 0);
        s_need[b] = need;
        s_have[b] = have;
        s_first[b] = len - fresh;
        s_cu[b] = fresh;
        mine.released += have > need ? have - need : 0;
        mine.missing += need > have ? need - have : 0;
        mine.rows += fresh;
    }
    int n_free = *a.n_free_in;
    if (n_free < 0 || n_free > a.n_pages) {
        flags |= CBX_EFLAG_LENGTH;
        n_free = clamp_int(n_free, 0, a.n_pages);
    }
    Sums tot;
    Sums at = block_exclusive(mine, warp_tot, &tot);
    for (int b = b0; b < b1; ++b) {
        const int need = s_need[b], have = s_have[b], fresh = s_cu[b];
        s_push[b] = at.released;
        s_pop[b] = at.missing;
        s_cu[b] = at.rows < a.max_rows ? (int)at.rows : a.max_rows;
        at.released += have > need ? have - need : 0;
        at.missing += need > have ? need - have : 0;
        at.rows += fresh;
    }
    const int n_rows = tot.rows < a.max_rows ? (int)tot.rows : a.max_rows;
    if (tid == 0) s_cu[B] = n_rows;
    if (tot.rows > a.max_rows) flags |= CBX_EFLAG_LENGTH;
    // A state whose counts are right never holds more pages than there are.
    int top = n_free;
    if (tot.released > a.n_pages - n_free) {
        flags |= CBX_EFLAG_LENGTH;
        top = a.n_pages;
    } else {
        top = n_free + tot.released;
    }
    if (tot.missing > top) flags |= CBX_EFLAG_NO_PAGE;
    __syncthreads();

    const int64_t me = (int64_t)blockIdx.x * kPlanThreads + tid, all = (int64_t)gridDim.x * kPlanThreads;
    // The last request whose exclusive sum is at most i.
    auto request_of = [&](const int* sums, int i) {
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sums[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    // The i-th released page, in table_in.
    auto released = [&](int i) {
        const int b = request_of(s_push, i);
        return a.table_in[(int64_t)b * a.max_blocks + s_need[b] + (i - s_push[b])];
    };
    if (IN_PLACE) {
        for (int64_t i = me; i < top - n_free; i += all) a.free_list[n_free + i] = released((int)i);
        if (a.free_list != a.free_in)
            for (int64_t i = me; i < a.n_pages; i += all)
                if (i < n_free || i >= top) a.free_list[i] = a.free_in[i];
        cluster_sync();
    } else {
        for (int64_t i = me; i < a.n_pages; i += all)
            a.free_list[i] = i < n_free || i >= top ? a.free_in[i] : released((int)i - n_free);
    }
    // Entry i of the stack after the pushes.
    auto on_stack = [&](int i) {
        if (IN_PLACE) return a.free_list[i];
        return i < n_free ? a.free_in[i] : released(i - n_free);
    };

    // Tables and counts.  In place the kept entries stay, but are checked like the
    // others; those behind the last page become -1 whatever they held.
    auto write_entry = [&](int b, int j, int need, int have) {
        const int64_t i = (int64_t)b * a.max_blocks + j;
        const int left = top - s_pop[b];  // pages on the stack when b's turn comes
        int page = -1;
        if (j < need && (j < have || j - have < left)) {
            page = j < have ? a.table_in[i] : on_stack(left - 1 - (j - have));
            if (page < 0 || page >= a.n_pages) flags |= CBX_EFLAG_PAGE_OOB;
        }
        a.table[i] = page;
    };
    if (IN_PLACE) {  // a warp takes a row: most of its entries are stores of -1
        const int lane = tid & 31, warps = (int)(all / 32);
        for (int b = (int)(me / 32); b < B; b += warps) {
            const int need = s_need[b], have = s_have[b];
            int first = 0;
            if (a.table == a.table_in) {  // (checked before the barrier: 10.1, not 8.2 us for the 512 requests)
                first = min(need, have);
                const int32_t* kept = a.table_in + (int64_t)b * a.max_blocks;
#pragma unroll 4
                for (int j = lane; j < first; j += 32)
                    if (kept[j] < 0 || kept[j] >= a.n_pages) flags |= CBX_EFLAG_PAGE_OOB;
            }
            for (int j = first + lane; j < a.max_blocks; j += 32) write_entry(b, j, need, have);
        }
    } else {
        const int64_t entries = (int64_t)B * a.max_blocks;
        for (int64_t i = me; i < entries; i += all) {
            const int b = (int)((uint32_t)i / (uint32_t)a.max_blocks);
            write_entry(b, (int)(i - (int64_t)b * a.max_blocks), s_need[b], s_have[b]);
        }
    }
    for (int64_t b = me; b < B; b += all) {
        const int need = s_need[b], have = s_have[b], left = top - s_pop[b];
        const int missing = need > have ? need - have : 0;
        const int got = missing < left ? missing : (left > 0 ? left : 0);
        a.n_blocks[b] = (need < have ? need : have) + got;
        if (a.row_start) a.row_start[b] = s_cu[b];
    }
    if (me == 0) {
        *a.n_free = tot.missing < top ? top - tot.missing : 0;
        if (a.row_start) a.row_start[B] = n_rows;
    }
    // Rows.
    for (int64_t t = me; t < a.max_rows; t += all) {
        int slot = -1, pos = 0, req = 0, len = 0;
        if (t < n_rows) {
            req = request_of(s_cu, (int)t);
            pos = s_first[req] + ((int)t - s_cu[req]);
            len = pos + 1;
            const int j = pos / S, have = s_have[req], left = top - s_pop[req];
            if (j < have || j - have < left) {
                const int page = j < have ? a.table_in[(int64_t)req * a.max_blocks + j]
                                          : on_stack(left - 1 - (j - have));
                if (page >= 0 && page < a.n_pages) slot = page * S + pos % S;
                else flags |= CBX_EFLAG_PAGE_OOB;
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
        if (a.row_reqs) a.row_reqs[t] = req;
        if (a.row_lens) a.row_lens[t] = len;
    }
    if (flags) atomicOr(a.err, flags);
}

// Two outputs overlap, or an output overlaps an input that is not its own.
bool overlaps(const void* p, int64_t np, const void* q, int64_t nq) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return p && q && np > 0 && nq > 0 && a < b + (uintptr_t)nq * 4 && b < a + (uintptr_t)np * 4;
}

}  // namespace
}  // namespace cbx

extern "C" CBX_API int cbx_paged_plan(const int32_t* seq_lens, const int32_t* n_new,
                                      int64_t n_reqs, int64_t max_blocks, int64_t page_size,
                                      int64_t n_pages, const int32_t* table_in,
                                      const int32_t* n_blocks_in, const int32_t* free_in,
                                      const int32_t* n_free_in, int32_t* table_out,
                                      int32_t* n_blocks_out, int32_t* free_out,
                                      int32_t* n_free_out, int64_t max_rows, int32_t* slots,
                                      int32_t* positions, int32_t* row_reqs, int32_t* row_lens,
                                      int32_t* row_start, int32_t* err_word,
                                      cbx_stream_t stream) {
    using namespace cbx;
    const char* name = "cbx_paged_plan";
    constexpr int64_t kInt = 2147483647;
    if (n_reqs < 0 || n_reqs > CBX_PAGED_MAX_REQS)
        return fail(CBX_ERR_INVALID_ARG, "%s: n_reqs %lld outside [0, %d]", name,
                    (long long)n_reqs, CBX_PAGED_MAX_REQS);
    if (max_blocks <= 0 || max_blocks > kInt || n_reqs * max_blocks > kInt)
        return fail(CBX_ERR_INVALID_ARG, "%s: max_blocks %lld (n_reqs %lld)", name,
                    (long long)max_blocks, (long long)n_reqs);
    if (page_size <= 0 || page_size > kInt || n_pages <= 0 || n_pages > kInt / page_size)
        return fail(CBX_ERR_INVALID_ARG, "%s: page_size %lld n_pages %lld", name,
                    (long long)page_size, (long long)n_pages);
    if (max_rows < 0 || max_rows > kInt)
        return fail(CBX_ERR_INVALID_ARG, "%s: max_rows %lld", name, (long long)max_rows);
    if (!free_in || !n_free_in || !free_out || !n_free_out || !err_word ||
        (n_reqs > 0 && (!seq_lens || !table_in || !n_blocks_in || !table_out || !n_blocks_out)) ||
        (max_rows > 0 && (!slots || !positions)))
        return fail(CBX_ERR_INVALID_ARG, "%s: NULL argument", name);
    {
        // Each state output may be its own input; no other overlap.
        const int64_t nt = n_reqs * max_blocks;
        bool aligned = aligned_to(err_word, 4);
        const void* in[6] = {table_in, n_blocks_in, free_in, n_free_in, seq_lens, n_new};
        const int64_t ni[6] = {nt, n_reqs, n_pages, 1, n_reqs, n_reqs};
        const void* out[9] = {table_out, n_blocks_out, free_out, n_free_out, slots,
                              positions, row_reqs, row_lens, row_start};
        const int64_t no[9] = {nt, n_reqs, n_pages, 1, max_rows,
                               max_rows, max_rows, max_rows, n_reqs + 1};
        for (int i = 0; i < 9; ++i) aligned = aligned && aligned_to(out[i], 4) && aligned_to(in[i < 6 ? i : 0], 4);
        if (!aligned) return fail(CBX_ERR_INVALID_ARG, "%s: an argument is not aligned to its type", name);
        for (int i = 0; i < 9; ++i) {
            for (int j = 0; j < 6; ++j)
                if (!(i == j && i < 4 && out[i] == in[j]) && overlaps(out[i], no[i], in[j], ni[j]))
                    return fail(CBX_ERR_INVALID_ARG, "%s: an output overlaps an input", name);
            for (int j = 0; j < i; ++j)
                if (overlaps(out[i], no[i], out[j], no[j]))
                    return fail(CBX_ERR_INVALID_ARG, "%s: two outputs overlap", name);
        }
    }
    PlanArgs a{seq_lens, n_new, (int)n_reqs, (int)max_blocks, (int)page_size, (int)n_pages,
               (int)max_rows, table_in, n_blocks_in, free_in, n_free_in, table_out, n_blocks_out,
               free_out, n_free_out, slots, positions, row_reqs, row_lens, row_start, err_word};
    const size_t smem = sizeof(int) * (6 * (size_t)n_reqs + 1);
    const bool in_place = table_out == table_in || n_blocks_out == n_blocks_in ||
                          free_out == free_in || n_free_out == n_free_in;
    auto kern = in_place ? k_paged_plan<true> : k_paged_plan<false>;
    if (smem > 40 * 1024 && !smem_opt_in(kern, smem))
        return fail(CBX_ERR_CUDA, "%s: shared memory opt-in of %zu bytes refused", name, smem);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (in_place) {
        e = launch_cluster(kern, dim3(8), dim3(kPlanThreads), smem, 8, st, a);
    } else {
        int64_t work = n_reqs * max_blocks;
        if (work < n_pages) work = n_pages;
        if (work < max_rows) work = max_rows;
        int64_t ctas = (work + kPlanThreads - 1) / kPlanThreads;
        if (ctas > num_sms()) ctas = num_sms();
        e = launch(kern, dim3((unsigned)ctas), dim3(kPlanThreads), smem, st, a);
    }
    return launch_status(e, name);
}
