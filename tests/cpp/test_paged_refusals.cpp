// The paged helpers of include/cbx_layer_helpers.hpp refuse tensors with gaps
// and 16-bit ones where they take dense int32 / f32 data: nullptr, and nothing is
// launched (the addresses below are made up).  Needs no GPU.  Built and run by
// tests/test_cpp_paged_refusals.py.
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "cbx_layer_helpers.hpp"

namespace {

int g_fail = 0;
uintptr_t g_next = 0x100000;

cbx::Tensor dense(int64_t ne0, int64_t ne1 = 1, int64_t ne2 = 1, int type = CBX_TYPE_F32) {
    return cbx::view(reinterpret_cast<void*>(g_next += 0x100000), type, ne0, ne1, ne2);
}
// The same tensor with every second element, or every second row.
cbx::Tensor gaps(cbx::Tensor t, int dim) {
    for (int i = dim; i < 4; ++i) t.nb[i] *= 2;
    return t;
}
// Each tensor in turn replaced by one with gaps, and by a 16-bit one.
template <typename F>
void each(const char* what, cbx::Tensor** ts, int n, F call) {
    for (int i = 0; i < n; ++i) {
        const cbx::Tensor good = *ts[i];
        cbx::Tensor bad[3] = {gaps(good, 0), gaps(good, 1), good};
        for (size_t& b : bad[2].nb) b /= 2;
        bad[2].type = CBX_TYPE_F16;
        for (int k = 0; k < 3; ++k) {
            *ts[i] = bad[k];
            // clears the last error; a launch, which fails without a GPU, would set it
            cbx_token_logprobs(nullptr, CBX_TYPE_F32, 0, 0, 8, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
            const bool ok = call() == nullptr && !std::strstr(cbx_last_error(), "launch");
            if (!ok) std::printf("FAIL %s: tensor %d, change %d\n", what, i, k);
            g_fail += !ok;
        }
        *ts[i] = good;
    }
}

}  // namespace

int main() {
    const int B = 3, MB = 4, P = 12, R = 5, S = 4, H = 4, Hk = 2, hd = 16, V = 40, K = 3;
    int32_t* err = reinterpret_cast<int32_t*>(0x80000);
    cbx::Tensor lens = dense(B), fresh = dense(B), slots = dense(R), pos = dense(R), reqs = dense(R), rl = dense(R);
    cbx::PagedState st{dense(MB, B), dense(B), dense(P), dense(1)};
    cbx::Tensor* plan[] = {&lens, &fresh, &st.block_table, &st.n_blocks, &st.free_list, &slots, &pos, &reqs, &rl};
    each("paged_plan", plan, 9, [&] { return cbx::paged_plan(lens, &fresh, st, S, slots, pos, &reqs, &rl, err); });

    cbx::Tensor qkv = dense((H + 2 * Hk) * hd, R), bias = dense((H + 2 * Hk) * hd), q = dense(H * hd, R);
    cbx::Tensor ck = dense(Hk * hd, S, P), cv = dense(Hk * hd, S, P);
    cbx::Tensor* append[] = {&slots, &bias, &q};
    each("qkv_kv_append_paged", append, 3,
         [&] { return cbx::qkv_kv_append_paged(qkv, &bias, ck, cv, slots, &q, err); });

    cbx::Tensor q3 = dense(hd, H, R), out = dense(hd, H, R), lse = dense(H, R);
    cbx::Tensor* attend[] = {&st.block_table, &reqs, &rl, &lse};
    each("paged_decode_attention", attend, 4, [&] {
        return cbx::paged_decode_attention(q3, ck, cv, st.block_table, &reqs, rl, 0.25f, out, &lse, nullptr, 0, err);
    });

    cbx::Tensor x = dense(V, R), tok = dense(R), lp = dense(R), en = dense(R), ids = dense(K, R), top = dense(K, R);
    cbx::Tensor* score[] = {&tok, &lp, &en, &ids, &top};
    each("token_logprobs", score, 5, [&] { return cbx::token_logprobs(x, &tok, &lp, &en, &ids, &top, err); });
    std::printf("%s: %d failure(s)\n", g_fail ? "FAILED" : "PASSED", g_fail);
    return g_fail ? 1 : 0;
}
