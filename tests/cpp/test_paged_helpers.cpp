// GPU test of the paged helpers of include/cbx_layer_helpers.hpp: a request's
// prompt and two decode steps against plain double loops.  Built and run by
// tests/test_cpp_paged_helpers.py; exits 0 when every check passes.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include "cbx_layer_helpers.hpp"

namespace {

int g_fail = 0;
void check(const char* what, bool ok) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", what);
    g_fail += !ok;
}

uint64_t g_rng = 0x9E3779B97F4A7C15ull;
float uniform() {
    g_rng = g_rng * 6364136223846793005ull + 1442695040888963407ull;
    return (float)((g_rng >> 40) + 0.5) / (float)(1ull << 24);
}
template <typename T>
T* to_dev(const std::vector<T>& h) {
    T* d = nullptr;
    cudaMalloc(&d, h.size() * sizeof(T) + 16);
    cudaMemcpy(d, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    return d;
}
template <typename T>
std::vector<T> to_host(const T* d, size_t n) {
    std::vector<T> h(n);
    cudaDeviceSynchronize();
    cudaMemcpy(h.data(), d, n * sizeof(T), cudaMemcpyDeviceToHost);
    return h;
}

}  // namespace

int main() {
    const int H = 4, Hk = 2, hd = 16, S = 4, P = 9, B = 2, MB = 5, QD = H * hd, KD = Hk * hd;
    const int W = QD + 2 * KD;
    std::vector<int32_t> ids(P);
    for (int i = 0; i < P; ++i) ids[i] = i;
    cbx::PagedState st;
    st.block_table = cbx::view(to_dev(std::vector<int32_t>(B * MB, -1)), CBX_TYPE_F32, MB, B);
    st.n_blocks = cbx::view(to_dev(std::vector<int32_t>(B, 0)), CBX_TYPE_F32, B);
    st.free_list = cbx::view(to_dev(ids), CBX_TYPE_F32, P);
    st.n_free = cbx::view(to_dev(std::vector<int32_t>{P}), CBX_TYPE_F32, 1);
    int32_t* err = to_dev(std::vector<int32_t>{0});
    // a pool of two layers; layer 1 is used
    float* pool = to_dev(std::vector<float>((size_t)P * 2 * 2 * S * KD, NAN));
    auto layer = [&](int kv) {
        cbx::Tensor t = cbx::view(pool + ((size_t)2 + kv) * S * KD, CBX_TYPE_F32, KD, S, P);
        t.nb[2] = (size_t)2 * 2 * S * KD * sizeof(float);
        return t;
    };
    cbx::Tensor ck = layer(0), cv = layer(1);
    std::vector<std::vector<std::vector<float>>> kept(B);  // per request: its rows of qkv
    const std::vector<std::vector<int32_t>> lens = {{6, 1}, {7, 2}, {8, 0}}, fed = {{6, 1}, {1, 1}, {1, 0}};
    for (size_t step = 0; step < lens.size(); ++step) {
        const int rows = 8;
        std::vector<float> qkv((size_t)rows * W), bias(W);
        for (auto& x : qkv) x = 2.0f * uniform() - 1.0f;
        for (auto& x : bias) x = 0.1f * uniform();
        std::vector<int> owner;
        for (int b = 0; b < B; ++b) {
            if (lens[step][b] == 0) kept[b].clear();
            for (int i = 0; i < fed[step][b]; ++i) {
                std::vector<float> row(W);
                for (int j = 0; j < W; ++j) row[j] = qkv[owner.size() * W + j] + bias[j];
                kept[b].push_back(row);
                owner.push_back(b);
            }
        }
        cbx::Tensor tl = cbx::view(to_dev(lens[step]), CBX_TYPE_F32, B), tn = cbx::view(to_dev(fed[step]), CBX_TYPE_F32, B);
        auto ints = [&] { return cbx::view(to_dev(std::vector<int32_t>(rows, 77)), CBX_TYPE_F32, rows); };
        cbx::Tensor slots = ints(), pos = ints(), reqs = ints(), rlen = ints();
        check("plan", cbx::paged_plan(tl, &tn, st, S, slots, pos, &reqs, &rlen, err) == &slots);
        cbx::Tensor tx = cbx::view(to_dev(qkv), CBX_TYPE_F32, W, rows), tb = cbx::view(to_dev(bias), CBX_TYPE_F32, W);
        cbx::Tensor tq = cbx::view(to_dev(std::vector<float>((size_t)rows * QD, 0.f)), CBX_TYPE_F32, QD, rows);
        check("append", cbx::qkv_kv_append_paged(tx, &tb, ck, cv, slots, &tq, err) == &tq);
        cbx::Tensor q3 = cbx::view(tq.data, CBX_TYPE_F32, hd, H, rows);
        cbx::Tensor out = cbx::view(to_dev(std::vector<float>((size_t)rows * QD, 5.f)), CBX_TYPE_F32, hd, H, rows);
        const int64_t wsb = cbx_paged_decode_attention_workspace(rows, H, Hk, hd, MB, S, CBX_TYPE_F32);
        void* ws = to_dev(std::vector<char>(wsb + 16));
        check("attend", cbx::paged_decode_attention(q3, ck, cv, st.block_table, &reqs, rlen, 0.25f, out, nullptr,
                                                    ws, wsb, err) == &out);
        auto got = to_host(static_cast<float*>(out.data), (size_t)rows * QD);
        auto rl = to_host(static_cast<int32_t*>(rlen.data), rows);
        double worst = 0.0;
        for (int r = 0; r < rows; ++r)
            for (int h = 0; h < H; ++h) {
                const int n = rl[r], b = r < (int)owner.size() ? owner[r] : 0, g = h / (H / Hk);
                std::vector<double> p(n);
                double m = -INFINITY, sum = 0.0;
                for (int j = 0; j < n; ++j) {
                    double s = 0.0;
                    for (int i = 0; i < hd; ++i) s += (double)kept[b][n - 1][h * hd + i] * kept[b][j][QD + g * hd + i];
                    p[j] = 0.25 * s;
                    m = std::fmax(m, p[j]);
                }
                for (auto& x : p) sum += x = std::exp(x - m);
                for (int i = 0; i < hd; ++i) {
                    double o = 0.0;
                    for (int j = 0; j < n; ++j) o += p[j] / sum * kept[b][j][QD + KD + g * hd + i];
                    worst = std::fmax(worst, std::fabs(o - got[((size_t)r * H + h) * hd + i]));
                }
            }
        // |values| <= 1.1, scores below 5: an f32 evaluation is off by less than 100 roundings of 2^-24
        check("attention values", worst < 100.0 / 16777216.0);
    }
    check("pages held", to_host(static_cast<int32_t*>(st.n_free.data), 1)[0] == P - 2);
    // log probabilities
    const int V = 301, N = 3, K = 4;
    std::vector<float> x((size_t)N * V);
    for (auto& v : x) v = 8.0f * uniform();
    std::vector<int32_t> tok = {0, 300, 17};
    cbx::Tensor lx = cbx::view(to_dev(x), CBX_TYPE_F32, V, N), lt = cbx::view(to_dev(tok), CBX_TYPE_F32, N);
    cbx::Tensor lp = cbx::view(to_dev(std::vector<float>(N)), CBX_TYPE_F32, N), en = cbx::view(to_dev(std::vector<float>(N)), CBX_TYPE_F32, N);
    cbx::Tensor ti = cbx::view(to_dev(std::vector<int32_t>(N * K)), CBX_TYPE_F32, K, N), tp = cbx::view(to_dev(std::vector<float>(N * K)), CBX_TYPE_F32, K, N);
    check("logprobs", cbx::token_logprobs(lx, &lt, &lp, &en, &ti, &tp, err) == &lp);
    auto glp = to_host(static_cast<float*>(lp.data), N);
    auto gid = to_host(static_cast<int32_t*>(ti.data), N * K);
    for (int r = 0; r < N; ++r) {
        double sum = 0.0;
        int best = 0;
        for (int j = 0; j < V; ++j) {
            sum += std::exp((double)x[r * V + j] - 8.0);
            if (x[r * V + j] > x[r * V + best]) best = j;
        }
        check("logprob", std::fabs(glp[r] - (x[r * V + tok[r]] - 8.0 - std::log(sum))) < 100.0 / 16777216.0 * 8.0);
        check("first alternative", gid[r * K] == best);
    }
    check("no error flags", to_host(err, 1)[0] == 0);
    // refusals: nullptr and no launch
    cbx::Tensor bad = cbx::view(lp.data, CBX_TYPE_F32, N + 1);
    check("refused sizes", cbx::token_logprobs(lx, &lt, &bad, nullptr, nullptr, nullptr, err) == nullptr &&
                               cbx::paged_plan(bad, nullptr, st, S, ti, tp, nullptr, nullptr, err) == nullptr);
    check("no CUDA error", cudaDeviceSynchronize() == cudaSuccess);
    std::printf("%s: %d failure(s)\n", g_fail ? "FAILED" : "PASSED", g_fail);
    return g_fail ? 1 : 0;
}
