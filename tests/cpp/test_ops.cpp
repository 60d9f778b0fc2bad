// C++ client of the flashrt_moe.hpp mirror's row moves and 4-bit products.
//   test_ops --host   refusals become std::runtime_error (no device work)
//   test_ops --gpu    tokens sorted by expert, quantized, multiplied by 4-bit weights of powers of two and summed back, in values
//                     that every step holds exactly, against plain loops
// Prints "all passed" and exits 0 on success.
#include "flashrt_moe.hpp"

#include <cstdio>
#include <cstring>
#include <vector>

namespace {

int g_fail = 0;
void check(bool ok, const char* what) {
    std::printf("%-60s %s\n", what, ok ? "ok" : "FAILED");
    if (!ok) ++g_fail;
}

template <typename F>
bool throws(F&& f) {
    try {
        f();
    } catch (const std::runtime_error&) {
        return true;
    }
    return false;
}

void host_checks() {
    using namespace flashrt;
    check(throws([] { moe_sort(nullptr, nullptr, 1, 1, 4, nullptr, nullptr, nullptr, nullptr); }), "moe_sort without ids throws");
    check(throws([] { moe_permute(nullptr, nullptr, 8, FRT_GGML_Q8_0, 1, 1, 8, nullptr, nullptr, 8); }), "moe_permute of Q8_0 rows throws");
    check(throws([] { moe_permute_grad(nullptr, nullptr, 8, FRT_GGML_F32, 1, 1, 8, nullptr, nullptr, 8); }), "moe_permute_grad of null throws");
    check(throws([] { moe_unpermute(nullptr, nullptr, 8, FRT_GGML_F32, 1, 0, 8, nullptr, nullptr, nullptr, 8); }), "moe_unpermute of no slots throws");
    check(throws([] {
              moe_unpermute_grad(nullptr, nullptr, 8, nullptr, 8, FRT_GGML_F32, 1, 1, 8, nullptr, nullptr, nullptr, 8, nullptr);
          }),
          "moe_unpermute_grad of null throws");
    check(throws([] { mx4::quantize(nullptr, nullptr, 48, FRT_GGML_F32, 1, 48, nullptr, nullptr); }), "mx4::quantize of 48 columns throws");
    check(throws([] { mx4::dequantize(nullptr, nullptr, nullptr, 1, 32, nullptr, 32, FRT_GGML_F32); }), "mx4::dequantize of null throws");
    check(throws([] {
              mx4::product(nullptr, nullptr, nullptr, 1, nullptr, nullptr, nullptr, nullptr, 2, 1, 8, 32, nullptr, 8, FRT_GGML_F32);
          }),
          "mx4::product of two groups without bounds throws");
}

template <typename T>
struct Buffer {   // device memory
    T* p = nullptr;
    size_t n;
    explicit Buffer(size_t count) : n(count) { flashrt::detail::hip_check(hipMalloc(reinterpret_cast<void**>(&p), n * sizeof(T)), "hipMalloc"); }
    explicit Buffer(const std::vector<T>& v) : Buffer(v.size()) {
        flashrt::detail::hip_check(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice), "hipMemcpy");
    }
    ~Buffer() { (void)hipFree(p); }
    std::vector<T> host() const {
        std::vector<T> v(n);
        flashrt::detail::hip_check(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost), "hipMemcpy");
        return v;
    }
};

void gpu_checks() {
    using namespace flashrt;
    const int T = 6, K = 2, E = 3, C = 64, N = 32, S = T * K;
    // x[t][c] in {1, 2, 4}: codes of scale 1 exactly; expert e's feature j picks value 2 j of the row, times 2^(e - 1)
    std::vector<float> x(T * C), wts(S);
    for (int i = 0; i < T * C; ++i) x[i] = float(1 << ((i / C + i) % 3));
    for (int t = 0; t < T; ++t) x[t * C] = x[t * C + 32] = 4.0f;   // (every block's largest)
    std::vector<int32_t> ids(S);
    for (int s = 0; s < S; ++s) {
        ids[s] = s == 5 ? -1 : (s * 7) % E;
        wts[s] = 0.25f * float(1 + s % 4);
    }
    std::vector<uint8_t> wq(E * N * C / 2, 0), ws(E * N * C / 32, 127);
    for (int e = 0; e < E; ++e)
        for (int j = 0; j < N; ++j) {
            wq[(size_t(e) * N + j) * (C / 2) + j] = 2;   // value 2 j: code 2, 1.0
            for (int b = 0; b < C / 32; ++b) ws[(size_t(e) * N + j) * (C / 32) + b] = uint8_t(126 + e);
        }
    Buffer<float> dx(x), dw(wts), xs(S * C), out(S * N), y(T * N), back(S * C), dys(S * N), dwts(S), dtok(T * C);
    Buffer<int32_t> di(ids), bounds(E + 1), tok(S), slot(S), row(S);
    Buffer<uint8_t> q(S * C / 2), sc(S * C / 32), dwq(wq), dws(ws);
    hipStream_t st = nullptr;
    moe_sort(st, di.p, T, K, E, bounds.p, tok.p, slot.p, row.p);
    moe_permute(st, dx.p, C, FRT_GGML_F32, T, K, C, row.p, xs.p, C);
    detail::hip_check(hipDeviceSynchronize(), "sync");
    const std::vector<int32_t> b = bounds.host(), r = row.host();
    check(b[0] == 0 && b[E] == S - 1 && r[5] == -1, "moe_sort: bounds and the dropped slot");
    mx4::quantize(st, xs.p, C, FRT_GGML_F32, b[E], C, q.p, sc.p);
    mx4::dequantize(st, q.p, sc.p, b[E], C, back.p, C, FRT_GGML_F32);
    mx4::product(st, q.p, sc.p, b[E], nullptr, dwq.p, dws.p, bounds.p, E, b[E], N, C, out.p, N, FRT_GGML_F32);
    moe_unpermute(st, out.p, N, FRT_GGML_F32, T, K, N, row.p, dw.p, y.p, N);
    moe_unpermute_grad(st, y.p, N, out.p, N, FRT_GGML_F32, T, K, N, row.p, dw.p, dys.p, N, dwts.p);
    moe_permute_grad(st, xs.p, C, FRT_GGML_F32, T, K, C, row.p, dtok.p, C);
    detail::hip_check(hipDeviceSynchronize(), "sync");
    const std::vector<float> hy = y.host(), hb = back.host(), hd = dwts.host(), ht = dtok.host(), hg = dys.host();
    bool values = true, sums = true, grads = true, tokens = true;
    for (int t = 0; t < T; ++t) {
        int slots = 0;
        for (int k = 0; k < K; ++k) slots += ids[t * K + k] >= 0;
        for (int c = 0; c < C; ++c) tokens = tokens && ht[t * C + c] == float(slots) * x[t * C + c];
        float dot[K] = {};
        for (int j = 0; j < N; ++j) {
            float want = 0.0f;
            for (int k = 0; k < K; ++k)
                if (ids[t * K + k] >= 0) want += wts[t * K + k] * x[t * C + 2 * j] * 0.5f * float(1 << ids[t * K + k]);
            sums = sums && hy[t * N + j] == want;
            for (int k = 0; k < K; ++k)
                if (ids[t * K + k] >= 0) {
                    dot[k] += want * x[t * C + 2 * j] * 0.5f * float(1 << ids[t * K + k]);
                    grads = grads && hg[size_t(r[t * K + k]) * N + j] == wts[t * K + k] * want;
                }
        }
        for (int k = 0; k < K; ++k) {
            grads = grads && hd[t * K + k] == dot[k];
            if (r[t * K + k] >= 0)
                for (int c = 0; c < C; ++c) values = values && hb[size_t(r[t * K + k]) * C + c] == x[t * C + c];
        }
    }
    check(values, "mx4::quantize and dequantize of the sorted rows");
    check(sums, "mx4::product and moe_unpermute");
    check(grads, "moe_unpermute_grad");
    check(tokens, "moe_permute_grad");
}

}  // namespace

int main(int argc, char** argv) {
    host_checks();
    if (argc > 1 && std::strcmp(argv[1], "--gpu") == 0) gpu_checks();
    if (g_fail) {
        std::printf("%d FAILED\n", g_fail);
        return 1;
    }
    std::printf("all passed\n");
    return 0;
}
