// C++ client of the flashrt_moe.hpp mirror's grouped products, 8-bit activations and gated activation.
//   test_train --host   refusals become std::runtime_error (no device work)
//   test_train --gpu    an expert layer's forward and backward pass, in values that every step holds exactly, against plain loops
// Prints "all passed" and exits 0 on success.
#include "flashrt_moe.hpp"

#include <cmath>
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
    check(throws([] { moe_product(nullptr, nullptr, 8, 1, nullptr, nullptr, nullptr, 1, 1, 8, 8, FRT_GGML_F32, nullptr, 8, FRT_GGML_F32); }),
          "moe_product of null throws");
    check(throws([] { moe_product_grad(nullptr, nullptr, 8, nullptr, nullptr, 2, 1, 8, 8, FRT_GGML_F32, nullptr, 8, FRT_GGML_F32); }),
          "moe_product_grad of two groups without bounds throws");
    check(throws([] {
              moe_product_wgrad(nullptr, nullptr, 8, nullptr, 8, nullptr, 1, nullptr, nullptr, 1, 1, 8, 8, FRT_GGML_Q8_0, nullptr, FRT_GGML_F32);
          }),
          "moe_product_wgrad of Q8_0 rows throws");
    check(throws([] { moe_swiglu(nullptr, nullptr, 8, FRT_GGML_F32, 1, 8, nullptr, nullptr, 8); }), "moe_swiglu of rows too close throws");
    check(throws([] { moe_swiglu_grad(nullptr, nullptr, 8, nullptr, 0, nullptr, nullptr, FRT_GGML_F32, 1, 8, nullptr, nullptr, 16); }),
          "moe_swiglu_grad of null throws");
    check(throws([] { mx8::quantize(nullptr, nullptr, 48, FRT_GGML_F32, 1, 48, nullptr, nullptr); }), "mx8::quantize of 48 columns throws");
    check(throws([] { mx8::dequantize(nullptr, nullptr, nullptr, 1, 32, nullptr, 32, FRT_GGML_F32); }), "mx8::dequantize of null throws");
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
    const int T = 5, K = 2, E = 3, n = 32, ff = 32, S = T * K;
    // x of small whole numbers with a 64 in it (its 8-bit scale is one); up weights small whole numbers, gate weights zero but for one far
    // positive row: the gate is 64 c there, its sigmoid one to fp32, and zero elsewhere, where h and the gradients vanish or halve exactly
    std::vector<float> x(T * n), w(E * 2 * ff * n, 0.0f), dh(S * ff);
    for (int t = 0; t < T; ++t)
        for (int c = 0; c < n; ++c) x[t * n + c] = c == 0 ? 64.0f : float((t + c) % 3);
    for (int e = 0; e < E; ++e)
        for (int f = 0; f < ff; ++f) {
            w[(size_t(e) * 2 * ff + f) * n] = f % 2 ? 1.0f : 0.0f;                    // gate: 64 or 0
            w[(size_t(e) * 2 * ff + ff + f) * n + 1 + (e + f) % (n - 1)] = float(1 + e);   // up
        }
    for (int i = 0; i < S * ff; ++i) dh[i] = float(i % 5 - 2);
    std::vector<int32_t> ids(S);
    for (int s = 0; s < S; ++s) ids[s] = s == 3 ? -1 : (s * 5) % E;
    Buffer<float> dx(x), dw(w), z(S * 2 * ff), h(S * ff), again(S * ff), ddh(dh), dz(S * 2 * ff), dxs(S * n), gw(w.size()), gw8(w.size());
    Buffer<int32_t> di(ids), bounds(E + 1), tok(S), slot(S), row(S);
    Buffer<int8_t> zc(S * 2 * ff), xc(T * n);
    Buffer<uint8_t> zs(S * ff / 16), xs(T * n / 32);
    hipStream_t st = nullptr;
    moe_sort(st, di.p, T, K, E, bounds.p, tok.p, slot.p, row.p);
    moe_product(st, dx.p, n, T, tok.p, dw.p, bounds.p, E, S, 2 * ff, n, FRT_GGML_F32, z.p, 2 * ff, FRT_GGML_F32);
    moe_swiglu(st, z.p, 2 * ff, FRT_GGML_F32, S, ff, bounds.p + E, h.p, ff, zc.p, zs.p);
    moe_swiglu_grad(st, ddh.p, ff, nullptr, 0, zc.p, zs.p, FRT_GGML_F32, S, ff, bounds.p + E, dz.p, 2 * ff, again.p, ff);
    moe_product_grad(st, dz.p, 2 * ff, dw.p, bounds.p, E, S, 2 * ff, n, FRT_GGML_F32, dxs.p, n, FRT_GGML_F32);
    moe_product_wgrad(st, dz.p, 2 * ff, dx.p, n, nullptr, T, tok.p, bounds.p, E, S, 2 * ff, n, FRT_GGML_F32, gw.p, FRT_GGML_F32);
    mx8::quantize(st, dx.p, n, FRT_GGML_F32, T, n, xc.p, xs.p);
    moe_product_wgrad(st, dz.p, 2 * ff, xc.p, n, xs.p, T, tok.p, bounds.p, E, S, 2 * ff, n, FRT_GGML_F32, gw8.p, FRT_GGML_F32);
    moe_product_wgrad(st, dz.p, 2 * ff, xc.p, n, xs.p, T, tok.p, bounds.p, E, S, 2 * ff, n, FRT_GGML_F32, gw8.p, FRT_GGML_F32, true);
    Buffer<float> back(T * n);
    mx8::dequantize(st, xc.p, xs.p, T, n, back.p, n, FRT_GGML_F32);
    detail::hip_check(hipDeviceSynchronize(), "sync");
    const std::vector<int32_t> b = bounds.host(), to = tok.host();
    const std::vector<float> hz = z.host(), hh = h.host(), ha = again.host(), hd = dz.host(), hx = dxs.host(), hw = gw.host(), hw8 = gw8.host();
    check(b[E] == S - 1 && back.host() == x, "moe_sort, and tokens kept in 8 bits");
    bool products = true, hidden = true, gates = true, rows = true, weights = true;
    std::vector<float> want_w(w.size(), 0.0f);
    for (int e = 0; e < E; ++e)
        for (int r = b[e]; r < b[e + 1]; ++r) {
            const float* xr = x.data() + size_t(to[r]) * n;
            std::vector<float> g(2 * ff, 0.0f), d(2 * ff);
            for (int f = 0; f < 2 * ff; ++f) {
                for (int c = 0; c < n; ++c) g[f] += w[(size_t(e) * 2 * ff + f) * n + c] * xr[c];
                products = products && hz[size_t(r) * 2 * ff + f] == g[f];
            }
            for (int f = 0; f < ff; ++f) {
                const float s = f % 2 ? 1.0f : 0.5f, u = g[ff + f], go = dh[size_t(r) * ff + f];
                hidden = hidden && hh[size_t(r) * ff + f] == g[f] * s * u && ha[size_t(r) * ff + f] == g[f] * s * u;
                d[f] = go * u * s;   // (1 + g (1 - s) is one in both)
                d[ff + f] = go * g[f] * s;
                gates = gates && hd[size_t(r) * 2 * ff + f] == d[f] && hd[size_t(r) * 2 * ff + ff + f] == d[ff + f];
            }
            for (int c = 0; c < n; ++c) {
                float sum = 0.0f;
                for (int f = 0; f < 2 * ff; ++f) {
                    sum += d[f] * w[(size_t(e) * 2 * ff + f) * n + c];
                    want_w[(size_t(e) * 2 * ff + f) * n + c] += d[f] * xr[c];
                }
                rows = rows && hx[size_t(r) * n + c] == sum;
            }
        }
    for (size_t i = 0; i < want_w.size(); ++i) weights = weights && hw[i] == want_w[i] && hw8[i] == 2 * want_w[i];
    check(products, "moe_product of picked rows");
    check(hidden, "moe_swiglu, and h again from 8 bits");
    check(gates, "moe_swiglu_grad from 8 bits");
    check(rows, "moe_product_grad");
    check(weights, "moe_product_wgrad, from 8 bits and added");
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
