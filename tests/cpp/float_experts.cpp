// Experts in block-scaled 8-bit floating point and in f16 from C++, through the C++ face over the C ABI (sfnx/kernels.hpp):
// quantize_f8, f8_gemm, the grouped gate|up + SwiGLU and down, and the grouped 16-bit products, over a window's jobs and a prompt
// chunk's BigJobs; each against its formula on the host in 64 bits, and with the experts behind a table of pointers (DW::ep) bit
// for bit as with a stride.  Bounds as in tests/f8_util.py.  Prints "ok" when every check holds; exit status 1 otherwise.  Built
// by the package's build step; run by tests/test_gpu_cpp_float.py.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <type_traits>
#include <vector>

#include "sfnx/kernels.hpp"

using namespace sfnx;

namespace {

constexpr double ULP = 0x1p-23;
constexpr int H = 272, FF = 144, E = 5, K = 3;
constexpr int nb(int n) { return (n + 127) / 128; }

void hk(hipError_t e, const char* what) {
    if (e != hipSuccess) throw std::runtime_error(std::string(what) + ": " + hipGetErrorString(e));
}
template <typename T> T* dev(size_t n) {
    void* p = nullptr;
    hk(hipMalloc(&p, n * sizeof(T) + 256), "hipMalloc");
    hk(hipMemset(p, 0, n * sizeof(T) + 256), "hipMemset");
    return (T*) p;
}
template <typename T> T* up(const std::vector<T>& v) {
    T* p = dev<T>(v.size());
    hk(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice), "copy");
    return p;
}
template <typename T> std::vector<T> host(const T* d, size_t n) {
    std::vector<T> h(n);
    hk(hipMemcpy(h.data(), d, n * sizeof(T), hipMemcpyDeviceToHost), "copy");
    return h;
}
std::vector<float> normal(size_t n, uint64_t seed, float std) {
    float* d = dev<float>(n);
    ck(sfnx_synth_normal(d, n, seed, 0, std, nullptr));
    return host(d, n);
}
double e4m3(uint8_t c) {
    const int e = c >> 3 & 15, m = c & 7;
    const double v = e ? std::ldexp(8 + m, e - 10) : std::ldexp(m, -9);
    return c & 128 ? -v : v;
}

int failed = 0;
void check(const char* what, size_t bad, size_t n) {
    std::printf("%s: %zu of %zu values off\n", what, bad, n);
    failed += bad != 0 || n == 0;
}
template <typename T> void same(const char* what, const std::vector<T>& a, const std::vector<T>& b) {
    size_t bad = 0;
    for (size_t i = 0; i < a.size(); ++i) bad += std::memcmp(&a[i], &b[i], sizeof(T)) != 0;
    check(what, bad, a.size());
}

// values in 64 bits, row-major
struct Mat {
    int rows, cols;
    std::vector<double> v;
    const double* row(int r) const { return v.data() + (size_t) r * cols; }
};
Mat rows8(const std::vector<uint8_t>& q, const std::vector<float>& s, int rows, int cols) {
    Mat m{rows, cols, std::vector<double>((size_t) rows * cols)};
    for (int r = 0; r < rows; ++r)
        for (int c = 0; c < cols; ++c) m.v[(size_t) r * cols + c] = e4m3(q[(size_t) r * cols + c]) * s[(size_t) r * nb(cols) + c / 128];
    return m;
}
struct Dot {
    double v, err;
};
// a product summed in fp32: its value, and its bound of `terms` roundings
Dot dot(const double* a, const double* b, int n, int terms) {
    double v = 0, size = 0;
    for (int i = 0; i < n; ++i) v += a[i] * b[i], size += std::fabs(a[i] * b[i]);
    return {v, terms * ULP * size};
}
Dot swiglu(const Dot& g, const Dot& u) {
    const double s = g.v / (1 + std::exp(-g.v));
    return {s * u.v, 1.1 * g.err * (std::fabs(u.v) + u.err) + (std::fabs(s) + 1.1 * g.err) * u.err + 8 * ULP * std::fabs(s * u.v)};
}

// n matrices of the 8-bit store: codes of normal values, a scale for each block
struct Store {
    DW dw;
    size_t stride;
    std::vector<Mat> m;
};
// the same experts behind a table of pointers
Store tabled(Store s, int n) {
    std::vector<const char*> t(n);
    for (int e = 0; e < n; ++e) t[e] = (const char*) s.dw.p + e * s.stride;
    s.dw.ep = up(t);
    s.dw.p = nullptr;
    return s;
}
Store store8(int n, int rows, int cols, uint64_t seed) {
    Store st;
    st.stride = sfnx_f8_matrix_bytes(rows, cols);
    const size_t vals = (size_t) rows * cols;
    const std::vector<float> w = normal((size_t) n * vals, seed, 1.f);
    uint8_t* q = dev<uint8_t>(n * vals);
    float* s = dev<float>((size_t) n * rows * nb(cols));
    quantize_f8(SFNX_F32, up(w), cols, n * rows, cols, q, s, nullptr);
    const std::vector<uint8_t> hq = host(q, n * vals);
    std::vector<uint8_t> blob(n * st.stride);
    for (int e = 0; e < n; ++e) {
        std::memcpy(&blob[e * st.stride], &hq[e * vals], vals);
        std::vector<float> bs(nb(rows) * nb(cols));
        for (size_t b = 0; b < bs.size(); ++b) bs[b] = 1e-4f * (1 + (float) ((b + e) % 3));
        std::memcpy(&blob[e * st.stride + vals], bs.data(), 4 * bs.size());
        Mat m{rows, cols, std::vector<double>(vals)};
        for (int r = 0; r < rows; ++r)
            for (int c = 0; c < cols; ++c) m.v[(size_t) r * cols + c] = e4m3(hq[e * vals + (size_t) r * cols + c]) * bs[r / 128 * nb(cols) + c / 128];
        st.m.push_back(std::move(m));
    }
    st.dw = DW{up(blob), 0, cols, rows};
    return st;
}
Store store16(int n, int rows, int cols, uint64_t seed) {
    Store st;
    const size_t vals = (size_t) rows * cols;
    st.stride = 2 * vals;
    const std::vector<float> w = normal(n * vals, seed, 0.05f);
    uint16_t* d = dev<uint16_t>(n * vals);
    ck(sfnx_to_f16(up(w), d, n * vals, nullptr));
    const std::vector<uint16_t> bits = host(d, n * vals);
    for (int e = 0; e < n; ++e) {
        Mat m{rows, cols, std::vector<double>(vals)};
        for (size_t i = 0; i < vals; ++i) {
            _Float16 h;
            std::memcpy(&h, &bits[e * vals + i], 2);
            m.v[i] = (double) h;
        }
        st.m.push_back(std::move(m));
    }
    st.dw = DW{d, SFNX_F16, cols, rows};
    return st;
}

// a job's rows: pair p = t K + k reads row t (gather) or p and writes row p
template <typename J> std::vector<J> jobs_of(int T, bool gather) {
    constexpr int SIZE = std::is_same<J, Job>::value ? MAXT : PF_JOB;
    std::vector<J> js;
    for (int e = 0; e < E; ++e)
        for (int t = 0; t < T; ++t)
            for (int k = 0; k < K; ++k) {
                if ((t * t + 2 * k) % E != e) continue;   // distinct experts a token: 2 k mod 5
                if (js.empty() || js.back().w != e || js.back().n == SIZE) js.push_back(J{}), js.back().w = e;
                J& j = js.back();
                j.y[j.n] = gather ? t : t * K + k;
                j.out[j.n++] = t * K + k;
            }
    return js;
}

template <typename J> void layer(int T, const Store& gu, const Store& dn, const Store& gu_t, const Store& dn_t) {
    constexpr bool BIG = std::is_same<J, BigJob>::value;
    const std::string tag = BIG ? "prompt: " : "window: ";
    const int P = T * K;
    const std::vector<J> jg = jobs_of<J>(T, true), jd = jobs_of<J>(T, false);
    const J *djg = up(jg), *djd = up(jd);
    const int n = (int) jg.size(), *dn_jobs = up(std::vector<int>{n, 0});
    const std::vector<float> x = normal((size_t) T * H, 7, 1.f);
    uint8_t* xq = dev<uint8_t>((size_t) T * H);
    float* xs = dev<float>((size_t) T * nb(H));
    quantize_f8(SFNX_F32, up(x), H, T, H, xq, xs, nullptr);
    const std::vector<uint8_t> hxq = host(xq, (size_t) T * H);
    const std::vector<float> hxs = host(xs, (size_t) T * nb(H));
    const Mat X = rows8(hxq, hxs, T, H);
    size_t bad = 0;
    for (int t = 0; t < T; ++t)
        for (int c = 0; c < H; ++c)
            bad += !(std::fabs(X.row(t)[c] - x[(size_t) t * H + c]) <= (0x1p-4 + 2 * ULP) * std::fabs(x[(size_t) t * H + c]) + 0x1p-10 * hxs[(size_t) t * nb(H) + c / 128]);
    check((tag + "quantize_f8").c_str(), bad, (size_t) T * H);

    // gate|up; a window's h is f32 and quantized by its down, a prompt's is 8-bit
    float *h = dev<float>((size_t) P * FF), *h2 = dev<float>((size_t) P * FF), *hs = dev<float>((size_t) P * nb(FF)), *hs2 = dev<float>((size_t) P * nb(FF));
    uint8_t *hq = dev<uint8_t>((size_t) P * FF), *hq2 = dev<uint8_t>((size_t) P * FF);
    float *part = dev<float>((size_t) P * H), *part2 = dev<float>((size_t) P * H);
    if constexpr (BIG) {
        moe_gate_up_swiglu_f8_big(gu.dw, gu.stride, djg, dn_jobs, n, xq, xs, hq, hs, nullptr);
        moe_gate_up_swiglu_f8_big(gu_t.dw, gu.stride, djg, dn_jobs, n, xq, xs, hq2, hs2, nullptr);
        moe_down_f8_big(dn.dw, dn.stride, djd, dn_jobs, n, hq, hs, SFNX_F32, part, nullptr);
        moe_down_f8_big(dn_t.dw, dn.stride, djd, dn_jobs, n, hq, hs, SFNX_F32, part2, nullptr);
        same((tag + "gate|up behind a table").c_str(), host(hq, (size_t) P * FF), host(hq2, (size_t) P * FF));
        same((tag + "gate|up's scales behind a table").c_str(), host(hs, (size_t) P * nb(FF)), host(hs2, (size_t) P * nb(FF)));
    } else {
        moe_gate_up_swiglu_f8(gu.dw, gu.stride, djg, dn_jobs, n, xq, xs, h, nullptr);
        moe_gate_up_swiglu_f8(gu_t.dw, gu.stride, djg, dn_jobs, n, xq, xs, h2, nullptr);
        moe_down_f8(dn.dw, dn.stride, djd, dn_jobs, n, h, SFNX_F32, part, nullptr);
        moe_down_f8(dn_t.dw, dn.stride, djd, dn_jobs, n, h, SFNX_F32, part2, nullptr);
        same((tag + "gate|up behind a table").c_str(), host(h, (size_t) P * FF), host(h2, (size_t) P * FF));
        quantize_f8(SFNX_F32, h, FF, P, FF, hq, hs, nullptr);   // as the call does itself
    }
    same((tag + "down behind a table").c_str(), host(part, (size_t) P * H), host(part2, (size_t) P * H));
    const std::vector<float> hh = host(h, (size_t) P * FF), hhs = host(hs, (size_t) P * nb(FF)), hp = host(part, (size_t) P * H);
    const Mat Hq = rows8(host(hq, (size_t) P * FF), hhs, P, FF);
    size_t bad_h = 0, bad_p = 0, rows = 0;
    for (size_t i = 0; i < jg.size(); ++i)
        for (int m = 0; m < jg[i].n; ++m, ++rows) {
            const int o = jg[i].out[m];
            const Mat &G = gu.m[jg[i].w], &D = dn.m[jd[i].w];
            const double* xr = X.row(jg[i].y[m]);
            for (int f = 0; f < FF; ++f) {
                const Dot w = swiglu(dot(xr, G.row(f), H, 131 + nb(H)), dot(xr, G.row(FF + f), H, 131 + nb(H)));
                const double got = BIG ? Hq.row(o)[f] : hh[(size_t) o * FF + f];
                const double lim = w.err + (BIG ? (0x1p-4 + 2 * ULP) * (std::fabs(w.v) + w.err) + 0x1p-10 * hhs[(size_t) o * nb(FF) + f / 128] : 0);
                bad_h += !(std::fabs(got - w.v) <= lim);
            }
            for (int r = 0; r < H; ++r) {
                const Dot w = dot(Hq.row(jd[i].y[m]), D.row(r), FF, 131 + nb(FF));
                bad_p += !(std::fabs(hp[(size_t) jd[i].out[m] * H + r] - w.v) <= w.err);
            }
        }
    check((tag + "gate|up").c_str(), bad_h, rows * FF);
    check((tag + "down").c_str(), bad_p, rows * H);
}

template <typename J> void mm16(int T, const Store& w, const Store& w_t) {
    constexpr bool BIG = std::is_same<J, BigJob>::value;
    const std::string tag = BIG ? "prompt: " : "window: ";
    const std::vector<J> js = jobs_of<J>(T, true);
    const J* djs = up(js);
    const int n = (int) js.size(), *nj = up(std::vector<int>{n, 0}), P = T * K, N = w.dw.n_out;
    uint16_t* x = dev<uint16_t>((size_t) T * H);
    ck(sfnx_to_f16(up(normal((size_t) T * H, 9, 1.f)), x, (size_t) T * H, nullptr));
    float *out = dev<float>((size_t) P * N), *out2 = dev<float>((size_t) P * N);
    if constexpr (BIG) {
        moe_mm_16_big(w.dw, w.stride, djs, nj, n, x, SFNX_F32, out, nullptr);
        moe_mm_16_big(w_t.dw, w.stride, djs, nj, n, x, SFNX_F32, out2, nullptr);
    } else {
        moe_mm_16(w.dw, w.stride, djs, nj, n, x, SFNX_F32, out, nullptr);
        moe_mm_16(w_t.dw, w.stride, djs, nj, n, x, SFNX_F32, out2, nullptr);
    }
    const std::vector<float> ho = host(out, (size_t) P * N);
    same((tag + "f16 experts behind a table").c_str(), ho, host(out2, (size_t) P * N));
    const std::vector<uint16_t> bits = host(x, (size_t) T * H);
    std::vector<double> X(bits.size());
    for (size_t i = 0; i < X.size(); ++i) {
        _Float16 v;
        std::memcpy(&v, &bits[i], 2);
        X[i] = (double) v;
    }
    size_t bad = 0, count = 0;
    for (const J& j : js)
        for (int m = 0; m < j.n; ++m)
            for (int r = 0; r < N; ++r, ++count) {
                const Dot d = dot(&X[(size_t) j.y[m] * H], w.m[j.w].row(r), H, H);
                bad += !(std::fabs(ho[(size_t) j.out[m] * N + r] - d.v) <= d.err);
            }
    check((tag + "f16 experts").c_str(), bad, count);
}

void dense(const Store& w) {
    const int C = 9, N = w.dw.n_out, ldo = N + 5;
    uint8_t* xq = dev<uint8_t>((size_t) C * H);
    float *xs = dev<float>((size_t) C * nb(H)), *out = dev<float>((size_t) C * ldo);
    quantize_f8(SFNX_F32, up(normal((size_t) C * H, 8, 1.f)), H, C, H, xq, xs, nullptr);
    f8_gemm(w.dw, xq, xs, C, SFNX_F32, out, ldo, nullptr);
    const Mat X = rows8(host(xq, (size_t) C * H), host(xs, (size_t) C * nb(H)), C, H);
    const std::vector<float> ho = host(out, (size_t) C * ldo);
    size_t bad = 0;
    for (int c = 0; c < C; ++c)
        for (int r = 0; r < ldo; ++r) {
            const Dot d = r < N ? dot(X.row(c), w.m[0].row(r), H, 131 + nb(H)) : Dot{0, 0};   // past the row's end as it was
            bad += !(std::fabs(ho[(size_t) c * ldo + r] - d.v) <= d.err);
        }
    check("dense", bad, (size_t) C * ldo);
}

bool refuses() {
    try {
        f8_gemm(DW{(const void*) 4096, 0, 120, 128}, (const uint8_t*) 4096, (const float*) 4096, 1, SFNX_F32, (void*) 4096, 128, nullptr);
    } catch (const std::runtime_error& e) {
        return std::strstr(e.what(), "multiple of 16") != nullptr;
    }
    return false;
}

}  // namespace

int main() {
    try {
        const Store gu = store8(E, 2 * FF, H, 1), dn = store8(E, H, FF, 2), w = store16(E, 100, H, 3);
        const Store gu_t = tabled(gu, E), dn_t = tabled(dn, E), w_t = tabled(w, E);
        layer<Job>(5, gu, dn, gu_t, dn_t);
        layer<BigJob>(130, gu, dn, gu_t, dn_t);
        mm16<Job>(5, w, w_t);
        mm16<BigJob>(130, w, w_t);
        dense(gu);
        if (!refuses()) std::printf("a width of 120 was not refused\n"), ++failed;
        if (!failed) std::printf("ok\n");
    } catch (const std::exception& e) {
        std::printf("failed: %s\n", e.what());
        return 1;
    }
    return failed != 0;
}
