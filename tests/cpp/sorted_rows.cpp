// Rows grouped by expert, sorted and combined with their gradients, and low-rank adapters from C++, through the C++ face over the C ABI
// (sfnx/kernels.hpp); each against its formula on the host in 64 bits, the adapters also behind tables of pointers (DW::ep) bit for bit as
// with a stride, and with a rank whose call takes a workspace.  Bounds as in tests/rows_util.py.  Prints "ok" when every check holds; exit status
// 1 otherwise.  Built by the package's build step; run by tests/test_gpu_cpp_rows.py.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "sfnx/kernels.hpp"

using namespace sfnx;

namespace {

constexpr double STEP = 0x1p-23;

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
std::vector<float> normal(size_t n, uint64_t seed) {
    float* d = dev<float>(n);
    ck(sfnx_synth_normal(d, n, seed, 0, 1.f, nullptr));
    return host(d, n);
}
std::vector<uint16_t> f16(const std::vector<float>& v) {
    uint16_t* d = dev<uint16_t>(v.size());
    ck(sfnx_to_f16(up(v), d, v.size(), nullptr));
    return host(d, v.size());
}
double half_value(uint16_t h) {
    const int e = h >> 10 & 31, m = h & 1023;
    const double v = e ? std::ldexp(1024 + m, e - 25) : std::ldexp(m, -24);
    return h & 0x8000 ? -v : v;
}

int failed = 0;
void check(const char* what, size_t bad, size_t n) {
    std::printf("%s: %zu of %zu values off\n", what, bad, n);
    failed += bad != 0 || n == 0;
}
// got against want within a bound each
void near(const char* what, const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& bound) {
    size_t bad = 0;
    for (size_t i = 0; i < got.size(); ++i) bad += !(std::fabs(got[i] - want[i]) <= bound[i] + std::fabs(want[i]) * 0x1p-24);
    check(what, bad, got.size());
}

void rows() {
    constexpr int T = 70, K = 3, E = 9, H = 200, n = T * K;
    std::vector<int> ids(n);
    for (int i = 0; i < n; ++i) ids[i] = (i * 7 + i / 5) % (E + 1) - 1;   // some of none
    const int cap = n / PF_JOB + E;
    int *off = dev<int>(E + 1), *pos = dev<int>(n), *order = dev<int>(n), *njobs = dev<int>(2);
    BigJob* jobs = dev<BigJob>(cap);
    group_rows(up(ids), n, E, off, pos, order, jobs, njobs, cap, false, nullptr, 0, nullptr);
    std::vector<int> want(n, -1);
    size_t bad = 0, nj = 0;
    int V = 0;
    const auto off_h = host(off, E + 1);
    for (int e = 0; e < E; ++e) {
        bad += off_h[e] != V;
        const int v0 = V;
        for (int i = 0; i < n; ++i)
            if (ids[i] == e) want[i] = V++;
        nj += (V - v0 + PF_JOB - 1) / PF_JOB;
    }
    const auto pos_h = host(pos, n);
    for (int i = 0; i < n; ++i) bad += pos_h[i] != want[i];
    check("group_rows", bad + (off_h[E] != V) + (host(njobs, 2)[0] != (int) nj), n);

    const auto x = normal((size_t) T * H, 1), ys = normal((size_t) V * H, 2), w = normal(n, 3), dy = normal((size_t) T * H, 4);
    float *xs = dev<float>((size_t) V * H), *y = dev<float>((size_t) T * H), *dys = dev<float>((size_t) V * H), *dw = dev<float>(n);
    moe_sort_rows(4, up(x), H, T, K, H, pos, xs, H, V, nullptr);
    const auto xs_h = host(xs, (size_t) V * H);
    bad = 0;
    for (int i = 0; i < n; ++i)
        if (want[i] >= 0) bad += std::memcmp(&xs_h[(size_t) want[i] * H], &x[(size_t) (i / K) * H], H * 4) != 0;
    check("moe_sort_rows", bad, n);
    for (int form = 0; form < 2; ++form) {   // with weights; the gradient of sorting
        if (form == 0) moe_combine_sorted(SFNX_F32, up(ys), H, V, up(w), pos, T, K, H, SFNX_F32, y, H, nullptr);
        else moe_sort_rows_backward(SFNX_F32, up(ys), H, V, pos, T, K, H, SFNX_F32, y, H, nullptr);
        std::vector<double> v((size_t) T * H), b(v.size());
        for (int i = 0; i < n; ++i)
            for (int h = 0; h < H && want[i] >= 0; ++h) {
                const double t = (form == 0 ? w[i] : 1.0) * ys[(size_t) want[i] * H + h];
                v[(size_t) (i / K) * H + h] += t;
                b[(size_t) (i / K) * H + h] += K * STEP / 2 * std::fabs(t);
            }
        near(form == 0 ? "moe_combine_sorted" : "moe_sort_rows_backward", host(y, v.size()), v, b);
    }
    moe_combine_sorted_backward(SFNX_F32, up(dy), H, SFNX_F32, up(ys), H, V, up(w), pos, T, K, H, dys, H, dw, nullptr);
    std::vector<double> v((size_t) V * H), b(v.size()), vw(n), bw(n);
    for (int i = 0; i < n; ++i)
        for (int h = 0; h < H && want[i] >= 0; ++h) {
            const double g = dy[(size_t) (i / K) * H + h], t = g * ys[(size_t) want[i] * H + h];
            v[(size_t) want[i] * H + h] = w[i] * g;
            vw[i] += t;
            bw[i] += H * STEP / 2 * std::fabs(t);
        }
    near("moe_combine_sorted_backward, rows", host(dys, v.size()), v, b);
    near("moe_combine_sorted_backward, weights", host(dw, n), vw, bw);
}

void adapters(int R, int T) {
    constexpr int N = 3, NI = 72, NO = 50;
    const auto A = f16(normal((size_t) N * R * NI, 5)), B = f16(normal((size_t) N * NO * R, 6)), x = f16(normal((size_t) T * NI, 7));
    const auto base = normal((size_t) T * NO, 8);
    const std::vector<float> scale = {0.5f, -1.25f, 2.f};
    std::vector<int> ids(T);
    for (int t = 0; t < T; ++t) ids[t] = t * 5 % (N + 1) - 1;
    const int cap = T / PF_JOB + N;
    int *off = dev<int>(N + 1), *njobs = dev<int>(2);
    BigJob* jobs = dev<BigJob>(cap);
    group_rows(up(ids), T, N, off, nullptr, nullptr, jobs, njobs, cap, true, nullptr, 0, nullptr);
    std::vector<double> v(base.begin(), base.end()), b(v.size());
    for (int t = 0; t < T; ++t) {
        if (ids[t] < 0) continue;
        const uint16_t *a = &A[(size_t) ids[t] * R * NI], *bm = &B[(size_t) ids[t] * NO * R];
        std::vector<double> s(R), e(R);
        for (int r = 0; r < R; ++r) {
            for (int k = 0; k < NI; ++k) {
                const double p = half_value(a[r * NI + k]) * half_value(x[(size_t) t * NI + k]);
                s[r] += p;
                e[r] += NI * STEP * std::fabs(p);
            }
            e[r] = (e[r] + STEP * (std::fabs(s[r]) + e[r])) * std::fabs(scale[ids[t]]);
            s[r] *= scale[ids[t]];
        }
        for (int c = 0; c < NO; ++c) {
            double &o = v[(size_t) t * NO + c], &w = b[(size_t) t * NO + c];
            w = (R + 1) * STEP * std::fabs(o);
            for (int r = 0; r < R; ++r) {
                const double m = half_value(bm[c * R + r]);
                o += m * s[r];
                w += std::fabs(m) * (e[r] + (R + 1) * STEP * (std::fabs(s[r]) + e[r]));
            }
        }
    }
    DW dA, dB;
    dA.type = dB.type = SFNX_F16;
    dA.n_in = NI, dA.n_out = dB.n_in = R, dB.n_out = NO;
    const uint16_t *pa = up(A), *pb = up(B), *px = up(x);
    dA.p = pa, dB.p = pb;
    const size_t ws = sfnx_adapter_workspace(T, R, NI, SFNX_F16);
    void* w = ws ? dev<uint8_t>(ws) : nullptr;
    std::vector<float> first;
    for (int table = 0; table < 2; ++table) {
        if (table) {
            std::vector<const char*> ea, eb;
            for (int i = 0; i < N; ++i) ea.push_back((const char*) (pa + (size_t) i * R * NI)), eb.push_back((const char*) (pb + (size_t) i * NO * R));
            dA.ep = up(ea), dB.ep = up(eb);
        }
        float* out = up(base);
        adapter_mm(dA, 2 * (size_t) R * NI, dB, 2 * (size_t) NO * R, up(scale), N, jobs, njobs, cap, SFNX_F16, px, NI, out, SFNX_F32, out, NO, T, w, ws, nullptr);
        const auto got = host(out, v.size());
        if (table) check("adapter_mm with tables", std::memcmp(got.data(), first.data(), got.size() * 4) != 0, got.size());
        else near("adapter_mm", got, v, b);
        first = got;
    }
    bool threw = false;
    try {
        dB.n_in = R + 8;
        adapter_mm(dA, 0, dB, 0, nullptr, N, jobs, njobs, cap, SFNX_F16, px, NI, nullptr, SFNX_F32, w, NO, T, w, ws, nullptr);
    } catch (const std::runtime_error&) {
        threw = true;
    }
    check("ranks that differ refused", !threw, 1);
}

}  // namespace

int main() {
    try {
        rows();
        adapters(16, 40);
        adapters(48, 200);
    } catch (const std::exception& e) {
        std::printf("failed: %s\n", e.what());
        return 1;
    }
    if (!failed) std::printf("ok\n");
    return failed ? 1 : 0;
}
