// Experts and dense matrices in block-scaled 8-bit floating point (e4m3 values, an f32 scale for each 128 x 128 block of a
// matrix and for each 128 values of an activation row): the activation quantizer, the dense product, and the products
// grouped by expert over the routers' jobs.
#include "mm_mid.hpp"
#include "mm_tiles.hpp"

namespace sfnx {
namespace {
using namespace mm;

// ------------------------------------------------------------------------------------------------ the quantizer
// eight values of a row, as fp32
template <int TYPE> __device__ __forceinline__ void load8(const void* x, size_t i, float (&v)[8]) {
    if constexpr (TYPE == SFNX_F32) {
        const float4 a = reinterpret_cast<const float4*>((const float*) x + i)[0], b = reinterpret_cast<const float4*>((const float*) x + i)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*) x + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = TYPE == SFNX_F16 ? h2f(w[k] & 0xffff) : __uint_as_float(w[k] << 16);
            v[2 * k + 1] = TYPE == SFNX_F16 ? h2f(w[k] >> 16) : __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}

// 16 lanes a block of 128 values.  A workgroup's 16 groups of lanes are GX along a row (as many as it has blocks, at most 16)
// by 16 / GX rows.  Bound by its reads and writes: 4096 x 4096 bf16, 51 MB, 9.3 us (5.5 TB/s; four rows a lane, all requested
// before the first is used, 11.7).
template <int TYPE>
__global__ void __launch_bounds__(256) k_quantize_f8(const void* __restrict__ x, int64_t ldx, int rows, int cols, int gx_log,
                                                     uint8_t* __restrict__ q, float* __restrict__ s) {
    const int g = threadIdx.x / 16, nb = blocks_of(cols), b = (blockIdx.y << gx_log) + (g & ((1 << gx_log) - 1)), k = b * BLK + 8 * (threadIdx.x % 16);
    const int r = blockIdx.x * (16 >> gx_log) + (g >> gx_log);
    const bool in = r < rows && k < cols;
    float v[8] = {};
    if (in) load8<TYPE>(x, (size_t) (r * ldx + k), v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
    top = (uint32_t) group_reduce<16>((int) top, [](int a, int c) { return max(a, c); });
    float am = __uint_as_float(top);
    const bool fin = top < 0x7f800000u;
    if (__any(!fin)) {
        am = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) am = fmaxf(am, finite_abs(v[i]));
        am = group_max<16>(am);
    }
    const F8Scale sc = f8_scale(am, fin);
    const uint2 o = {f8_pack4(v[0], v[1], v[2], v[3], sc), f8_pack4(v[4], v[5], v[6], v[7], sc)};
    if (in) *reinterpret_cast<uint2*>(q + (size_t) r * cols + k) = o;
    if (r < rows && b < nb && threadIdx.x % 16 == 0) s[(size_t) r * nb + b] = sc.s;
}

template <int TYPE> void quantize(const void* x, int64_t ldx, int rows, int cols, uint8_t* q, float* s, hipStream_t st) {
    const int nb = blocks_of(cols);
    int gx_log = 0;
    while (gx_log < 4 && (1 << gx_log) < nb) ++gx_log;
    const int gx = 1 << gx_log, gy = 16 / gx;
    k_quantize_f8<TYPE><<<dim3((rows + gy - 1) / gy, (nb + gx - 1) / gx), 256, 0, st>>>(x, ldx, rows, cols, gx_log, q, s);
}

// ------------------------------------------------------------------------------------------------ checks
constexpr const char* ALIGN_MSG = "pointers must be 16-byte aligned";
constexpr const char* SCALES_MSG = "scales must be 4-byte aligned";
bool al16(const void* p) { return ((uintptr_t) p & 15) == 0; }
void check_out(const void* out, uint32_t out_type) {
    require(out_type_ok(out_type), "out type must be F32 (0), F16 (1) or BF16 (30)");
    require(out != nullptr, "null pointer");
    require(((uintptr_t) out & (out_size(out_type) - 1)) == 0, "out must be aligned to its type");
}
// rows of n_out values ldo apart whose aligned groups of four can be stored at once
int vec_ok(const void* out, uint32_t out_type, int64_t ldo) {
    return ((uintptr_t) out & (4 * out_size(out_type) - 1)) == 0 && ldo % 4 == 0;
}
void check_jobs(const void* jobs, const int* njobs, int cap) {
    require(cap >= 0 && cap <= (1 << 20), "njobs out of range");
    require(cap == 0 || (jobs != nullptr && njobs != nullptr), "null pointer");
}
void check_f8_matrix(const void* A, size_t sa, int n_in, int n_out) {
    require(A != nullptr, "null pointer");
    require(al16(A), ALIGN_MSG);
    require(n_in > 0 && n_in % 16 == 0 && n_in <= (1 << 20), "input width must be a multiple of 16, at most 2^20");
    require(n_out > 0 && n_out <= (1 << 20), "n_out out of range");
    require((uint64_t) n_out * n_in < ((uint64_t) 1 << 32), "a matrix must be smaller than 4 GiB");
    require(stride_ok(sa, sfnx_f8_matrix_bytes(n_out, n_in)), "expert stride smaller than a matrix");
    require(sa % 16 == 0, "expert stride must be a multiple of 16");
}
void check_f8_rows(const uint8_t* xq, const float* xs) {
    require(xq != nullptr && xs != nullptr, "null pointer");
    require(al16(xq), ALIGN_MSG);
    require(((uintptr_t) xs & 3) == 0, SCALES_MSG);
}

// A dense product of more than 16 rows: the form of the least estimated time.  A form's tile takes `one` us for 4096 columns
// when all tiles run at once, `more` in further rounds of 256 workgroups, and `fixed` us whatever the columns; fitted to
// matrices of 256 to 4096 rows, 512 to 4096 columns and 17 to 4096 rows of activations.  Of them, with 4096 columns, us in a
// graph, into bf16 and (F8X) into f32, whose third form has 64 rows by 32:
//   rows x rows      32x16 mid     32x32 mid     32x64 mid     64x128 streamed  64x256 streamed  256x256 grouped
//   128 x 256         9.7   9.8    11.7  11.8    15.8  18.1     18.9  29.7       28.1  40.6       37.0  69.5
//   256 x 1024       16.8  17.0    11.9  12.2    15.9  18.4     19.3  30.4       28.5  41.1       55.7 122
//   512 x 2048       58.7  59.0    38.1  42.3    30.5  35.5     23.9  34.1       31.4  42.7       61.2 126
//   1024 x 4096     226   226     143   162     114   134       46.7  66.1       34.8  47.5       66.0 128
//   4096 x 4096                                                168   238        120   174         76.2 138
struct DenseForm {
    int rows, cols;
    float one, more, fixed;
};
template <Elem EL> void dense_many(const Args& a, hipStream_t st) {
    constexpr DenseForm forms[2][6] = {
        {{32, 16, 4.4f, 6.6f, 0.5f}, {32, 32, 6.3f, 8.1f, 0.5f}, {32, 64, 10.5f, 12.5f, 0.5f}, {64, 128, 21.f, 21.f, 1.5f}, {64, 256, 28.f, 29.f, 1.7f}, {256, 256, 47.f, 51.f, 9.f}},
        {{32, 16, 4.5f, 6.6f, 0.5f}, {32, 32, 6.5f, 9.1f, 0.5f}, {64, 32, 13.f, 15.5f, 0.5f}, {64, 128, 32.f, 31.f, 1.5f}, {64, 256, 38.f, 39.f, 1.7f}, {256, 256, 110.f, 112.f, 9.f}}};
    int best = 0;
    float least = 0.f;
    for (int i = 0; i < 6; ++i) {
        const DenseForm& f = forms[EL == F8X][i];
        const int64_t tiles = (int64_t) ((a.dense_c + f.rows - 1) / f.rows) * ((a.n_out + f.cols - 1) / f.cols), rounds = (tiles + CUS - 1) / CUS;
        const float t = rounds * ((rounds == 1 ? f.one : f.more) * a.n_in / 4096.f + f.fixed);
        if (i == 0 || t < least) best = i, least = t;
    }
    const int jobs = (a.dense_c + BM1 - 1) / BM1;
    switch (best) {
        case 0: return launch_mid<EL, 2, 1>(a, st);
        case 1: return launch_mid<EL, 2, 2>(a, st);
        case 2: return launch_mid<EL, EL == F8X ? 4 : 2, EL == F8X ? 2 : 4>(a, st);
        case 3: return launch_stream<EL, STORE, 1>(a, jobs, st);
        case 4: return launch_stream<EL, STORE>(a, jobs, st);
        default: return launch_group<EL>(a, jobs, st);
    }
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" size_t sfnx_f8_matrix_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    const size_t n = (size_t) rows * cols + 4 * (size_t) blocks_of(rows) * blocks_of(cols);
    return (n + 15) / 16 * 16;
}

extern "C" int sfnx_quantize_f8(uint32_t type, const void* x, int64_t ldx, int rows, int cols, uint8_t* q, float* s, void* st) {
    return guarded("sfnx_quantize_f8", [&] {
        require(out_type_ok(type), "x type must be F32 (0), F16 (1) or BF16 (30)");
        require(cols > 0 && cols % 16 == 0 && cols <= (1 << 20), "cols must be a multiple of 16, at most 2^20");
        require(rows >= 0 && rows < (1 << 24), "rows out of range");   // with a workgroup a row, fewer than 2^32 threads
        require(ldx >= cols && ldx % 16 == 0, "ldx must be a multiple of 16, at least cols");
        if (rows == 0) return;
        require(x != nullptr && q != nullptr && s != nullptr, "null pointer");
        require(al16(x) && al16(q), ALIGN_MSG);
        require(((uintptr_t) s & 3) == 0, SCALES_MSG);
        hipStream_t h = stream_of(st);
        if (type == SFNX_F32) quantize<SFNX_F32>(x, ldx, rows, cols, q, s, h);
        else if (type == SFNX_F16) quantize<SFNX_F16>(x, ldx, rows, cols, q, s, h);
        else quantize<SFNX_BF16>(x, ldx, rows, cols, q, s, h);
    });
}

extern "C" int sfnx_f8_gemm(const void* W, int rows, int cols, const uint8_t* xq, const float* xs, int C, uint32_t out_type,
                            void* out, int ldo, void* st) {
    return guarded("sfnx_f8_gemm", [&] {
        check_f8_matrix(W, 0, cols, rows);
        require(C >= 0 && C <= (1 << 24), "C out of range");
        require(ldo >= rows, "ldo smaller than rows");
        if (C == 0) return;
        check_f8_rows(xq, xs);
        check_out(out, out_type);
        Args a{(const uint8_t*) W, sfnx_f8_matrix_bytes(rows, cols), cols, rows, nullptr, nullptr, C, xq, xs, out, nullptr, out_type, ldo,
               vec_ok(out, out_type, ldo)};
        if (C <= FEW_M) launch_few<F8X, STORE, false>(a, 1, stream_of(st));
        else if (out_type == SFNX_F32) dense_many<F8X>(a, stream_of(st));
        else dense_many<F8>(a, stream_of(st));
    });
}

extern "C" int sfnx_moe_gate_up_swiglu_f8(const void* A, size_t sa, int n_in, int ff, const sfnx_job* jobs, const int* njobs,
                                          int njobs_max, const uint8_t* xq, const float* xs, float* h, void* st) {
    return guarded("sfnx_moe_gate_up_swiglu_f8", [&] {
        require(ff > 0 && ff % 16 == 0 && ff <= (1 << 19), "FF must be a multiple of 16");
        check_f8_matrix(A, sa, n_in, 2 * ff);
        check_jobs(jobs, njobs, njobs_max);
        if (njobs_max == 0) return;
        check_f8_rows(xq, xs);
        check_out(h, SFNX_F32);
        Args a{(const uint8_t*) A, sa, n_in, 2 * ff, jobs, njobs, 0, xq, xs, h, nullptr, SFNX_F32, ff, vec_ok(h, SFNX_F32, ff)};
        launch_few<F8X, SWIGLU, false>(a, njobs_max, stream_of(st));
    });
}

extern "C" int sfnx_moe_down_f8(const void* A, size_t sa, int n_in, int n_out, const sfnx_job* jobs, const int* njobs,
                                int njobs_max, const float* h, uint32_t out_type, void* out, void* st) {
    return guarded("sfnx_moe_down_f8", [&] {
        check_f8_matrix(A, sa, n_in, n_out);
        require(n_in <= 8192, "input width must be at most 8192");
        check_jobs(jobs, njobs, njobs_max);
        if (njobs_max == 0) return;
        require(h != nullptr, "null pointer");
        require(al16(h), ALIGN_MSG);
        check_out(out, out_type);
        Args a{(const uint8_t*) A, sa, n_in, n_out, jobs, njobs, 0, (const uint8_t*) h, nullptr, out, nullptr, out_type, n_out,
               vec_ok(out, out_type, n_out)};
        launch_few<F8X, STORE, true>(a, njobs_max, stream_of(st));
    });
}

extern "C" int sfnx_moe_gate_up_swiglu_f8_big(const void* A, size_t sa, int n_in, int ff, const sfnx_bigjob* jobs,
                                              const int* njobs, int njobs_cap, const uint8_t* xq, const float* xs, uint8_t* hq,
                                              float* hs, void* st) {
    return guarded("sfnx_moe_gate_up_swiglu_f8_big", [&] {
        require(ff > 0 && ff % 16 == 0 && ff <= (1 << 19), "FF must be a multiple of 16");
        check_f8_matrix(A, sa, n_in, 2 * ff);
        check_jobs(jobs, njobs, njobs_cap);
        if (njobs_cap == 0) return;
        check_f8_rows(xq, xs);
        check_f8_rows(hq, hs);
        Args a{(const uint8_t*) A, sa, n_in, 2 * ff, jobs, njobs, 0, xq, xs, hq, hs, SFNX_F32, ff, 1};
        launch_stream<F8X, SWIGLU>(a, njobs_cap, stream_of(st));
    });
}

extern "C" int sfnx_moe_down_f8_big(const void* A, size_t sa, int n_in, int n_out, const sfnx_bigjob* jobs, const int* njobs,
                                    int njobs_cap, const uint8_t* hq, const float* hs, uint32_t out_type, void* out, void* st) {
    return guarded("sfnx_moe_down_f8_big", [&] {
        check_f8_matrix(A, sa, n_in, n_out);
        check_jobs(jobs, njobs, njobs_cap);
        if (njobs_cap == 0) return;
        check_f8_rows(hq, hs);
        check_out(out, out_type);
        Args a{(const uint8_t*) A, sa, n_in, n_out, jobs, njobs, 0, hq, hs, out, nullptr, out_type, n_out, vec_ok(out, out_type, n_out)};
        if (out_type == SFNX_F32) launch_stream<F8X, STORE>(a, njobs_cap, stream_of(st));
        else launch_stream<F8, STORE>(a, njobs_cap, stream_of(st));
    });
}
