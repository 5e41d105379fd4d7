// Experts and dense matrices in block-scaled 8-bit floating point (e4m3 values, an f32 scale for each 128 x 128 block of a
// matrix and for each 128 values of an activation row): the activation quantizer, the dense product, and the products
// grouped by expert over the routers' jobs.
#include "mm_mid.hpp"
#include "mm_tiles.hpp"

namespace sfnx {
namespace {
using namespace mm;

// ------------------------------------------------------------------------------------------------ the quantizer
// four values of a row from column k on, as fp32
template <int TYPE> __device__ __forceinline__ float4 load4(const void* x, size_t i) {
    if constexpr (TYPE == SFNX_F32) {
        return *reinterpret_cast<const float4*>((const float*) x + i);
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*) x + i);
        if constexpr (TYPE == SFNX_F16)
            return float4{h2f(u.x & 0xffff), h2f(u.x >> 16), h2f(u.y & 0xffff), h2f(u.y >> 16)};
        else
            return float4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                          __uint_as_float(u.y & 0xffff0000u)};
    }
}

// half a wavefront a block of 128 values
template <int TYPE>
__global__ void __launch_bounds__(256) k_quantize_f8(const void* __restrict__ x, int64_t ldx, int rows, int cols,
                                                     uint8_t* __restrict__ q, float* __restrict__ s) {
    const int nb = blocks_of(cols), c = 4 * (threadIdx.x % 32);
    for (int64_t i = (int64_t) blockIdx.x * 8 + threadIdx.x / 32; i < (int64_t) rows * nb; i += (int64_t) gridDim.x * 8) {
        const int64_t r = i / nb;
        const int k = (int) (i % nb) * BLK + c;
        float4 v = {0, 0, 0, 0};
        if (k < cols) v = load4<TYPE>(x, (size_t) (r * ldx + k));
        const float am = group_max<32>(fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))));
        const float sc = f8_scale(am);
        if (k < cols) *reinterpret_cast<uint32_t*>(q + r * cols + k) = f8_pack4(v.x, v.y, v.z, v.w, sc);
        if (c == 0) s[i] = sc;
    }
}

// ------------------------------------------------------------------------------------------------ checks
constexpr const char* ALIGN_MSG = "pointers must be 16-byte aligned";
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
    require(jobs != nullptr && njobs != nullptr, "null pointer");
    require(cap >= 0 && cap <= (1 << 20), "njobs out of range");
}
void check_f8_matrix(const void* A, size_t sa, int n_in, int n_out) {
    require(A != nullptr, "null pointer");
    require(al16(A), ALIGN_MSG);
    require(n_in > 0 && n_in % 16 == 0 && n_in <= (1 << 20), "input width must be a multiple of 16, at most 2^20");
    require(n_out > 0 && n_out <= (1 << 20), "n_out out of range");
    require(stride_ok(sa, sfnx_f8_matrix_bytes(n_out, n_in)), "expert stride smaller than a matrix");
    require(sa % 16 == 0, "expert stride must be a multiple of 16");
}
void check_f8_rows(const uint8_t* xq, const float* xs) {
    require(xq != nullptr && xs != nullptr, "null pointer");
    require(al16(xq), ALIGN_MSG);
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
        require(cols > 0 && cols % 16 == 0, "cols must be a multiple of 16");
        require(rows >= 0, "rows out of range");
        require(ldx >= cols && ldx % 16 == 0, "ldx must be a multiple of 16, at least cols");
        if (rows == 0) return;
        require(x != nullptr && q != nullptr && s != nullptr, "null pointer");
        require(al16(x) && al16(q), ALIGN_MSG);
        const int64_t items = (int64_t) rows * blocks_of(cols);
        const unsigned grid = (unsigned) std::min<int64_t>((items + 7) / 8, 1 << 16);
        hipStream_t h = stream_of(st);
        if (type == SFNX_F32) k_quantize_f8<SFNX_F32><<<grid, 256, 0, h>>>(x, ldx, rows, cols, q, s);
        else if (type == SFNX_F16) k_quantize_f8<SFNX_F16><<<grid, 256, 0, h>>>(x, ldx, rows, cols, q, s);
        else k_quantize_f8<SFNX_BF16><<<grid, 256, 0, h>>>(x, ldx, rows, cols, q, s);
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
        if (getenv("SFNX_MID")) {
            int v = atoi(getenv("SFNX_MID"));
            hipStream_t h = stream_of(st);
            if (out_type == SFNX_F32) { if (v == 42) launch_mid_as<F8X, 4, 2>(a, h); if (v == 41) launch_mid_as<F8X, 4, 1>(a, h); if (v == 22) launch_mid_as<F8X, 2, 2>(a, h); if (v == 21) launch_mid_as<F8X, 2, 1>(a, h); if (v==44) launch_mid_as<F8X,4,4>(a,h); }
            else { if (v == 44) launch_mid_as<F8, 4, 4>(a, h); if (v == 42) launch_mid_as<F8, 4, 2>(a, h); if (v == 41) launch_mid_as<F8, 4, 1>(a, h); if (v == 22) launch_mid_as<F8, 2, 2>(a, h); if (v == 24) launch_mid_as<F8, 2, 4>(a, h); if (v==21) launch_mid_as<F8,2,1>(a,h); }
            if (v == 3) { if (out_type == SFNX_F32) launch_narrow<F8X>(a, (C + 63) / 64, h); else launch_narrow<F8>(a, (C + 63) / 64, h); }
            if (v > 2) return;
        }
        if (C <= FEW_M) launch_few<F8X, STORE, false>(a, 1, stream_of(st));
        else if (out_type == SFNX_F32) launch_tiles<F8X, STORE>(a, (C + BM1 - 1) / BM1, stream_of(st));
        else launch_tiles<F8, STORE>(a, (C + BM1 - 1) / BM1, stream_of(st));
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
        launch_tiles<F8X, SWIGLU>(a, njobs_cap, stream_of(st));
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
        if (out_type == SFNX_F32) launch_tiles<F8X, STORE>(a, njobs_cap, stream_of(st));
        else launch_tiles<F8, STORE>(a, njobs_cap, stream_of(st));
    });
}
