// Matrix products of 8-bit (e4m3, with a scale for each block of 128) and 16-bit floating-point weights, dense and grouped
// by expert: out[job.out[m]][n] = sum_k W_e[n][k] x[job.y[m]][k], on the matrix cores.
//
// One K step is 128 bytes of a row: one scale block of 128 e4m3 values, or 64 f16 / bf16 values.  The weights are the A operand
// (16 rows), the activations the B operand (16 tokens): lane l = 16 q + r holds bytes 16 q .. 16 q + 15 and 64 + 16 q ..
// 64 + 16 q + 15 of row r's step for both (the order of k within a step does not matter to the sum), and of the result token
// r, rows 4 q .. 4 q + 3: four consecutive values of an output row.
//
// e4m3 steps start their matrix instructions from zero and add the result times the block's two scales in fp32.  There are two
// forms.  F8, v_mfma_f32_16x16x128_f8f6f4: measured, it adds the products of 8 consecutive k to a common unit of 2^-13 of
// the largest (a product 2^-14 of a neighbour's size is lost) and these sums in fp32: an output is off by at most 7 2^-13 of the
// sum of its terms' sizes, on normal data by 1.5e-5 of the result's norm, where large terms cancel by up to all of it.  It serves
// outputs that are rounded to 16 bits (2^-9, 2^-12) anyway.  F8X: the values converted to f16,
// exactly, and summed by four v_mfma_f32_16x16x32_f16, whose sums are fp32's (1e-8 on the same data), at half the rate; it
// serves outputs kept in 32 bits, the scales of quantized ones, and products of few rows, which wait for the weights anyway.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace sfnx {
namespace mm {

typedef int int8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));

typedef _Float16 half2f __attribute__((ext_vector_type(2)));

enum Elem { F8, F8X, F16, BF16 };
template <Elem EL> constexpr bool IS8 = EL == F8 || EL == F8X;
template <Elem EL> constexpr int ESZ = IS8<EL> ? 1 : 2;   // bytes of a weight or activation
constexpr int CUS = 256;                                   // compute units
constexpr int STEP = 128;                                  // bytes of a row in a K step
constexpr int BLK = 128;                                   // values of a scale block
constexpr float F8_MAX = 448.f, F8_INV = 1.f / 448.f, S_MIN = 0x1p-126f;

// a lane's 32 bytes of a row's K step
struct Frag {
    uint4 lo, hi;
};

// the matrix instruction's operand of a fragment
struct FragX {
    half8v h[4];
};
template <Elem EL> struct OperandOf { typedef Frag type; };
template <> struct OperandOf<F8X> { typedef FragX type; };
template <Elem EL> using Operand = typename OperandOf<EL>::type;
__device__ __forceinline__ half8v f8_to_f16(uint32_t a, uint32_t b) {
    const half2f v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true),
                         __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true)};
    return half8v{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}
template <Elem EL> __device__ __forceinline__ Operand<EL> operand(const Frag& f) {
    if constexpr (EL == F8X) return FragX{{f8_to_f16(f.lo.x, f.lo.y), f8_to_f16(f.lo.z, f.lo.w), f8_to_f16(f.hi.x, f.hi.y), f8_to_f16(f.hi.z, f.hi.w)}};
    else return f;
}

// the product of a K step of e4m3 values, without its scales
template <Elem EL> __device__ __forceinline__ float4v step_dot(const Operand<EL>& w, const Operand<EL>& x) {
    float4v d = {};
    if constexpr (EL == F8) {
        const int8v a = {(int) w.lo.x, (int) w.lo.y, (int) w.lo.z, (int) w.lo.w, (int) w.hi.x, (int) w.hi.y, (int) w.hi.z, (int) w.hi.w};
        const int8v b = {(int) x.lo.x, (int) x.lo.y, (int) x.lo.z, (int) x.lo.w, (int) x.hi.x, (int) x.hi.y, (int) x.hi.z, (int) x.hi.w};
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, d, 0, 0, 0, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.h[i], x.h[i], d, 0, 0, 0);
    }
    return d;
}
__device__ __forceinline__ float4v scaled_add(float4v d, float s, float4v acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(d[i], s, acc[i]);
    return acc;
}

// acc += W . x over one K step; s: the product of the step's scales (e4m3 only)
template <Elem EL> __device__ __forceinline__ float4v step_mma(const Operand<EL>& w, const Operand<EL>& x, float4v acc, float s) {
    if constexpr (IS8<EL>) {
        return scaled_add(step_dot<EL>(w, x), s, acc);
    } else if constexpr (EL == F16) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, w.lo), __builtin_bit_cast(half8v, x.lo), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, w.hi), __builtin_bit_cast(half8v, x.hi), acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, w.lo), __builtin_bit_cast(bf8v, x.lo), acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, w.hi), __builtin_bit_cast(bf8v, x.hi), acc, 0, 0, 0);
    }
}

// a matrix of the 8-bit store: e4m3 values [rows][cols], then the f32 scales of its 128 x 128 blocks
__host__ __device__ __forceinline__ int blocks_of(int n) { return (n + BLK - 1) / BLK; }
__device__ __forceinline__ const float* scales_of(const uint8_t* mat, int rows, int cols) {
    return reinterpret_cast<const float*>(mat + (size_t) rows * cols);
}

// ------------------------------------------------------------------------------------------------ e4m3 with a scale
// s = max(max |x| c, 2^-126) over a block's finite values, c = 1 / 448 rounded to fp32; q = e4m3(x / s), one rounding of the
// fp32 quotient, at most 448 in size.  The floor of s keeps the quotient of a block of zeros (or of values below 448 2^-126) defined.  What is not
// finite becomes the type's NaN.
//
// The quotient: with r = 1 / s rounded, x r is within 1.5 units of x / s, and ((x r) s - x) r, both products fused, is taken away
// (Markstein's step): three instructions for a division's ten.  r is within 2^-24 of 1 / s, so what is rounded last is within
// 1.5 2^-24 units of x / s; its rounding could be another one only beside a border of fp32, which matters to a code only at
// e4m3's ties.  Compared there: all 2^23 scales of a binade with the seven values nearest to each of its ties, 940 million
// quotients, every one the division's.  The remainder has to stay above the smallest numbers, so scales below 2^-90 divide; so
// do blocks with values that are not finite.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }   // not finite: 0x7f800000 on
struct F8Scale {
    float s, r;
    bool plain;   // by division, value by value
};
__device__ __forceinline__ float finite_abs(float v) { return abs_bits(v) < 0x7f800000u ? fabsf(v) : 0.f; }
// amax: over the block's finite values; all_finite: whether there are others
__device__ __forceinline__ F8Scale f8_scale(float amax, bool all_finite) {
    const float s = fmaxf(amax * F8_INV, S_MIN);
    return F8Scale{s, 1.f / s, !all_finite || s < 0x1p-90f};
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d, const F8Scale& k) {
    const float v[4] = {a, b, c, d};
    float t[4];
    if (!k.plain) {   // at most 448 (1 + 2^-22), which rounds to 448
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = v[i] * k.r;
            t[i] = fmaf(-fmaf(q, k.s, -v[i]), k.r, q);   // in this order a zero keeps its sign: -0 s + 0 = +0, then (-0) r + -0 = -0
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = fminf(fmaxf(v[i] / k.s, -F8_MAX), F8_MAX);
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], r, true);
    uint32_t u = (uint32_t) r;
    if (k.plain)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (abs_bits(v[i]) >= 0x7f800000u) u = (u & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
    return u;
}

// ------------------------------------------------------------------------------------------------ outputs
__device__ __forceinline__ uint32_t bf16_bits(float f) { return (uint32_t) __builtin_bit_cast(uint16_t, (__bf16) f); }
__device__ __forceinline__ uint32_t half_bits(uint32_t type, float f) { return type == SFNX_F16 ? (uint32_t) f2h(f) : bf16_bits(f); }
// four consecutive values of an output row from element i on, those below `left`, in the output's type (one rounding);
// vec: the row's elements i .. i + 3 are aligned to their size
__device__ __forceinline__ void store4(void* out, uint32_t type, size_t i, float4v v, int left, bool vec) {
    if (vec && left >= 4) {
        if (type == SFNX_F32)
            *reinterpret_cast<float4v*>((float*) out + i) = v;
        else
            *reinterpret_cast<uint2*>((uint16_t*) out + i) = uint2{half_bits(type, v[0]) | half_bits(type, v[1]) << 16,
                                                                   half_bits(type, v[2]) | half_bits(type, v[3]) << 16};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) {
            if (type == SFNX_F32) ((float*) out)[i + e] = v[e];
            else ((uint16_t*) out)[i + e] = (uint16_t) half_bits(type, v[e]);
        }
}
__host__ __device__ inline int out_size(uint32_t type) { return type == SFNX_F32 ? 4 : 2; }
inline bool out_type_ok(uint32_t type) { return type == SFNX_F32 || type == SFNX_F16 || type == SFNX_BF16; }

// What a launch multiplies.  dense_c > 0: no job list, dense_c rows of x times one matrix.
struct Args {
    const uint8_t* A;        // expert matrices, sa bytes apart (0: a table of their pointers)
    size_t sa;
    int n_in, n_out;         // columns and rows of a matrix
    const void* jobs;        // sfnx_job or sfnx_bigjob
    const int* njobs;
    int dense_c;
    const uint8_t* x;        // activation rows of n_in values
    const float* xs;         // e4m3: their scales, [rows][ceil(n_in / 128)]
    void* out;               // rows of ldo values
    float* out_s;            // quantized outputs: their scales
    uint32_t out_type;
    int ldo;
    int vec;                 // four consecutive outputs at a multiple of 4 are aligned to their size
    int slices = 0;          // of a matrix, 256 rows each
    bool across = false;     // tiles: an XCD's are slices of all groups, not groups' slices
};

// workgroups of a launch: a job's slices for each job; a launch holds fewer than 2^32 threads
inline unsigned grid_of(int slices, int jobs, int threads) {
    require((int64_t) slices * jobs * threads < ((int64_t) 1 << 32), "too many jobs for one launch");
    return (unsigned) slices * (unsigned) jobs;
}

// an address that is always readable, for the lanes past a row's end
static __device__ const uint4 ZERO16 = {0, 0, 0, 0};

// a pointer that all lanes share, in scalar registers
__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
    const uint64_t u = (uint64_t) p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t) u), hi = __builtin_amdgcn_readfirstlane((uint32_t) (u >> 32));
    return (const uint8_t*) ((uint64_t) hi << 32 | lo);
}

// Copies to LDS as lds_copy_async, but no compiler barrier, so LDS reads of other places move across them; the order against
// vm_wait and lds_barrier stays.  to: a wave-uniform LDS address (Lds::at); lane l's bytes land at to + 16 l (copy4: 4 l).
// copy16's source is a uniform base and a lane's 32-bit offset, or a lane's pointer.
__device__ __forceinline__ void copy16(const uint8_t* base, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to) : "m0");
}
__device__ __forceinline__ void copy16(const uint8_t* p, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(to) : "m0");
}
__device__ __forceinline__ void copy4(const void* p, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(to) : "m0");
}
__device__ __forceinline__ void copy4(const uint8_t* base, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(to) : "m0");
}
// a workgroup's LDS, as a pointer to read through and as the address copies take: cast once, where the compiler sees the array
// itself (a generic pointer's cast tests it for null each time)
struct Lds {
    uint8_t* p;
    uint32_t base;
    __device__ __forceinline__ uint32_t at(const void* q) const { return base + (uint32_t) ((const uint8_t*) q - p); }
};
__device__ __forceinline__ Lds lds_of(uint8_t* p) {
    return Lds{p, (uint32_t) reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*) p)};
}

enum Mode { STORE, SWIGLU };

}  // namespace mm
}  // namespace sfnx
