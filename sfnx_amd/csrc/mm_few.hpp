// Products of few rows (jobs of up to 16): the weight stream alone counts, each weight byte is used once.  Bound by HBM where
// there are many jobs (16 tokens: 5.2 TB/s of gate|up weights, 4.2 of down's), by a chain of loads where there are few: the job,
// then for each of a wavefront's steps x and the first row tile, and after their product the second (gate|up of one token, two
// steps a wavefront: five round trips, the kernel 8.2 us for 23 MB; down 5.9 for 12; a dense row of 2048 by 1024 5.2).
#pragma once

#include "mm.hpp"

namespace sfnx {
namespace mm {

constexpr int FEW_WAVES = 8, FEW_THREADS = FEW_WAVES * WAVE, FEW_M = 16;

// the lane's 32 bytes of the step at byte k0 of a row; zero past the row's end (both operands', whatever lies there)
__device__ __forceinline__ Frag load_frag(const uint8_t* row, int k0, int q, int row_bytes) {
    Frag f{};
    const int k = k0 + 16 * q;
    if (k < row_bytes) f.lo = *reinterpret_cast<const uint4*>(row + k);
    if (k + 64 < row_bytes) f.hi = *reinterpret_cast<const uint4*>(row + k + 64);
    return f;
}

// A block's wavefronts are WK along K and 8 / WK along the rows; a wavefront owns two row tiles of 16 (SWIGLU: the gate
// tile and its up tile) and the steps wk, wk + WK, ... of K.  The partial sums meet in LDS and are added in wavefront order.
// QH: x holds fp32 rows, quantized here into LDS (each block quantizes the job's rows: a few thousand values).
template <Elem EL, Mode MODE, int WK, bool QH>
__global__ void __launch_bounds__(FEW_THREADS, EL == F8X && !QH ? 6 : 8) k_mm_few(Args a) {
    constexpr int WR = FEW_WAVES / WK, ROWS = MODE == SWIGLU ? 16 * WR : 32 * WR;   // output values of a block
    __shared__ float red[WK][WR][2][FEW_M][16];
    extern __shared__ __align__(16) uint8_t hq[];   // QH: [16][pitch] e4m3, then [16][blocks] scales
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, wk = wave % WK, wr = wave / WK;
    const int n_eff = MODE == SWIGLU ? a.n_out / 2 : a.n_out, nsl = (n_eff + ROWS - 1) / ROWS;
    const int sl = blockIdx.x % nsl, ji = blockIdx.x / nsl;
    const sfnx_job* jb = (const sfnx_job*) a.jobs + ji;
    int n, e = 0, y;
    if (a.dense_c > 0) {
        n = a.dense_c;
        y = min(r, n - 1);
    } else {   // the job's fields at once with the count that says whether it is one; a lane without a row takes the first
        const int nj = *a.njobs, yr = jb->y[r], y0 = jb->y[0];
        n = __builtin_amdgcn_readfirstlane(min(jb->n, FEW_M));
        e = __builtin_amdgcn_readfirstlane(jb->w);
        if (ji >= nj || n <= 0) return;
        y = r < n ? yr : y0;
    }
    const uint8_t* mat = expert_at(a.A, a.sa, e);
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const int f0 = sl * ROWS + (MODE == SWIGLU ? 16 : 32) * wr;
    int row0[2];   // the wavefront's row tiles
    row0[0] = f0;
    row0[1] = MODE == SWIGLU ? n_eff + f0 : f0 + 16;
    const uint8_t* wrow[2];
    const float* ws[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        row0[t] = min(row0[t], a.n_out - 1);
        wrow[t] = mat + (size_t) min(row0[t] + r, a.n_out - 1) * rb;
        if (IS8<EL>) ws[t] = scales_of(mat, a.n_out, a.n_in) + (size_t) (row0[t] / BLK) * nb;
    }
    // QH: the first step's weights are on their way while the job's rows are quantized
    Frag w0[2];
    if (QH && wk < steps)
#pragma unroll
        for (int t = 0; t < 2; ++t) w0[t] = load_frag(wrow[t], wk * STEP, q, rb);
    const int pitch = steps * STEP + 16;
    float* hs = reinterpret_cast<float*>(hq + 16 * pitch);
    if constexpr (QH) {   // half a wavefront a block of 128 values
        const float* h = reinterpret_cast<const float*>(a.x);
        for (int i = threadIdx.x / 32; i < n * nb; i += FEW_THREADS / 32) {
            const int m = i / nb, b = i % nb, c = 4 * (threadIdx.x % 32), k = b * BLK + c;
            const int yy = a.dense_c > 0 ? m : jb->y[m];
            float4 v = {0, 0, 0, 0};
            if (k < a.n_in) v = *reinterpret_cast<const float4*>(h + (size_t) yy * a.n_in + k);
            const uint32_t top = max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
            const bool fin = (uint32_t) group_reduce<32>((int) top, [](int a, int b) { return max(a, b); }) < 0x7f800000u;
            const float am = group_max<32>(fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))));
            const F8Scale s = f8_scale(am, fin);
            *reinterpret_cast<uint32_t*>(hq + m * pitch + k) = f8_pack4(v.x, v.y, v.z, v.w, s);
            if (c == 0) hs[m * nb + b] = s.s;
        }
        lds_barrier();
    }
    const int m = r < n ? r : 0;
    const uint8_t* xrow = QH ? hq + m * pitch : a.x + (size_t) y * rb;
    const float* xs = QH ? hs + m * nb : a.xs + (size_t) y * nb;
    float4v acc[2] = {};
    for (int s = wk; s < steps; s += WK) {
        Frag x;
        if constexpr (QH) {
            x.lo = *reinterpret_cast<const uint4*>(xrow + s * STEP + 16 * q);
            x.hi = *reinterpret_cast<const uint4*>(xrow + s * STEP + 16 * q + 64);
        } else {
            x = load_frag(xrow, s * STEP, q, rb);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Frag w = QH && s == wk ? w0[t] : load_frag(wrow[t], s * STEP, q, rb);
            acc[t] = step_mma<EL>(operand<EL>(w), operand<EL>(x), acc[t], IS8<EL> ? xs[s] * ws[t][s] : 1.f);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) *reinterpret_cast<float4v*>(&red[wk][wr][t][r][4 * q]) = acc[t];
    __syncthreads();
    // four consecutive outputs of a row a thread
    for (int i = threadIdx.x; i < n * (ROWS / 4); i += FEW_THREADS) {
        const int mm = i / (ROWS / 4), f = 4 * (i % (ROWS / 4));
        const int w = f / (MODE == SWIGLU ? 16 : 32), t = MODE == SWIGLU ? 0 : f / 16 % 2, c = f % 16;
        float4v v[2] = {};
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            v[0] += *reinterpret_cast<const float4v*>(&red[k][w][t][mm][c]);
            if (MODE == SWIGLU) v[1] += *reinterpret_cast<const float4v*>(&red[k][w][1][mm][c]);
        }
        const int col = sl * ROWS + f, left = n_eff - col;
        if (left <= 0) continue;
        if (MODE == SWIGLU)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[0][j] = silu_f(v[0][j]) * v[1][j];
        const size_t o = a.dense_c > 0 ? mm : jb->out[mm];
        store4(a.out, a.out_type, o * a.ldo + col, v[0], left, a.vec);
    }
}

// WK: as many wavefronts along K as there are steps, for the shortest chain and the most blocks; where each block quantizes the
// job's rows, half as many, for blocks of twice the rows.  In a graph, the weights in no cache: gate|up (2048 columns, 16 steps)
// with 8, 4, 2 along K: one token 9.7, 11.3, 16.3 us, 16 tokens (133 jobs) 57, 59, 64; down (512 columns, 4 steps) with 4, 2, 1:
// one token 7.2, 7.5, 10.2, 16 tokens 37, 34, 36; f16 experts of 2048 columns, 16 tokens, with 8, 4, 2: 108, 116, 123 (5.2 TB/s).
template <Elem EL, Mode MODE, bool QH> void launch_few(const Args& a, int njobs_cap, hipStream_t s) {
    const int steps = (a.n_in * ESZ<EL> + STEP - 1) / STEP, n_eff = MODE == SWIGLU ? a.n_out / 2 : a.n_out;
    const int per = MODE == SWIGLU ? 16 : 32;
    const size_t lds = QH ? 16 * (size_t) (steps * STEP + 16) + 16 * (size_t) blocks_of(a.n_in) * 4 : 0;
    auto go = [&](auto wk) {
        constexpr int WK = decltype(wk)::value;
        const int rows = per * (FEW_WAVES / WK);
        k_mm_few<EL, MODE, WK, QH><<<grid_of((n_eff + rows - 1) / rows, njobs_cap, FEW_THREADS), FEW_THREADS, lds, s>>>(a);
    };
    const int along = QH ? steps / 2 : steps;
    if (along >= 8) go(std::integral_constant<int, 8>{});
    else if (along >= 4) go(std::integral_constant<int, 4>{});
    else if (along >= 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
}

}  // namespace mm
}  // namespace sfnx
