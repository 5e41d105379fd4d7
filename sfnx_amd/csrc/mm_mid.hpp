// Dense products of some tens to some hundreds of rows: too many rows for the weights to be all there is, too few tiles of
// the large kind to fill the chip.  Bound by the latency of their loads: 128 rows of 4096 columns by a matrix of 256 rows 9.7 us
// (18.9 streamed), 256 by 1024 11.9 (19.3).
#pragma once

#include "mm_few.hpp"

namespace sfnx {
namespace mm {

constexpr int MID_WAVES = 8, MID_THREADS = MID_WAVES * WAVE;
template <int MT, int NT> constexpr int MID_PITCH = 16 * NT + 4;                                  // floats a row of a partial tile
template <int MT, int NT> constexpr int MID_LDS = MID_WAVES * 16 * MT * MID_PITCH<MT, NT> * 4;

// A block takes 16 MT rows of x times 16 NT rows of the matrix, its wavefronts the steps w, w + 8, ... of K: no wavefront waits
// for another before the sums meet in LDS, where they are added in wavefront order.  Both operands go straight to registers,
// a step ahead.
template <Elem EL, int MT, int NT> __global__ void __launch_bounds__(MID_THREADS, 2) k_mm_mid(Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const int nsl = (a.n_out + 16 * NT - 1) / (16 * NT), n0 = (int) (blockIdx.x % nsl) * 16 * NT, m0 = (int) (blockIdx.x / nsl) * 16 * MT;
    const uint8_t *xrow[MT], *wrow[NT];
    const float *xs[MT], *ws[NT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = min(m0 + 16 * j + r, a.dense_c - 1);
        xrow[j] = a.x + (size_t) m * rb;
        if constexpr (IS8<EL>) xs[j] = a.xs + (size_t) m * nb;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row0 = min(n0 + 16 * t, a.n_out - 1);
        wrow[t] = a.A + (size_t) min(row0 + r, a.n_out - 1) * rb;
        if constexpr (IS8<EL>) ws[t] = scales_of(a.A, a.n_out, a.n_in) + (size_t) (row0 / BLK) * nb;
    }
    struct Raw {
        Frag x[MT], w[NT];
        float xs[MT], ws[NT];
    };
    auto load = [&](Raw& f, int s) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f.w[t] = load_frag(wrow[t], s * STEP, q, rb);
            if constexpr (IS8<EL>) f.ws[t] = ws[t][s];
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            f.x[j] = load_frag(xrow[j], s * STEP, q, rb);
            if constexpr (IS8<EL>) f.xs[j] = xs[j][s];
        }
    };
    float4v acc[NT][MT] = {};
    Raw f, g;
    if (wave < steps) load(f, wave);
    for (int s = wave; s < steps; s += MID_WAVES) {
        if (s + MID_WAVES < steps) load(g, s + MID_WAVES);
        Operand<EL> x[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) x[j] = operand<EL>(f.x[j]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const Operand<EL> w = operand<EL>(f.w[t]);
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[t][j] = step_mma<EL>(w, x[j], acc[t][j], IS8<EL> ? f.xs[j] * f.ws[t] : 1.f);
        }
        f = g;
    }
    constexpr int P = MID_PITCH<MT, NT>, W = 16 * MT * P;
    float* red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) *reinterpret_cast<float4v*>(red + wave * W + (16 * j + r) * P + 16 * t + 4 * q) = acc[t][j];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * MT * 4 * NT; i += MID_THREADS) {
        const int m = i / (4 * NT), c = 4 * (i % (4 * NT));
        if (m0 + m >= a.dense_c || n0 + c >= a.n_out) continue;
        float4v v = {};
#pragma unroll
        for (int w = 0; w < MID_WAVES; ++w) v += *reinterpret_cast<const float4v*>(red + w * W + m * P + c);
        store4(a.out, a.out_type, (size_t) (m0 + m) * a.ldo + n0 + c, v, a.n_out - n0 - c, a.vec);
    }
}

template <Elem EL, int MT, int NT> void launch_mid(const Args& a, hipStream_t s) {
    const int nsl = (a.n_out + 16 * NT - 1) / (16 * NT), rows = (a.dense_c + 16 * MT - 1) / (16 * MT);
    k_mm_mid<EL, MT, NT><<<grid_of(nsl, rows, MID_THREADS), MID_THREADS, MID_LDS<MT, NT>, s>>>(a);
}

}  // namespace mm
}  // namespace sfnx
