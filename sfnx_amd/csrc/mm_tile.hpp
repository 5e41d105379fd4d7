// Products of many rows: jobs of up to 64 rows (sfnx_bigjob), or the rows of a dense product 64 at a time.
#pragma once

#include "mm.hpp"

namespace sfnx {
namespace mm {

constexpr int TL_WAVES = 8, TL_THREADS = TL_WAVES * WAVE, TL_BM = 64, TL_BN = 256;
constexpr int TL_STAGE = (TL_BN + TL_BM) * STEP, TL_LDS = 2 * TL_STAGE;

// A block takes 256 weight rows (SWIGLU: 128 gate rows and their up rows) and a job's 64 activation rows.  A K step's rows
// come into LDS by asynchronous copies of whole 128-byte lines (8 rows a request), two buffers in turn; 16-byte piece p of
// row r lies at place p ^ (r % 8), so that the 16 lanes of a fragment's rows read different banks.  A wavefront owns 32 of
// the block's weight rows (SWIGLU: 16 gate rows and their up rows) for all of the job's rows.
template <Elem EL, Mode MODE, int MT>
__device__ __forceinline__ void tile_job(const Args& a, const uint8_t* mat, const int* ys, const int* outs, int y0, int n,
                                         int sl, uint8_t* lds) {
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, r8 = lane / 8, p8 = (lane % 8) ^ r8;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const int n_eff = MODE == SWIGLU ? a.n_out / 2 : a.n_out;
    auto act_row = [&](int m) { m = min(m, n - 1); return ys ? ys[m] : y0 + m; };
    // LDS row i of the weights: SWIGLU: wavefront w's rows 32 w .. 32 w + 15 are gate rows f0 + 16 w + ., the next 16 their up rows
    auto weight_row = [&](int i) {
        const int row = MODE == SWIGLU ? min(sl * (TL_BN / 2) + 16 * (i / 32) + i % 16, n_eff - 1) + (i / 16 % 2 ? n_eff : 0) : sl * TL_BN + i;
        return min(row, a.n_out - 1);
    };
    const uint8_t* wsrc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) wsrc[i] = mat + (size_t) weight_row(32 * wave + 8 * i + r8) * rb + 16 * p8;
    const uint8_t* xsrc = a.x + (size_t) act_row(8 * wave + r8) * rb + 16 * p8;
    auto request = [&](int s, uint8_t* buf) {
        const bool in = s * STEP + 16 * p8 < rb;
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_copy_async<16>(in ? wsrc[i] + s * STEP : (const uint8_t*) &ZERO16, buf + (32 * wave + 8 * i) * STEP);
        lds_copy_async<16>(in ? xsrc + s * STEP : (const uint8_t*) &ZERO16, buf + (TL_BN + 8 * wave) * STEP);
    };
    const float* xsp[MT];
    const float* wsp[2];
    if constexpr (IS8<EL>) {
#pragma unroll
        for (int j = 0; j < MT; ++j) xsp[j] = a.xs + (size_t) act_row(16 * j + r) * nb;
#pragma unroll
        for (int t = 0; t < 2; ++t) wsp[t] = scales_of(mat, a.n_out, a.n_in) + (size_t) (weight_row(32 * wave + 16 * t) / BLK) * nb;
    }
    float4v acc[2][MT] = {};
    request(0, lds);
    for (int s = 0; s < steps; ++s) {
        uint8_t* buf = lds + (s & 1) * TL_STAGE;
        float xs[MT], ws[2];
        if constexpr (IS8<EL>) {
#pragma unroll
            for (int j = 0; j < MT; ++j) xs[j] = xsp[j][s];
#pragma unroll
            for (int t = 0; t < 2; ++t) ws[t] = wsp[t][s];
        }
        vm_wait<0>();
        if constexpr (IS8<EL>)
#pragma unroll
            for (int j = 0; j < MT; ++j) asm volatile("" : "+v"(xs[j]));   // the compiler's wait for them here, not after the next requests
        lds_barrier();   // every wavefront's rows of step s landed, and every wavefront is past step s - 1
        if (s + 1 < steps) request(s + 1, lds + ((s + 1) & 1) * TL_STAGE);
        auto frag = [&](int row) {
            const uint8_t* b = buf + row * STEP;
            return Frag{*reinterpret_cast<const uint4*>(b + 16 * (q ^ (row & 7))), *reinterpret_cast<const uint4*>(b + 16 * ((q + 4) ^ (row & 7)))};
        };
        // e4m3 converted to f16 takes twice the registers: the wavefront's weights are kept, the activations come one tile at a time
        Operand<EL> w[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) w[t] = operand<EL>(frag(32 * wave + 16 * t + r));
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const Operand<EL> x = operand<EL>(frag(TL_BN + 16 * j + r));
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[t][j] = step_mma<EL>(w[t], x, acc[t][j], IS8<EL> ? xs[j] * ws[t] : 1.f);
        }
    }
    if constexpr (MODE == STORE) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int m = 16 * j + r;
            if (m >= n) continue;
            const size_t o = (size_t) (outs ? outs[m] : y0 + m) * a.ldo;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int col = sl * TL_BN + 32 * wave + 16 * t + 4 * q;
                store4(a.out, a.out_type, o + col, acc[t][j], a.n_out - col, a.vec);
            }
        }
    } else {
        // h = silu(gate) up on the accumulators; the block's 128 columns are a scale block of h
        const int f = 16 * wave + 4 * q;
        const bool in = sl * (TL_BN / 2) + 16 * wave < n_eff;   // FF is a multiple of 16
        lds_barrier();
        float* mx = reinterpret_cast<float*>(lds);               // [8 wavefronts][64 tokens]
        uint8_t* hb = lds + TL_WAVES * TL_BM * 4;                // [64][144] quantized
        constexpr int HP = BLK + 16;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            float am = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[0][j][i] = in ? silu_f(acc[0][j][i]) * acc[1][j][i] : 0.f;
                am = fmaxf(am, finite_abs(acc[0][j][i]));
            }
            am = fmaxf(am, lane_xor<16>(am));
            am = fmaxf(am, lane_xor<32>(am));
            if (q == 0) mx[wave * TL_BM + 16 * j + r] = am;
        }
        lds_barrier();
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int m = 16 * j + r;
            float am = 0.f;
#pragma unroll
            for (int w = 0; w < TL_WAVES; ++w) am = fmaxf(am, mx[w * TL_BM + m]);
            const float s = f8_scale(am);
            *reinterpret_cast<uint32_t*>(hb + m * HP + f) = f8_pack4(acc[0][j][0], acc[0][j][1], acc[0][j][2], acc[0][j][3], s);
            if (wave == 0 && q == 0 && m < n) a.out_s[(size_t) outs[m] * blocks_of(n_eff) + sl] = s;
        }
        lds_barrier();
        const int m = threadIdx.x / 8, c = 16 * (threadIdx.x % 8);
        if (m < n && sl * BLK + c < n_eff)
            *reinterpret_cast<uint4*>((uint8_t*) a.out + (size_t) outs[m] * n_eff + sl * BLK + c) = *reinterpret_cast<const uint4*>(hb + m * HP + c);
    }
}

template <Elem EL, Mode MODE>
__global__ void __launch_bounds__(TL_THREADS, 4) k_mm_tile(Args a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int nsl = (a.n_out + TL_BN - 1) / TL_BN;   // SWIGLU: n_out = 2 FF, 128 of FF a block
    const int sl = blockIdx.x % nsl, ji = blockIdx.x / nsl;
    const int* ys = nullptr;
    const int* outs = nullptr;
    int n, e = 0, y0 = 0;
    if (a.dense_c > 0) {
        y0 = TL_BM * ji;
        n = min(TL_BM, a.dense_c - y0);
    } else {
        if (ji >= *a.njobs) return;
        const sfnx_bigjob* jb = (const sfnx_bigjob*) a.jobs + ji;
        n = min(jb->n, TL_BM);
        e = jb->w;
        ys = jb->y;
        outs = jb->out;
    }
    if (n <= 0) return;
    const uint8_t* mat = expert_at(a.A, a.sa, e);
    if (n > 32) tile_job<EL, MODE, 4>(a, mat, ys, outs, y0, n, sl, lds);
    else if (n > 16) tile_job<EL, MODE, 2>(a, mat, ys, outs, y0, n, sl, lds);
    else tile_job<EL, MODE, 1>(a, mat, ys, outs, y0, n, sl, lds);
}

template <Elem EL, Mode MODE> void launch_tile(const Args& a, int njobs_cap, hipStream_t s) {
    const int nsl = (a.n_out + TL_BN - 1) / TL_BN;
    k_mm_tile<EL, MODE><<<grid_of(nsl, njobs_cap, TL_THREADS), TL_THREADS, TL_LDS, s>>>(a);
}

}  // namespace mm
}  // namespace sfnx
