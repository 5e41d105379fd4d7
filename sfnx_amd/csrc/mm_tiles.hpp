// Products of many rows: jobs of up to 64 rows (sfnx_bigjob), or the rows of a dense product.
//
// One workgroup a compute unit walks tiles of 256 weight rows (SWIGLU: 128 gate rows and their up rows) times either one job
// (stream_tiles: where the weights' way from HBM is the time) or up to four consecutive jobs of one expert, 256 rows
// (group_tiles: where experts have many rows and the matrix cores are).  Both bring a K step of both operands and its scales
// into LDS by asynchronous copies: whole 128-byte lines, 8 rows a request; 16-byte piece p of row r at place p ^ (r % 8), so
// that the 16 lanes of a fragment's rows read different banks.
#pragma once

#include "mm.hpp"

namespace sfnx {
namespace mm {

constexpr int TW = 8, TT = TW * WAVE;        // wavefronts and threads
constexpr int BM1 = SFNX_PF_JOB, BN = 256;   // rows of a job and of a slice
constexpr int GJ = 4, BMG = GJ * BM1;        // jobs and rows of a group
constexpr int HP = BLK + 16;                 // row pitch of the quantized h on its way out

// a stage in LDS: BN weight rows, M activation rows, their scales, a scale for each 16 weight rows (padded to a request)
template <int M> struct Stage {
    static constexpr int X = BN * STEP, XS = X + M * STEP, WS = XS + M * 4, SIZE = WS + 256;
};
constexpr int S1_STAGES = 3, S1_SLOT = 768, S1_SLOTS = 4;   // S1_SLOT: a job's description
constexpr int S1_JOBS = S1_STAGES * Stage<BM1>::SIZE, S1_EPI = S1_JOBS + S1_SLOTS * S1_SLOT;
constexpr int S1_LDS = S1_EPI + TW * BM1 * 4 + BM1 * HP;
constexpr int SG_LIST = 2 * Stage<BMG>::SIZE, WINDOW = 8192;   // the groups of WINDOW jobs, as 16-bit job numbers
constexpr int T_LDS = SG_LIST + 2 * WINDOW > S1_LDS ? SG_LIST + 2 * WINDOW : S1_LDS;
static_assert(T_LDS + 64 <= 160 * 1024 && 4 * WINDOW <= SG_LIST && 2 * BMG * 4 + BMG * HP <= SG_LIST, "LDS");

// Workgroup b runs on XCD b % 8: the slices of xg consecutive groups (an expert's jobs are consecutive) go to one XCD, so
// an expert's weights come from HBM once for them; xg = 4, or 1 where there are too few to use all XCDs evenly.  false: no
// such group
__device__ __forceinline__ bool tile_at(int b, int nsl, int n, int& sl, int& i) {
    const int xg = n >= 64 ? 4 : 1;
    const int x = b % XCDS, k = b / XCDS, m = k / nsl;
    sl = k % nsl;
    i = xg * (XCDS * (m / xg) + x) + m % xg;
    return i < n;
}
__host__ __device__ __forceinline__ int64_t tiles_of(int nsl, int n) { return (int64_t) nsl * ((n + 31) / 32) * 32; }

// The place of a slice's weight row in LDS.  STORE: wavefronts' rows in order.  SWIGLU: of each W = 2 NT tiles of 16 that a
// wavefront owns, the first NT are gate tiles and the others their up tiles.
template <Mode MODE, int NT2> __device__ __forceinline__ int weight_row(const Args& a, int sl, int i) {
    const int n_eff = MODE == SWIGLU ? a.n_out / 2 : a.n_out;
    if (MODE == STORE) return min(sl * BN + i, a.n_out - 1);
    const int w = i / (16 * NT2), u = i / 16 % NT2, nt = NT2 / 2;
    return min(sl * (BN / 2) + 16 * (nt * w + u % nt) + i % 16, n_eff - 1) + (u >= nt ? n_eff : 0);
}

__device__ __forceinline__ Frag lds_frag(const uint8_t* rows, int row, int q) {
    const uint8_t* p = rows + row * STEP;
    return Frag{*reinterpret_cast<const uint4*>(p + 16 * (q ^ (row & 7))), *reinterpret_cast<const uint4*>(p + 16 * ((q + 4) ^ (row & 7)))};
}

// h = silu(gate) up on the accumulators acc[u][j] (gate) and acc[NT + u][j] (up), quantized: the tile's 128 columns are a
// scale block of h.  WN wavefronts share a token's columns; lds: scratch of all wavefronts.
template <int WN, int NT, int MT, int M, typename Out>
__device__ __forceinline__ void swiglu_out(const Args& a, float4v (&acc)[2 * NT][MT], int sl, int wn, int m0, int n, int rows, uint8_t* lds, Out out_row) {
    const int lane = threadIdx.x % WAVE, r = lane % 16, q = lane / 16, n_eff = a.n_out / 2;
    float* mx = reinterpret_cast<float*>(lds);     // [WN][M]
    uint8_t* hb = lds + WN * M * 4;                // [M][HP]
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        if (16 * j >= n) continue;
        float am = 0.f;
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = sl * BLK + 16 * (NT * wn + u) < n_eff;   // FF is a multiple of 16
                acc[u][j][i] = in ? silu_f(acc[u][j][i]) * acc[NT + u][j][i] : 0.f;
                am = fmaxf(am, finite_abs(acc[u][j][i]));
            }
        am = fmaxf(am, lane_xor<16>(am));
        am = fmaxf(am, lane_xor<32>(am));
        if (q == 0) mx[wn * M + m0 + 16 * j + r] = am;
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        if (16 * j >= n) continue;
        const int m = 16 * j + r;
        float am = 0.f;
#pragma unroll
        for (int w = 0; w < WN; ++w) am = fmaxf(am, mx[w * M + m0 + m]);
        const float s = f8_scale(am);
#pragma unroll
        for (int u = 0; u < NT; ++u)
            *reinterpret_cast<uint32_t*>(hb + (m0 + m) * HP + 16 * (NT * wn + u) + 4 * q) =
                f8_pack4(acc[u][j][0], acc[u][j][1], acc[u][j][2], acc[u][j][3], s);
        if (wn == 0 && q == 0 && m < n) a.out_s[out_row(m0 + m) * blocks_of(n_eff) + sl] = s;
    }
    lds_barrier();
    for (int i = threadIdx.x; i < M * 8; i += TT) {
        const int m = i / 8, c = 16 * (i % 8);
        if (m < rows && sl * BLK + c < n_eff) {
            const int64_t o = out_row(m);
            if (o >= 0) *reinterpret_cast<uint4*>((uint8_t*) a.out + (size_t) o * n_eff + sl * BLK + c) = *reinterpret_cast<const uint4*>(hb + m * HP + c);
        }
    }
}

// ------------------------------------------------------------------------------------------------ one job a tile
// The tiles are one unbroken stream of K steps: while a step is multiplied the next two are on their way into LDS, across
// the ends of tiles too, so no tile waits for its first weights.  The descriptions of later jobs come by asynchronous copies
// as well: a load the compiler waits for would drain the stream.  A wavefront owns 32 of the tile's weight rows for all of
// the job's rows.
template <Elem EL, Mode MODE> __device__ __forceinline__ void stream_tiles(const Args& a, int nj, uint8_t* lds) {
    constexpr int REQ = 5 + (IS8<EL> ? 2 : 0);   // copies a wavefront issues for a step
    typedef Stage<BM1> S;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, r8 = lane / 8, p8 = (lane % 8) ^ r8;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const int nsl = a.slices, grid = (int) gridDim.x, tiles = (int) tiles_of(nsl, nj);
    const bool dense = a.dense_c > 0;
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs;

    auto next_tile = [&](int b, int& sl, int& ji) {   // the first tile of this workgroup from b on; its number, or -1
        for (; b < tiles; b += grid)
            if (tile_at(b, nsl, nj, sl, ji)) return b;
        return -1;
    };
    auto slot_of = [&](int c) { return reinterpret_cast<const int*>(lds + S1_JOBS + (c % S1_SLOTS) * S1_SLOT); };
    auto request_job = [&](int c, int ji) {   // the job's 130 words
        if (dense) return;
        const int* src = reinterpret_cast<const int*>(jobs + (nj - 1 - ji));   // the last job first: the shared expert's are the longest
#pragma unroll
        for (int i = 0; i < 3; ++i) lds_copy_async<4>(src + min(64 * i + lane, 129), slot_of(c) + 64 * i);
    };
    auto job_rows = [&](int c, int ji) {
        return __builtin_amdgcn_readfirstlane(dense ? min(BM1, a.dense_c - BM1 * ji) : min(slot_of(c)[1], BM1));
    };
    auto act_row = [&](int c, int ji, int n, int m) {
        if (n <= 0) return 0;
        m = min(m, n - 1);
        return dense ? BM1 * ji + m : slot_of(c)[2 + m];
    };

    // the producer: tile pt (its pc-th), whose step ps is requested next; nt, the tile after it, whose job is under way
    int pt, psl, pji, pc = 0, ps = 0, nt, nsl_ = 0, nji = 0;
    const uint8_t *wbase, *xsrc;
    uint32_t woff[4];
    const float *xs_src, *ws_src;
    auto enter = [&]() {   // the pc-th tile's addresses; its job is in its slot
        const int n = job_rows(pc, pji), e = dense ? 0 : __builtin_amdgcn_readfirstlane(slot_of(pc)[0]);
        wbase = uniform_ptr(expert_at(a.A, a.sa, e));
#pragma unroll
        for (int i = 0; i < 4; ++i) woff[i] = (uint32_t) weight_row<MODE, 2>(a, psl, 32 * wave + 8 * i + r8) * (uint32_t) rb + 16 * p8;
        xsrc = a.x + (size_t) act_row(pc, pji, n, 8 * wave + r8) * rb + 16 * p8;
        if constexpr (IS8<EL>) {
            xs_src = a.xs + (size_t) act_row(pc, pji, n, lane) * nb;
            ws_src = scales_of(wbase, a.n_out, a.n_in) + (size_t) (weight_row<MODE, 2>(a, psl, 16 * r) / BLK) * nb;
        }
        nt = next_tile(pt + grid, nsl_, nji);
        if (nt >= 0) request_job(pc + 1, nji);
    };
    auto produce = [&](uint8_t* buf) {   // the next step of the stream into a stage; false: there is none
        if (ps == steps) {
            if (nt < 0) return false;
            if (steps < 2) vm_wait<0>();   // the job was requested in the step before this one; else an older wait covers it
            pt = nt, psl = nsl_, pji = nji, ps = 0, ++pc;
            enter();
        }
        const int k = ps * STEP;
        const uint8_t* x = xsrc + k;
        if (k + STEP <= rb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) copy16(uniform_ptr(wbase + k), woff[i], buf + (32 * wave + 8 * i) * STEP);
        } else {   // zero past the rows' end
            const bool in = k + 16 * p8 < rb;
#pragma unroll
            for (int i = 0; i < 4; ++i) copy16(in ? wbase + k + woff[i] : (const uint8_t*) &ZERO16, buf + (32 * wave + 8 * i) * STEP);
            if (!in) x = (const uint8_t*) &ZERO16;
        }
        copy16(x, buf + S::X + 8 * wave * STEP);
        if constexpr (IS8<EL>) {   // every wavefront copies them all: the same values, and each counts the same requests
            copy4(xs_src + ps, buf + S::XS);
            copy4(ws_src + ps, buf + S::WS);
        }
        ++ps;
        return true;
    };

    pt = next_tile((int) blockIdx.x, psl, pji);
    if (pt < 0) return;
    request_job(0, pji);
    vm_wait<0>();
    int ct = pt, csl = psl, cji = pji;   // the tile that is multiplied
    enter();
    produce(lds);
    bool ahead = produce(lds + S::SIZE);   // whether a stage after the one to be multiplied has been requested
    int at = 0;                            // the stage to be multiplied
    for (int c = 0; ct >= 0; ++c) {
        const int n = job_rows(c, cji);
        float4v acc[2][4] = {};
        auto walk = [&](auto mt) {
            constexpr int MT = decltype(mt)::value;
            for (int s = 0; s < steps; ++s) {
                if (ahead) vm_wait<REQ>();
                else vm_wait<0>();
                lds_barrier();   // every wavefront's copies of this stage landed, and every wavefront is past the one before
                const uint8_t* buf = lds + at * S::SIZE;
                ahead = produce(lds + (at == 0 ? 2 : at - 1) * S::SIZE);
                at = at == 2 ? 0 : at + 1;
                Operand<EL> w[2];
                float ws[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    w[t] = operand<EL>(lds_frag(buf, 32 * wave + 16 * t + r, q));
                    if constexpr (IS8<EL>) ws[t] = reinterpret_cast<const float*>(buf + S::WS)[2 * wave + t];
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const Operand<EL> x = operand<EL>(lds_frag(buf + S::X, 16 * j + r, q));
                    float xs = 1.f;
                    if constexpr (IS8<EL>) xs = reinterpret_cast<const float*>(buf + S::XS)[16 * j + r];
#pragma unroll
                    for (int t = 0; t < 2; ++t) acc[t][j] = step_mma<EL>(w[t], x, acc[t][j], IS8<EL> ? xs * ws[t] : 1.f);
                }
            }
        };
        // the 16-row tiles that hold the job's rows
        if (n > 48) walk(std::integral_constant<int, 4>{});
        else if (n > 32) walk(std::integral_constant<int, 3>{});
        else if (n > 16) walk(std::integral_constant<int, 2>{});
        else walk(std::integral_constant<int, 1>{});

        const int* outs = slot_of(c) + 2 + SFNX_PF_JOB;
        auto out_row = [&](int m) { return (int64_t) (dense ? BM1 * cji + m : outs[m]); };
        if constexpr (MODE == STORE) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = 16 * j + r;
                if (m >= n) continue;
                const size_t o = (size_t) out_row(m) * a.ldo;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int col = csl * BN + 32 * wave + 16 * t + 4 * q;
                    store4(a.out, a.out_type, o + col, acc[t][j], a.n_out - col, a.vec);
                }
            }
        } else {
            swiglu_out<TW, 1, 4, BM1>(a, acc, csl, wave, 0, n, n, lds + S1_EPI, out_row);
        }
        ct = next_tile(ct + grid, csl, cji);
    }
}

// ------------------------------------------------------------------------------------------------ a group of jobs a tile
// A wavefront owns a job's 64 rows (wavefronts 2 w and 2 w + 1 the w-th of the group) and 128 of the tile's weight rows.
template <Elem EL, Mode MODE> __device__ __forceinline__ void group_tile(const Args& a, int sl, int j0, int count, uint8_t* lds) {
    typedef Stage<BMG> S;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, r8 = lane / 8, p8 = (lane % 8) ^ r8, wm = wave / 2, wn = wave % 2;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const bool dense = a.dense_c > 0;
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs + j0;
    // rows of the group's job i, its activation rows and output rows
    auto rows_of = [&](int i) {
        if (i >= count) return 0;
        return dense ? min(BM1, a.dense_c - BM1 * (j0 + i)) : max(0, min(jobs[i].n, BM1));
    };
    auto act_row = [&](int m) {
        const int n = rows_of(m / BM1);
        if (n == 0) return 0;   // some row: a job that the group does not have
        const int mm = min(m % BM1, n - 1);
        return dense ? BM1 * (j0 + m / BM1) + mm : jobs[m / BM1].y[mm];
    };
    auto out_row = [&](int m) {
        if (m % BM1 >= rows_of(m / BM1)) return (int64_t) -1;
        return (int64_t) (dense ? BM1 * j0 + m : jobs[m / BM1].out[m % BM1]);
    };
    const uint8_t* mat = uniform_ptr(expert_at(a.A, a.sa, dense ? 0 : jobs[0].w));
    const int n = __builtin_amdgcn_readfirstlane(rows_of(wm));

    uint32_t woff[4];
    const uint8_t* xsrc[4];
    const float *xs_src = nullptr, *ws_src = nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        woff[i] = (uint32_t) weight_row<MODE, 8>(a, sl, 32 * wave + 8 * i + r8) * (uint32_t) rb;
        xsrc[i] = a.x + (size_t) act_row(32 * wave + 8 * i + r8) * rb;
    }
    if constexpr (IS8<EL>) {
        xs_src = a.xs + (size_t) act_row(64 * wm + lane) * nb;
        ws_src = scales_of(mat, a.n_out, a.n_in) + (size_t) (weight_row<MODE, 8>(a, sl, 16 * r) / BLK) * nb;
    }
    // the u-th eighth of step s into a stage; past the rows' end their last piece (see below), past the last step that again
    auto copy = [&](int u, int s, uint8_t* buf) {
        s = min(s, steps - 1);
        const uint32_t k = (uint32_t) min(s * STEP + 16 * p8, rb - 16);
        const int i = u % 4;
        if (u < 4) copy16(mat, woff[i] + k, buf + (32 * wave + 8 * i) * STEP);
        else copy16(xsrc[i] + k, buf + S::X + (32 * wave + 8 * i) * STEP);
        if constexpr (IS8<EL>) {
            if (u == 2) copy4(xs_src + s, buf + S::XS + 256 * wm);
            if (u == 3) copy4(ws_src + s, buf + S::WS);
        }
    };
    auto fence = [] { asm volatile("" ::: "memory"); };   // LDS reads stay where they are: all at once they would not fit the registers
    // what a wavefront copies of the next step beside its u-th weight tile (of 8): all of it in the first half of the step, so
    // that it is there at the step's end, but not at once
    auto ahead = [&](int u, int s, uint8_t* buf) {
        if (u < 4) {
            copy(2 * u, s, buf);
            copy(2 * u + 1, s, buf);
        }
        fence();
    };
    float4v acc[8][4] = {};
    lds_barrier();   // the tile before is done with LDS
#pragma unroll
    for (int u = 0; u < 8; ++u) copy(u, 0, lds);
    for (int s = 0; s < steps; ++s) {
        uint8_t* buf = lds + (s & 1) * S::SIZE;
        uint8_t* to = lds + ((s + 1) & 1) * S::SIZE;
        vm_wait<0>();
        if (s == steps - 1 && rb % STEP) {   // zero past the rows' end, whatever lies there: each wavefront in what it copied
            const int k = s * STEP + 16 * p8;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k >= rb) {
                    *reinterpret_cast<uint4*>(buf + (32 * wave + 8 * i) * STEP + 16 * lane) = uint4{};
                    *reinterpret_cast<uint4*>(buf + S::X + (32 * wave + 8 * i) * STEP + 16 * lane) = uint4{};
                }
        }
        lds_barrier();   // every wavefront's copies of this stage landed, and every wavefront is past the one before
        if constexpr (EL == F8) {
            // the products of a weight tile are added while the next tile's are made
            Frag x[4];
            float xs[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = lds_frag(buf + S::X, 64 * wm + 16 * j + r, q);
                xs[j] = reinterpret_cast<const float*>(buf + S::XS)[64 * wm + 16 * j + r];
            }
            Frag w = lds_frag(buf, 128 * wn + r, q);
            float ws = reinterpret_cast<const float*>(buf + S::WS)[8 * wn];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                float4v d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = step_dot<EL>(w, x[j]);
                const float sc = ws;
                if (u < 7) {
                    w = lds_frag(buf, 128 * wn + 16 * (u + 1) + r, q);
                    ws = reinterpret_cast<const float*>(buf + S::WS)[8 * wn + u + 1];
                }
                ahead(u, s + 1, to);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[u][j] = scaled_add(d[j], xs[j] * sc, acc[u][j]);
            }
        } else if constexpr (EL == F8X) {
            // converted, 64 activation rows are too many registers beside the sums: half of them at a time
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                FragX x[2];
                float xs[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[j] = operand<EL>(lds_frag(buf + S::X, 64 * wm + 32 * h + 16 * j + r, q));
                    xs[j] = reinterpret_cast<const float*>(buf + S::XS)[64 * wm + 32 * h + 16 * j + r];
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const FragX w = operand<EL>(lds_frag(buf, 128 * wn + 16 * u + r, q));
                    const float ws = reinterpret_cast<const float*>(buf + S::WS)[8 * wn + u];
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[u][2 * h + j] = step_mma<EL>(w, x[j], acc[u][2 * h + j], xs[j] * ws);
                    if (h == 0) copy(u, s + 1, to);
                    fence();
                }
            }
        } else {
            Frag x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = lds_frag(buf + S::X, 64 * wm + 16 * j + r, q);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const Frag w = lds_frag(buf, 128 * wn + 16 * u + r, q);
                ahead(u, s + 1, to);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[u][j] = step_mma<EL>(w, x[j], acc[u][j], 1.f);
            }
        }
    }
    vm_wait<0>();   // the copies past the end
    if constexpr (MODE == STORE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = 16 * j + r;
            if (m >= n) continue;
            const size_t o = (size_t) out_row(64 * wm + m) * a.ldo;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int col = sl * BN + 128 * wn + 16 * u + 4 * q;
                store4(a.out, a.out_type, o + col, acc[u][j], a.n_out - col, a.vec);
            }
        }
    } else {
        lds_barrier();   // the stages are free
        swiglu_out<2, 4, 4, BMG>(a, acc, sl, wn, 64 * wm, n, BMG, lds, out_row);
    }
}

// The groups of the jobs [w0, w0 + count): the numbers (from w0) of the jobs that start one, in LDS; returns how many.
// A group is up to GJ consecutive jobs of one expert.
__device__ __forceinline__ int list_groups(const sfnx_bigjob* jobs, int w0, int count, uint8_t* lds) {
    int* w = reinterpret_cast<int*>(lds);                                   // the jobs' experts, where the stages come later
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + SG_LIST);
    int* total = reinterpret_cast<int*>(lds + T_LDS);
    lds_barrier();
    for (int i = threadIdx.x; i < count; i += TT) w[i] = jobs[w0 + i].w;
    __syncthreads();
    if (threadIdx.x < WAVE) {
        const int lane = threadIdx.x;
        int start = 0, n = 0;   // where the run of the job before this chunk began
        for (int i0 = 0; i0 < count; i0 += WAVE) {
            const int i = i0 + lane;
            const bool first = i < count && (i == 0 || w[i] != w[i - 1]);
            const uint64_t m = __ballot(first), below = m & (~0ull >> (63 - lane));
            const int run = below ? i0 + 63 - __clzll((long long) below) : start;
            const bool lead = i < count && (i - run) % GJ == 0;
            const uint64_t l = __ballot(lead);
            if (lead) list[n + __popcll(l & ((1ull << lane) - 1))] = (uint16_t) i;
            n += __popcll(l);
            if (m) start = i0 + 63 - __clzll((long long) m);
        }
        if (lane == 0) *total = n;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*total);
}

// group: whether tiles are groups of jobs; 0 in a grouped product: they are where the jobs make less than half as many groups,
// which the jobs themselves say
template <Elem EL, Mode MODE> __global__ void __launch_bounds__(TT, 2) k_mm_tiles(Args a, int cap, int group) {
    extern __shared__ __align__(16) uint8_t lds[];
    const bool dense = a.dense_c > 0;
    const int nj = dense ? cap : min(*a.njobs, cap);
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs;
    for (int w0 = 0; w0 < nj; w0 += WINDOW) {
        const int count = min(WINDOW, nj - w0);
        const int n = dense ? (count + GJ - 1) / GJ : list_groups(jobs, w0, count, lds);
        if (!group && (dense || count < 2 * n)) break;
        group = 1;
        const uint16_t* list = reinterpret_cast<const uint16_t*>(lds + SG_LIST);
        const int tiles = (int) tiles_of(a.slices, n);
        for (int b = blockIdx.x; b < tiles; b += gridDim.x) {
            int sl, i;
            if (!tile_at(b, a.slices, n, sl, i)) continue;
            i = n - 1 - i;   // the last group first: the shared expert's
            const int j0 = dense ? GJ * i : list[i], j1 = dense ? min(j0 + GJ, count) : i + 1 < n ? list[i + 1] : count;
            group_tile<EL, MODE>(a, sl, w0 + j0, j1 - j0, lds);
        }
    }
    if (!group) stream_tiles<EL, MODE>(a, nj, lds);
}

template <Elem EL, Mode MODE> void launch_tiles(Args a, int njobs_cap, hipStream_t s) {
    require((uint64_t) a.n_out * a.n_in * ESZ<EL> < ((uint64_t) 1 << 32), "a matrix must be smaller than 4 GiB");
    a.slices = (a.n_out + BN - 1) / BN;
    const int64_t tiles = tiles_of(a.slices, njobs_cap);
    require(tiles < (1 << 30), "too many jobs for one launch");
    const int group = a.dense_c > 0 && (int64_t) a.slices * ((njobs_cap + GJ - 1) / GJ) >= CUS / 2;
    k_mm_tiles<EL, MODE><<<(unsigned) std::min<int64_t>(tiles, CUS), TT, T_LDS + 64, s>>>(a, njobs_cap, group);
}

}  // namespace mm
}  // namespace sfnx
