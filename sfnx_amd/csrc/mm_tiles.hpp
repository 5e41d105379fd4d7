// Products of many rows: jobs of up to 64 rows (sfnx_bigjob), or the rows of a dense product.
//
// One workgroup a compute unit walks tiles of 256 weight rows (SWIGLU: 128 gate rows and their up rows) times either one job
// (stream_tiles: where the weights' way from HBM is the time) or up to four consecutive jobs of one expert, 256 rows
// (group_tiles: large dense products, and 16-bit experts of many rows, where the matrix cores are).  Both bring a K step of both
// operands and its scales into LDS by asynchronous copies: whole 128-byte lines, 8 rows a request; 16-byte piece p of row r at
// place p ^ (r % 8), so that the 16 lanes of a fragment's rows read different banks (no conflicts counted).
#pragma once

#include "mm.hpp"

namespace sfnx {
namespace mm {

constexpr int TW = 8, TT = TW * WAVE;        // wavefronts and threads
constexpr int BM1 = SFNX_PF_JOB, BN = 256;   // rows of a job and of a slice
constexpr int GJ = 4, BMG = GJ * BM1;        // jobs and rows of a group
constexpr int HP = BLK + 16;                 // row pitch of the quantized h on its way out

// a stage in LDS: N weight rows, M activation rows, their scales, a scale for each 16 weight rows (padded to a request)
template <int M, int N = BN> struct Stage {
    static constexpr int X = N * STEP, XS = X + M * STEP, WS = XS + M * 4, SIZE = WS + 256;
};
// streamed tiles: NT row tiles a wavefront, so slices of 128 NT rows; KS K steps a stage, so that a wavefront has as many matrix
// instructions between barriers with one tile as with two
constexpr int S1_SLOT = 768, S1_SLOTS = 4;   // a job's description
template <int NT> struct Stream {
    typedef Stage<BM1, 128 * NT> S;
    static constexpr int STAGES = 3, KS = NT == 2 ? 1 : 2, JOBS = STAGES * KS * S::SIZE, EPI = JOBS + (NT == 2 ? S1_SLOTS * S1_SLOT : 0);
    static constexpr int LDS = EPI + (NT == 2 ? TW * BM1 * 4 + BM1 * HP : 0);   // NT = 1: dense products, stored as they are
};
constexpr int S1_LDS = Stream<2>::LDS;
constexpr int SG_LIST = 2 * Stage<BMG>::SIZE, WINDOW = 8192;   // the groups of WINDOW jobs, as 16-bit job numbers
constexpr int T_LDS = SG_LIST + 2 * WINDOW + 64;   // and their number
static_assert(T_LDS <= 160 * 1024 && T_LDS >= S1_LDS && 4 * WINDOW <= SG_LIST, "LDS");

// Workgroup b runs on XCD b % 8: the slices of xg consecutive groups (an expert's jobs are consecutive) go to one XCD, so
// an expert's weights come from HBM once for them; xg = XG, or 1 where there are too few to use all XCDs evenly (single jobs, few
// of one expert, 2 for 4: down of 777 tokens 129 -> 124 us; groups 4 for 1: bf16 experts of 4096 tokens 307 -> 297).  A dense
// product of few groups leaves XCDs idle that way: where fewer rounds of the compute units come of it, an XCD takes every 8th
// slice of all groups (across; 128 rows, 4096 -> 8192: 41.8 -> 20.5 us).  false: no such group or slice
template <int XG> __device__ __forceinline__ bool tile_at(int b, int nsl, int n, bool across, int& sl, int& i) {
    const int p = across ? n : nsl, xg = n >= 64 ? XG : 1;
    const int x = b % XCDS, k = b / XCDS, m = k / p, u = k % p, v = xg * (XCDS * (m / xg) + x) + m % xg;
    sl = across ? v : u;
    i = across ? u : v;
    return v < (across ? nsl : n);
}
inline bool across_of(int nsl, int n) {
    const int64_t per = CUS / XCDS;   // an XCD's compute units
    return n < 64 && ((nsl + XCDS - 1) / XCDS * n + per - 1) / per < ((n + XCDS - 1) / XCDS * nsl + per - 1) / per;
}
__host__ __device__ __forceinline__ int64_t tiles_of(int nsl, int n, bool across) {
    return across ? (int64_t) (nsl + XCDS - 1) / XCDS * XCDS * n : (int64_t) nsl * ((n + 31) / 32) * 32;
}

// The weight row at place i of a slice.  STORE: the rows in order.  SWIGLU: of the NT2 tiles of 16 that a wavefront owns, the
// first half are gate tiles and the others their up tiles.
template <Mode MODE, int NT2, int N = BN> __device__ __forceinline__ int weight_row(const Args& a, int sl, int i) {
    const int n_eff = MODE == SWIGLU ? a.n_out / 2 : a.n_out;
    if (MODE == STORE) return min(sl * N + i, a.n_out - 1);
    const int w = i / (16 * NT2), u = i / 16 % NT2, nt = NT2 / 2;
    return min(sl * (BN / 2) + 16 * (nt * w + u % nt) + i % 16, n_eff - 1) + (u >= nt ? n_eff : 0);
}

__device__ __forceinline__ Frag lds_frag(const uint8_t* rows, int row, int q) {
    const uint8_t* p = rows + row * STEP;
    return Frag{*reinterpret_cast<const uint4*>(p + 16 * (q ^ (row & 7))), *reinterpret_cast<const uint4*>(p + 16 * ((q + 4) ^ (row & 7)))};
}

// h = silu(gate) up on the accumulators (gate tile, up tile) of a tile's n <= 64 rows, quantized: the tile's 128 columns, 16 a
// wavefront, are a scale block of h.  lds: scratch of all wavefronts.
template <typename Out> __device__ __forceinline__ void swiglu_out(const Args& a, float4v (&acc)[2][4], int sl, int wave, int n, uint8_t* lds, Out out_row) {
    const int lane = threadIdx.x % WAVE, r = lane % 16, q = lane / 16, ff = a.n_out / 2;
    const bool in = sl * BLK + 16 * wave < ff;     // FF is a multiple of 16
    uint32_t* mx = reinterpret_cast<uint32_t*>(lds);   // [TW][BM1]: the largest finite |h|, the top bit set where there are others
    uint8_t* hb = lds + TW * BM1 * 4;                  // [BM1][HP]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (16 * j >= n) continue;
        float am = 0.f;
        int odd = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[0][j][i] = in ? silu_f(acc[0][j][i]) * acc[1][j][i] : 0.f;
            am = fmaxf(am, finite_abs(acc[0][j][i]));
            odd |= abs_bits(acc[0][j][i]) >= 0x7f800000u;
        }
        am = fmaxf(am, lane_xor<16>(am));
        am = fmaxf(am, lane_xor<32>(am));
        odd |= lane_xor<16>(odd);
        odd |= lane_xor<32>(odd);
        if (q == 0) mx[wave * BM1 + 16 * j + r] = __float_as_uint(am) | (uint32_t) odd << 31;
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (16 * j >= n) continue;
        const int m = 16 * j + r;
        uint32_t top = 0, any = 0;   // of values that are not negative, the largest has the largest bits
#pragma unroll
        for (int w = 0; w < TW; ++w) {
            const uint32_t v = mx[w * BM1 + m];
            top = max(top, v & 0x7fffffffu);
            any |= v;
        }
        const F8Scale s = f8_scale(__uint_as_float(top), any < 0x80000000u);
        *reinterpret_cast<uint32_t*>(hb + m * HP + 16 * wave + 4 * q) = f8_pack4(acc[0][j][0], acc[0][j][1], acc[0][j][2], acc[0][j][3], s);
        if (wave == 0 && q == 0 && m < n) a.out_s[out_row(m) * blocks_of(ff) + sl] = s.s;
    }
    lds_barrier();
    const int m = threadIdx.x / 8, c = 16 * (threadIdx.x % 8);
    if (m < n && sl * BLK + c < ff)
        *reinterpret_cast<uint4*>((uint8_t*) a.out + out_row(m) * ff + sl * BLK + c) = *reinterpret_cast<const uint4*>(hb + m * HP + c);
}

// ------------------------------------------------------------------------------------------------ one job a tile
// The tiles are a stream of stages: while one is multiplied the next two are on their way into LDS, across the ends of tiles
// too.  The descriptions of later jobs come by asynchronous copies as well.  Two places still drain the stream: enter(), once a
// tile, where a table's entry is waited for after its branch (whether there is a table or not), and a tile's first wait, which
// counts the stores of the tile before it among the copies (down of five steps a tile: every fifth step).  A wavefront owns 32
// of the tile's weight rows for all of the job's rows.  Bound by memory where an expert has some tens of rows: gate|up of 2048
// tokens over 513 experts of 2048 x 1024, 1.07 GB of weights, 245 us, 4.4 TB/s (a copy of that size 4.9, reads into LDS alone
// 6.0); the matrix cores are 21% busy.  With hundreds of rows an expert by passing the weights through LDS and their conversion
// once for each 64 rows, and by converting the activations in every wavefront: 4096 tokens over 65 experts, 120 GFLOP, gate|up
// 187 us, down into bf16 108, into f32 131, the matrix cores 29% and 14% busy (gate|up, down into bf16).
template <Elem EL, Mode MODE, int NT> __device__ __forceinline__ void stream_tiles(const Args& a, int nj, const Lds& L) {
    uint8_t* const lds = L.p;
    constexpr int KS = Stream<NT>::KS, D = Stream<NT>::STAGES, N = 128 * NT;
    constexpr int REQ = KS * (2 * NT + 1);   // copies a wavefront issues for a stage, and KS of scales the first two wavefronts
    typedef typename Stream<NT>::S S;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, r8 = lane / 8, p8 = (lane % 8) ^ r8;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    const int nsl = (a.n_out + N - 1) / N, grid = (int) gridDim.x, tiles = (int) tiles_of(nsl, nj, IS8<EL> && MODE == STORE && a.across);
    const bool dense = a.dense_c > 0;
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs;

    auto next_tile = [&](int b, int& sl, int& ji) {   // the first tile of this workgroup from b on; its number, or -1
        for (; b < tiles; b += grid)
            if (tile_at<2>(b, nsl, nj, IS8<EL> && MODE == STORE && a.across, sl, ji)) return b;
        return -1;
    };
    auto slot_of = [&](int c) { return reinterpret_cast<const int*>(lds + Stream<NT>::JOBS + (c % S1_SLOTS) * S1_SLOT); };
    auto request_job = [&](int c, int ji) {   // the job's 130 words
        if (dense) return;
        const int* src = reinterpret_cast<const int*>(jobs + (nj - 1 - ji));   // the last job first: the shared expert's are the longest
#pragma unroll
        for (int i = 0; i < 3; ++i) copy4(src + min(64 * i + lane, 129), L.at(slot_of(c) + 64 * i));
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
    uint32_t woff[2 * NT];
    const float *xs_src, *ws_src;
    auto enter = [&]() {   // the pc-th tile's addresses; its job is in its slot
        const int n = job_rows(pc, pji), e = dense ? 0 : __builtin_amdgcn_readfirstlane(slot_of(pc)[0]);
        wbase = uniform_ptr(expert_at(a.A, a.sa, e));
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) woff[i] = (uint32_t) weight_row<MODE, NT, N>(a, psl, 16 * NT * wave + 8 * i + r8) * (uint32_t) rb + 16 * p8;
        xsrc = a.x + (size_t) act_row(pc, pji, n, 8 * wave + r8) * rb + 16 * p8;
        if constexpr (IS8<EL>) {
            xs_src = a.xs + (size_t) act_row(pc, pji, n, lane) * nb;
            ws_src = scales_of(wbase, a.n_out, a.n_in) + (size_t) (weight_row<MODE, NT, N>(a, psl, 16 * (r % (8 * NT))) / BLK) * nb;
        }
        nt = next_tile(pt + grid, nsl_, nji);
        if (nt >= 0) request_job(pc + 1, nji);
    };
    auto produce = [&](uint8_t* stage) {   // the next KS steps of the stream into a stage; false: there are none
        if (ps >= steps) {
            if (nt < 0) return false;
            if (steps <= KS) vm_wait<0>();   // the job was requested in the stage before this one; else an older wait covers it
            pt = nt, psl = nsl_, pji = nji, ps = 0, ++pc;
            enter();
        }
#pragma unroll
        for (int h = 0; h < KS; ++h) {
            const int s = min(ps + h, steps - 1), k = s * STEP;   // past the last step that again
            uint8_t* buf = stage + h * S::SIZE;
            const uint8_t* x = xsrc + k;
            if (k + STEP <= rb) {
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) copy16(uniform_ptr(wbase + k), woff[i], L.at(buf + (16 * NT * wave + 8 * i) * STEP));
            } else {   // zero past the rows' end
                const bool in = k + 16 * p8 < rb;
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i)
                    copy16(in ? wbase + k + woff[i] : (const uint8_t*) &ZERO16, L.at(buf + (16 * NT * wave + 8 * i) * STEP));
                if (!in) x = (const uint8_t*) &ZERO16;
            }
            copy16(x, L.at(buf + S::X + 8 * wave * STEP));
            if constexpr (IS8<EL>) {   // each copy touches a line a row: once a block (by every wavefront: gate|up of 2048 tokens 267 us for 263, 777 x 1301 x 2000 15.9 for 14.8)
                if (wave == 0) copy4(xs_src + s, L.at(buf + S::XS));
                if (wave == 1) copy4(ws_src + s, L.at(buf + S::WS));
            }
        }
        ps += KS;
        return true;
    };

    pt = next_tile((int) blockIdx.x, psl, pji);
    if (pt < 0) return;
    request_job(0, pji);
    vm_wait<0>();
    int ct = pt, csl = psl, cji = pji;   // the tile that is multiplied
    enter();
    int ahead = -1;   // how many stages after the one to be multiplied have been requested
#pragma unroll
    for (int i = 0; i < D - 1; ++i) ahead += produce(lds + i * KS * S::SIZE);
    int at = 0;       // the stage to be multiplied
    for (int c = 0; ct >= 0; ++c) {
        const int n = job_rows(c, cji);
        float4v acc[NT][4] = {};
        auto walk = [&](auto mt) {
            constexpr int MT = decltype(mt)::value;
            for (int s = 0; s < steps; s += KS) {
                if (ahead < D - 2) vm_wait<0>();
                else if (IS8<EL> && wave < 2) vm_wait<(REQ + KS) * (D - 2)>();
                else vm_wait<REQ * (D - 2)>();
                lds_barrier();   // every wavefront's copies of this stage landed, and every wavefront is past the one before
                const uint8_t* stage = lds + at * KS * S::SIZE;
                uint8_t* to = lds + (at == 0 ? D - 1 : at - 1) * KS * S::SIZE;
                at = at == D - 1 ? 0 : at + 1;
#pragma unroll
                for (int h = 0; h < KS; ++h) {
                    if (h > 0 && s + h >= steps) break;
                    const uint8_t* buf = stage + h * S::SIZE;
                    // the next stage's copies go out while the first reads come in
                    Frag w[NT], x[MT];
                    float ws[NT], xs[MT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        w[t] = lds_frag(buf, 16 * NT * wave + 16 * t + r, q);
                        ws[t] = IS8<EL> ? reinterpret_cast<const float*>(buf + S::WS)[NT * wave + t] : 1.f;
                    }
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        x[j] = lds_frag(buf + S::X, 16 * j + r, q);
                        xs[j] = IS8<EL> ? reinterpret_cast<const float*>(buf + S::XS)[16 * j + r] : 1.f;
                    }
                    if (h == 0) ahead += (int) produce(to) - 1;
                    Operand<EL> wo[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) wo[t] = operand<EL>(w[t]);
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        const Operand<EL> xo = operand<EL>(x[j]);
#pragma unroll
                        for (int t = 0; t < NT; ++t) acc[t][j] = step_mma<EL>(wo[t], xo, acc[t][j], xs[j] * ws[t]);
                    }
                }
            }
        };
        // the 16-row tiles that hold the job's rows
        if (n > 48) walk(std::integral_constant<int, 4>{});
        else if (n > 32) walk(std::integral_constant<int, 3>{});
        else if (n > 16) walk(std::integral_constant<int, 2>{});
        else walk(std::integral_constant<int, 1>{});

        const int* outs = slot_of(c) + 2 + SFNX_PF_JOB;
        auto out_row = [&](int m) { return (size_t) (dense ? BM1 * cji + m : outs[m]); };
        if constexpr (MODE == STORE) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = 16 * j + r;
                if (m >= n) continue;
                const size_t o = (size_t) out_row(m) * a.ldo;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int col = csl * N + 16 * NT * wave + 16 * t + 4 * q;
                    store4(a.out, a.out_type, o + col, acc[t][j], a.n_out - col, a.vec);
                }
            }
        } else {
            swiglu_out(a, acc, csl, wave, n, lds + Stream<NT>::EPI, out_row);
        }
        ct = next_tile(ct + grid, csl, cji);
    }
}

// ------------------------------------------------------------------------------------------------ a group of jobs a tile
// A wavefront owns a job's 64 rows and NT of the tile's 16 weight tiles: of a group of C jobs (3 are taken as 4), 8 / C wavefronts
// share a job.  4096 x 4096 x 4096 e4m3 into bf16 69 us, 2.0 PFLOP/s (72.5 with all wavefronts reading and multiplying at once);
// 4096 tokens over 65 bf16 experts of 2048 x 2048 282 us, 0.85 PFLOP/s (295); its 154 groups, 58 of them of one to three jobs, are
// 4.8 rounds of workgroups where full ones would be 3.5.  Of the 69 us, all of a step's copies but 10 us hide behind its
// products, and all of its fragments' reads but 20.
template <Elem EL, int C> __device__ __forceinline__ void group_tile(const Args& a, int sl, int j0, int count, const Lds& L) {
    uint8_t* const lds = L.p;
    constexpr int WN = TW / C, NT = 16 / WN;
    typedef Stage<BM1 * C> S;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, q = lane / 16, r8 = lane / 8, p8 = (lane % 8) ^ r8, wm = wave / WN, wn = wave % WN;
    const int rb = a.n_in * ESZ<EL>, steps = (rb + STEP - 1) / STEP, nb = blocks_of(a.n_in);
    constexpr bool dense = IS8<EL>;   // grouped are dense products in 8 bits and jobs in 16
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs + j0;
    // rows of the group's job i, its activation rows and output rows
    auto rows_of = [&](int i) {
        if (i >= count) return 0;
        return dense ? min(BM1, a.dense_c - BM1 * (j0 + i)) : max(0, min(jobs[i].n, BM1));
    };
    auto act_row = [&](int m) {
        const int n = rows_of(m / BM1);
        if (n == 0) return dense ? BM1 * j0 : 0;   // some row: a job that the group does not have
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
    const uint8_t* xsrc[C];
    uint32_t xs_off = 0, ws_off = 0;
    int wto[4];   // this wavefront's 8-row pieces of the weights: two of first, two of other tiles
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int h = 2 * wave + i % 2;
        wto[i] = 16 * NT * (h / NT) + 8 * NT * (i / 2) + 8 * (h % NT);
        if constexpr (!dense) woff[i] = (uint32_t) weight_row<STORE, NT>(a, sl, wto[i] + r8) * (uint32_t) rb;
    }
    if constexpr (!dense)
#pragma unroll
        for (int i = 0; i < C; ++i) xsrc[i] = a.x + (size_t) act_row(8 * (C * wave + i) + r8) * rb;
    const uint8_t *xs_base = nullptr, *ws_base = nullptr;
    if constexpr (IS8<EL>) {
        xs_base = uniform_ptr((const uint8_t*) (a.xs + (size_t) BM1 * j0 * nb));
        ws_base = uniform_ptr((const uint8_t*) scales_of(mat, a.n_out, a.n_in));
        xs_off = 4 * (uint32_t) (act_row(64 * wm + lane) - BM1 * j0) * (uint32_t) nb;
        ws_off = 4 * (uint32_t) (weight_row<STORE, NT>(a, sl, 16 * r) / BLK) * (uint32_t) nb;
    }
    // copy u (0 .. 3 weights, 4 .. 3 + C activations) of step s into a stage; past the rows' end their last piece (see below), past
    // the last step that again
    auto copy = [&](int u, int s, uint8_t* buf) {
        const uint32_t k = (uint32_t) min(min(s, steps - 1) * STEP + 16 * p8, rb - 16);
        const uint32_t to = L.at(buf + (u < 4 ? wto[u] * STEP : S::X + 8 * (C * wave + u - 4) * STEP));
        if constexpr (dense) {   // 8 consecutive rows (past the last that again): their addresses are cheaper made than kept
            const int end = u < 4 ? a.n_out : a.dense_c, first = min(u < 4 ? sl * BN + wto[u] : BM1 * j0 + 8 * (C * wave + u - 4), end - 1);
            copy16(uniform_ptr((u < 4 ? mat : a.x) + (size_t) first * rb), (uint32_t) __umul24(min(r8, end - 1 - first), rb) + k, to);
        } else if (u < 4) {
            copy16(mat, woff[u] + k, to);
        } else {
            copy16(xsrc[u - 4] + k, to);
        }
    };
    auto copy_scales = [&](int s, uint8_t* xs_to, uint8_t* ws_to) {
        const int k = 4 * min(s, steps - 1);
        if (EL == F8X || wn == 0) copy4(xs_base + k, xs_off, L.at(xs_to + 256 * wm));   // F8X: without branches, which would spill
        if (EL == F8X || wave == 1) copy4(ws_base + k, ws_off, L.at(ws_to));
    };
    auto clear = [&](int u, uint8_t* buf) {   // zero past the rows' end, whatever lies there: each wavefront in what it copied
        if ((steps - 1) * STEP + 16 * p8 >= rb)
            *reinterpret_cast<uint4*>(buf + (u < 4 ? wto[u] * STEP : S::X + 8 * (C * wave + u - 4) * STEP) + 16 * lane) = uint4{};
    };
    const bool tail = rb % STEP != 0;
    float4v acc[NT][4] = {};
    if constexpr (EL != F8X) {
        // The wavefronts of one half read fragments while those of the other, the second ones of their SIMDs, multiply, and the
        // other way about: a step is four turns (read x and the first weight tiles, multiply, read the others, multiply), and the
        // second half is a turn behind.  Copies into a place go out when both halves have read it, to be waited for four
        // turns later, before the first half reads them: those of x and the first tiles two steps ahead, the others one.
        // (Raised priority for the multiplying half: 72.5 us for 69.)
        constexpr int H = NT / 2, SLOT = BMG * 4 + 256;
        static_assert(!IS8<EL> || 4 * SLOT <= 2 * WINDOW, "the scales' places, where a list of groups would be");
        const bool behind = wave >= TW / 2;
        auto slot_of = [&](int s) { return lds + SG_LIST + (s & 3) * SLOT; };
        auto copy_first = [&](int s, uint8_t* buf) {
#pragma unroll
            for (int u = 0; u < 4 + C; ++u)
                if (u < 2 || u >= 4) copy(u, s, buf);
            if constexpr (IS8<EL>) copy_scales(s, slot_of(s), slot_of(s) + BMG * 4);
        };
        auto landed = [] { vm_wait<2 + C + 2>(); };   // all but this turn's copies and those of the reading turn before it
        auto clear_first = [&](uint8_t* buf) {
#pragma unroll
            for (int u = 0; u < 4 + C; ++u)
                if (u < 2 || u >= 4) clear(u, buf);
        };
        auto turn = [] {
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        Frag x[4], w[H];
        float xs[4], ws[H];
        auto read = [&](int s, const uint8_t* buf, int u0) {
#pragma unroll
            for (int u = 0; u < H; ++u) {
                w[u] = lds_frag(buf, 16 * NT * wn + 16 * (u0 + u) + r, q);
                if constexpr (IS8<EL>) ws[u] = reinterpret_cast<const float*>(slot_of(s) + BMG * 4)[NT * wn + u0 + u];
            }
        };
        auto multiply = [&](int u0) {
            if constexpr (IS8<EL>) {   // a product is scaled and added while the three after it are made
                float4v d[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = step_dot<EL>(w[0], x[j]);
#pragma unroll
                for (int u = 0; u < H; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        __builtin_amdgcn_sched_barrier(0);
                        acc[u0 + u][j] = scaled_add(d[j], xs[j] * ws[u], acc[u0 + u][j]);
                        if (u < H - 1) d[j] = step_dot<EL>(w[u + 1], x[j]);
                    }
            } else {
#pragma unroll
                for (int u = 0; u < H; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[u0 + u][j] = step_mma<EL>(w[u], x[j], acc[u0 + u][j], 1.f);
            }
            if constexpr (IS8<EL>)
#pragma unroll
                for (int u = 0; u < H; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(acc[u0 + u][j]));   // here, not sunk past the turn's end
        };
        lds_barrier();   // the tile before is done with LDS
        copy_first(0, lds);
        copy(2, 0, lds);
        copy(3, 0, lds);
        copy_first(1, lds + S::SIZE);
        landed();
        if (steps == 1 && tail) clear_first(lds);
        lds_barrier();
        if (behind) lds_barrier();
        for (int s = 0; s < steps; ++s) {
            uint8_t* buf = lds + (s & 1) * S::SIZE;
            uint8_t* to = lds + ((s + 1) & 1) * S::SIZE;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = lds_frag(buf + S::X, 64 * wm + 16 * j + r, q);
                if constexpr (IS8<EL>) xs[j] = reinterpret_cast<const float*>(slot_of(s))[64 * wm + 16 * j + r];
            }
            read(s, buf, 0);
            copy(2, s + 1, to);
            copy(3, s + 1, to);
            landed();
            if (s == steps - 1 && tail) clear(2, buf), clear(3, buf);
            turn();
            multiply(0);
            turn();
            read(s, buf, H);
            copy_first(s + 2, buf);
            landed();
            if (s == steps - 2 && tail) clear_first(to);
            turn();
            multiply(H);
            turn();
        }
    } else {
        // one step ahead, spread over the step's first half; converted, 64 activation rows are too many registers beside the sums:
        // half of them at a time
        auto fence = [] { asm volatile("" ::: "memory"); };   // LDS reads stay where they are: all at once they would not fit the registers
        lds_barrier();   // the tile before is done with LDS
#pragma unroll
        for (int u = 0; u < 4 + C; ++u) copy(u, 0, lds);
        copy_scales(0, lds + S::XS, lds + S::WS);
        for (int s = 0; s < steps; ++s) {
            uint8_t* buf = lds + (s & 1) * S::SIZE;
            uint8_t* to = lds + ((s + 1) & 1) * S::SIZE;
            vm_wait<0>();
            if (s == steps - 1 && tail)
#pragma unroll
                for (int u = 0; u < 4 + C; ++u) clear(u, buf);
            lds_barrier();   // every wavefront's copies of this stage landed, and every wavefront is past the one before
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
                for (int u = 0; u < NT; ++u) {
                    const FragX w = operand<EL>(lds_frag(buf, 16 * NT * wn + 16 * u + r, q));
                    const float ws = reinterpret_cast<const float*>(buf + S::WS)[NT * wn + u];
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[u][2 * h + j] = step_mma<EL>(w, x[j], acc[u][2 * h + j], xs[j] * ws);
                    if (h == 0)
#pragma unroll
                        for (int i = u * (4 + C) / NT; i < (u + 1) * (4 + C) / NT; ++i) copy(i, s + 1, to);
                    if (h == 0 && u == NT - 1) copy_scales(s + 1, to + S::XS, to + S::WS);
                    fence();
                }
            }
        }
    }
    vm_wait<0>();   // the copies past the end
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int m = 16 * j + r;
        if (m >= n) continue;
        const size_t o = (size_t) out_row(64 * wm + m) * a.ldo;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const int col = sl * BN + 16 * NT * wn + 16 * u + 4 * q;
            store4(a.out, a.out_type, o + col, acc[u][j], a.n_out - col, a.vec);
        }
    }
    if (EL != F8X && wave < TW / 2) lds_barrier();   // the turn the second half was behind
}

// The groups of the jobs [w0, w0 + count): the numbers (from w0) of the jobs that start one, in LDS; returns how many.
// A group is up to GJ consecutive jobs of one expert.
__device__ __forceinline__ int list_groups(const sfnx_bigjob* jobs, int w0, int count, uint8_t* lds) {
    int* w = reinterpret_cast<int*>(lds);                                   // the jobs' experts, where the stages come later
    uint16_t* list = reinterpret_cast<uint16_t*>(lds + SG_LIST);
    int* total = reinterpret_cast<int*>(lds + SG_LIST + 2 * WINDOW);
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

// the tiles of the groups in list (or of a dense product's jobs [0, count), every GJ)
template <Elem EL> __device__ __forceinline__ void group_tiles(const Args& a, int w0, int count, int n, const uint16_t* list, const Lds& L) {
    const bool across = IS8<EL> && a.across;
    const int tiles = (int) tiles_of(a.slices, n, across);
    for (int b = blockIdx.x; b < tiles; b += gridDim.x) {
        int sl, i;
        if (!tile_at<4>(b, a.slices, n, across, sl, i)) continue;
        i = n - 1 - i;   // the last group first: the shared expert's
        const int j0 = list ? list[i] : GJ * i, j1 = list ? (i + 1 < n ? list[i + 1] : count) : min(j0 + GJ, count);
        if (j1 - j0 > 2) group_tile<EL, 4>(a, sl, w0 + j0, j1 - j0, L);
        else if (j1 - j0 == 2) group_tile<EL, 2>(a, sl, w0 + j0, 2, L);
        else group_tile<EL, 1>(a, sl, w0 + j0, 1, L);
    }
}

// ------------------------------------------------------------------------------------------------ kernels
template <Elem EL, Mode MODE, int NT> __global__ void __launch_bounds__(TT, 2) k_mm_stream(Args a, int cap) {
    extern __shared__ __align__(16) uint8_t lds[];
    stream_tiles<EL, MODE, NT>(a, a.dense_c > 0 ? cap : min(*a.njobs, cap), lds_of(lds));
}

template <Elem EL> __global__ void __launch_bounds__(TT, 2) k_mm_group(Args a, int jobs) {
    extern __shared__ __align__(16) uint8_t lds[];
    group_tiles<EL>(a, 0, jobs, (jobs + GJ - 1) / GJ, nullptr, lds_of(lds));
}

// 16-bit experts: groups where their rounds of workgroups, each of which takes twice a round of single jobs, are fewer than half
// of those; which the jobs themselves say.  Streamed and grouped (us; 2048 columns, 1024 rows, bf16, tokens / experts / top k):
// 600 / 8 / 2 27 and 48; 1024 / 64 / 6 96 and 99; 2048 / 64 / 6 130 and 125; 4096 / 64 / 6 215 and 169; 4096 / 128 / 8 276 and 206.
// The 8-bit products of experts are streamed: grouped, their steps' scales and conversions keep the matrix cores waiting (gate|up
// of 1024 / 64 / 6 streamed 79 us, grouped 150, of 4096 / 64 / 6 201 and 230).  Only down into 16 bits, whose sums are the matrix
// instruction's own, gained from groups at 400 rows an expert (2048 rows, 1024 columns: 4096 / 64 / 6 159 us streamed, 144 grouped;
// 512 columns 109 and 110).
template <Elem EL> __global__ void __launch_bounds__(TT, 2) k_mm_experts(Args a, int cap) {
    extern __shared__ __align__(16) uint8_t lds[];
    const Lds L = lds_of(lds);
    const int nj = min(*a.njobs, cap);
    const sfnx_bigjob* jobs = (const sfnx_bigjob*) a.jobs;
    auto rounds = [&](int n) { return ((int64_t) n * a.slices + CUS - 1) / CUS; };
    bool group = false;
    for (int w0 = 0; w0 < nj; w0 += WINDOW) {
        const int count = min(WINDOW, nj - w0);
        const int n = list_groups(jobs, w0, count, lds);
        if (!group && 2 * rounds(n) >= rounds(count)) break;
        group = true;
        group_tiles<EL>(a, w0, count, n, reinterpret_cast<const uint16_t*>(lds + SG_LIST), L);
    }
    if (!group) stream_tiles<EL, STORE, 2>(a, nj, L);
}

inline unsigned tile_grid(int slices, int jobs, bool across) {
    const int64_t tiles = tiles_of(slices, jobs, across);
    require(tiles < (1 << 30), "too many jobs for one launch");
    return (unsigned) std::min<int64_t>(tiles, CUS);
}
template <Elem EL, Mode MODE, int NT = 2> void launch_stream(Args a, int jobs, hipStream_t s) {
    const int slices = (a.n_out + 128 * NT - 1) / (128 * NT);
    a.across = a.dense_c > 0 && across_of(slices, jobs);
    k_mm_stream<EL, MODE, NT><<<tile_grid(slices, jobs, a.across), TT, Stream<NT>::LDS, s>>>(a, jobs);
}
template <Elem EL> void launch_group(Args a, int jobs, hipStream_t s) {
    const int groups = (jobs + GJ - 1) / GJ;
    a.slices = (a.n_out + BN - 1) / BN;
    a.across = across_of(a.slices, groups);
    k_mm_group<EL><<<tile_grid(a.slices, groups, a.across), TT, T_LDS, s>>>(a, jobs);
}
template <Elem EL> void launch_experts(Args a, int njobs_cap, hipStream_t s) {
    a.slices = (a.n_out + BN - 1) / BN;
    k_mm_experts<EL><<<tile_grid(a.slices, njobs_cap, false), TT, T_LDS, s>>>(a, njobs_cap);
}

}  // namespace mm
}  // namespace sfnx
