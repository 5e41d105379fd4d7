// Low-rank adapters of many requests beside a shared projection: out = base + scale_a B_a (A_a x) for the rows of each job,
// whose adapter is a.
//
// s = A_a x is a product on the matrix cores (the adapter's rows are the A operand, the tokens the B operand).  Activations of the
// adapters' type are multiplied on 16x16x32, whose products are exact, those of 32 bits on v_mfma_f32_16x16x4_f32.  s stays in
// 32 bits, so that the one rounding is that of the output.  There are two forms:
//   one launch    a workgroup takes 16 rows of a job and a slice of the outputs; every slice computes s again.  For few rows, where
//                 a launch and the loads' latency are what counts.
//   two launches  the first takes a job's rows and a slice of the input columns, and writes its part of s to the workspace; the second
//                 a job's rows and a slice of the outputs.  Each byte of x, base and out goes once.
#include "mm.hpp"

namespace sfnx {
namespace {
using namespace mm;

constexpr int AD_ROWS = 16, AD_UNIT = 32;   // a tile's rows; columns of a unit of outputs

struct AdapterArgs {
    const uint8_t *A, *B;     // adapters' matrices [rank][n_in] and [n_out][rank], sa / sb bytes apart (0: tables of their pointers)
    size_t sa, sb;
    const float* scale;       // an adapter's factor, or null (1)
    int n, rank, n_in, n_out;
    const sfnx_bigjob* jobs;
    const int* njobs;
    const uint8_t* x;         // rows ldx bytes apart
    int64_t ldx;
    const void* base;         // null: zeros
    void* out;                // base's and out's rows ldo values apart
    int64_t ldo;
    int rows;                 // of x, base and out
    int slices, units;        // of the outputs: slices of `units` units
    int subs;                 // one launch: workgroups a slice of a job has, which take its tiles of 16 entries in turn
    float* part;              // two launches: parts of s, [parts][rows][rank rounded up to 16, 32, 64 or 128]
    int parts, steps;         // of `steps` steps of 128 input columns each
};

__device__ __forceinline__ float wide16(bool f16, uint32_t v) { return f16 ? h2f((uint16_t) v) : __uint_as_float(v << 16); }
template <Elem EL> __device__ __forceinline__ void widen8(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[2 * k] = wide16(EL == F16, w[k] & 0xffff);
        f[2 * k + 1] = wide16(EL == F16, w[k] >> 16);
    }
}

// eight consecutive values of a row of base or out, as they lie in memory; the addresses have their type's alignment, which is
// enough for wide accesses
template <int OT> struct Eight { uint4 v[OT == SFNX_F32 ? 2 : 1]; };
template <int OT> using OutBits = typename std::conditional<OT == SFNX_F32, uint32_t, uint16_t>::type;
template <int OT> __device__ __forceinline__ Eight<OT> load_eight(const void* p, int64_t i, int left) {
    constexpr bool O32 = OT == SFNX_F32;
    typedef OutBits<OT> T;
    const T* f = (const T*) p + i;
    Eight<OT> e{};
    if (left >= 8) {
        __builtin_memcpy(&e, __builtin_assume_aligned(f, sizeof(T)), 8 * sizeof(T));
        return e;
    }
    uint32_t w[8] = {};
#pragma unroll
    for (int k = 0; k < 7; ++k)
        if (k < left) w[k] = f[k];
    if constexpr (O32) e.v[0] = uint4{w[0], w[1], w[2], w[3]}, e.v[1] = uint4{w[4], w[5], w[6], w[7]};
    else e.v[0] = uint4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
    return e;
}
template <int OT> __device__ __forceinline__ void store_eight(void* p, int64_t i, int left, const Eight<OT>& e) {
    constexpr bool O32 = OT == SFNX_F32;
    typedef OutBits<OT> T;
    T* f = (T*) p + i;
    if (left >= 8) {
        __builtin_memcpy(__builtin_assume_aligned(f, sizeof(T)), &e, 8 * sizeof(T));
        return;
    }
    const uint4 a = e.v[0], b = e.v[O32 ? 1 : 0];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 7; ++k)
        if (k < left) f[k] = (T) (O32 ? w[k] : w[k / 2] >> 16 * (k & 1));
}
template <int OT> __device__ __forceinline__ void unpack(const Eight<OT>& e, float (&v)[8]) {
    if constexpr (OT == SFNX_F32) {
        const float4v a = __builtin_bit_cast(float4v, e.v[0]), b = __builtin_bit_cast(float4v, e.v[1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
    } else {
        widen8<OT == SFNX_F16 ? F16 : BF16>(e.v[0], v);
    }
}
template <int OT> __device__ __forceinline__ Eight<OT> pack(const float (&v)[8]) {
    Eight<OT> e;
    if constexpr (OT == SFNX_F32) {
        e.v[0] = __builtin_bit_cast(uint4, float4v{v[0], v[1], v[2], v[3]});
        e.v[1] = __builtin_bit_cast(uint4, float4v{v[4], v[5], v[6], v[7]});
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {   // two at once
            typedef float float2v __attribute__((ext_vector_type(2)));
            typedef typename std::conditional<OT == SFNX_F16, _Float16, __bf16>::type T;
            typedef T pair __attribute__((ext_vector_type(2)));
            w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{v[2 * k], v[2 * k + 1]}, pair));
        }
        e.v[0] = uint4{w[0], w[1], w[2], w[3]};
    }
    return e;
}
// one value of base or out
template <int OT> __device__ __forceinline__ float load_one(const void* p, int64_t i) {
    if constexpr (OT == SFNX_F32) return ((const float*) p)[i];
    else return wide16(OT == SFNX_F16, ((const uint16_t*) p)[i]);
}
template <int OT> __device__ __forceinline__ void store_one(void* p, int64_t i, float v) {
    if constexpr (OT == SFNX_F32) ((float*) p)[i] = v;
    else ((uint16_t*) p)[i] = (uint16_t) half_bits(OT, v);
}

// a row of a job, -1 where it is none of x's and out's
struct JobRow {
    int y, o;
};
__device__ __forceinline__ JobRow job_row(const sfnx_bigjob& job, int n, int m, int rows) {
    const int y = job.y[m], o = job.out[m];
    const bool ok = m < n && (unsigned) y < (unsigned) rows && (unsigned) o < (unsigned) rows;
    return JobRow{ok ? y : -1, ok ? o : -1};
}

// rows without an adapter: base's
template <int OT> __device__ __forceinline__ void copy_base(const AdapterArgs& a, int o, int c, int c1, int step) {
    if (a.base == a.out || o < 0) return;
#pragma unroll 1
    for (; c < c1; c += step)
        store_eight<OT>(a.out, o * a.ldo + c, c1 - c, a.base ? load_eight<OT>(a.base, o * a.ldo + c, c1 - c) : Eight<OT>{});
}

// ------------------------------------------------------------------------------------------------ A x
// Rows of columns go to LDS by asynchronous copies whose 64 lanes take whole pieces of rows, 16 bytes each (a fragment read straight from
// memory is 16 rows' 64 bytes, and rows a power of two apart are one channel).  Piece c of row m lies at place c ^ (m % 16), so that a
// fragment's 16 rows lie in different banks.
template <int ROW> __device__ __forceinline__ const uint8_t* lds_piece(const uint8_t* rows, int m, int c) { return rows + m * ROW + 16 * (c ^ (m & 15)); }
// rows of ROW bytes from m0 on, 1024 bytes of them: lane l's piece of what it copies
template <int ROW> __device__ __forceinline__ int lane_row(int m0, int lane) { return m0 + lane / (ROW / 16); }
template <int ROW> __device__ __forceinline__ int lane_piece(int m, int lane) { return lane % (ROW / 16) ^ (m & 15); }

// acc += w . x over 32 columns: 8 of an adapter's row and of x in each lane
template <Elem EL, bool X32> __device__ __forceinline__ float4v shrink_mma(const uint4& w, const uint4& xa, const uint4& xb, float4v acc) {
    if constexpr (X32) {
        float f[8];
        widen8<EL>(w, f);
        const float4v a = __builtin_bit_cast(float4v, xa), b = __builtin_bit_cast(float4v, xb);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], e < 4 ? a[e] : b[e - 4], acc, 0, 0, 0);
        return acc;
    } else if constexpr (EL == F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, w), __builtin_bit_cast(half8v, xa), acc, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, w), __builtin_bit_cast(bf8v, xa), acc, 0, 0, 0);
    }
}
__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// ------------------------------------------------------------------------------------------------ one launch
// For few rows and small ranks.  Bound by a chain of reads: the job, its rows of x and A, B's tail, a launch's start (1 row, rank 16, 2048 -> 1024, f32: 5.2 us; 16 rows of
// 16 adapters, 2048 -> 2048, bf16: 6.2).  Each wavefront copies its own chunks of columns and multiplies them, so that none waits for another
// before the sum; base and B are on their way meanwhile.  Loops stay rolled: a launch of few workgroups runs its code once, and fetching it is
// part of its time (f32 x, 16 ranks, 2048 columns, unrolled to one pass: 12.7 us a launch).
constexpr int AW_WAVES = 8, AW_THREADS = AW_WAVES * WAVE;
template <bool X32, int RT> struct Few {
    static constexpr int KC = X32 || RT == 2 ? 128 : 256;                     // columns of a chunk
    static constexpr int XROW = KC * (X32 ? 4 : 2), AROW = KC * 2;
    static constexpr int BYTES = AD_ROWS * XROW + 16 * RT * AROW;             // a wavefront's
    static constexpr int P = 16 * RT + 4;                                     // floats of a token's s in LDS
    static constexpr int LDS = AW_WAVES * BYTES;
    static_assert(AW_WAVES * AD_ROWS * P * 4 <= LDS && LDS <= 160 * 1024, "");
};

// a tile: the n rows (16 at most count) of lanes' jr, the outputs c0 .. c1 - 1
template <Elem EL, bool X32, int RT, int OT>
__device__ __forceinline__ void few_rows(const AdapterArgs& a, const Lds& L, const uint8_t* Aw, const uint8_t* Bw, float sc, JobRow jr, int n, int c0, int c1) {
    typedef Few<X32, RT> F;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), r = lane % 16, q = lane / 16, o = jr.o;
    uint8_t* const xl = L.p + wave * F::BYTES;
    uint8_t* const al = xl + AD_ROWS * F::XROW;
    // ---- a unit's base and B: a tile's row r is column u + 8 (r / 4) + 4 t + r % 4, so that lane l's results are the columns u + 8 q ..
    // u + 8 q + 7; of B's row lane l takes the 4 RT ranks from 4 RT q on
    struct Unit {
        Eight<OT> base;
        uint4 b[2];
    };
    const auto request = [&](int u) {
        Unit g{};
        if (u >= c1) return g;
        if (o >= 0 && a.base) g.base = load_eight<OT>(a.base, o * a.ldo + u + 8 * q, c1 - u - 8 * q);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = u + 8 * (r / 4) + 4 * t + r % 4;
            const uint8_t* b = Bw + 2 * ((size_t) c * a.rank + 4 * RT * q);
            if (c < c1 && 4 * RT * q < a.rank) {   // rank is a multiple of 8
                if constexpr (RT == 1) {
                    const uint2 h = *reinterpret_cast<const uint2*>(b);
                    g.b[t] = uint4{h.x, h.y, 0, 0};
                } else {
                    g.b[t] = *reinterpret_cast<const uint4*>(b);
                }
            }
        }
        return g;
    };
    int u = c0 + wave * AD_UNIT;
    Unit g = request(u);
    // ---- s = A x
    float4v acc[RT] = {};
    for (int k0 = wave * F::KC; k0 < a.n_in; k0 += AW_WAVES * F::KC) {
        const int last = min(a.n_in - k0, F::KC);   // columns of the chunk
#pragma unroll 1
        for (int m = 0; m < min(n, AD_ROWS); m += 1024 / F::XROW) {
            const int row = lane_row<F::XROW>(m, lane), c = lane_piece<F::XROW>(row, lane);
            const int y = __shfl(jr.y, row);
            const bool in = y >= 0 && c * (X32 ? 4 : 8) < last;
            copy16(in ? a.x + (int64_t) y * a.ldx + (size_t) k0 * (X32 ? 4 : 2) + 16 * c : (const uint8_t*) &ZERO16, L.at(xl + m * F::XROW));
        }
        constexpr int AT = 1024 / F::AROW;   // rows of a copy; a row's place among 16 repeats every 16 / AT copies
#pragma unroll 1
        for (int m = 0; m < a.rank; m += 8) {   // rank is a multiple of 8
#pragma unroll
            for (int h = 0; h < 8; h += AT) {
                const int row = lane_row<F::AROW>(m + h, lane), c = lane_piece<F::AROW>(row, lane);
                copy16(8 * c < last ? Aw + 2 * ((size_t) row * a.n_in + k0) + 16 * c : (const uint8_t*) &ZERO16, L.at(al + (m + h) * F::AROW));
            }
        }
        vm_wait<0>();
        if (X32 && n == 1) {   // one row of 32-bit values: lane l its products with row r of A, a quarter of them
#pragma unroll 1
            for (int c = q; 8 * (c - q) < last; c += 4) {
                const float4v xa = __builtin_bit_cast(float4v, lds16(lds_piece<F::XROW>(xl, 0, 2 * c))), xb = __builtin_bit_cast(float4v, lds16(lds_piece<F::XROW>(xl, 0, 2 * c + 1)));
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float f[8];
                    widen8<EL>(lds16(lds_piece<F::AROW>(al, 16 * t + r, c)), f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[t][e % 4] = fmaf(f[e], e < 4 ? xa[e] : xb[e - 4], acc[t][e % 4]);
                }
            }
        } else
#pragma unroll 1
        for (int c = q; 8 * (c - q) < last; c += 4) {   // 32 columns; of rows beyond n and the rank LDS holds anything
            const uint4 xa = lds16(lds_piece<F::XROW>(xl, r, X32 ? 2 * c : c)), xb = X32 ? lds16(lds_piece<F::XROW>(xl, r, 2 * c + 1)) : xa;
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t] = shrink_mma<EL, X32>(lds16(lds_piece<F::AROW>(al, 16 * t + r, c)), xa, xb, acc[t]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the chunk is read before the next overwrites it
    }
    __syncthreads();   // all chunks are read
    float* const part = reinterpret_cast<float*>(L.p);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (X32 && n == 1) {
            float v = (acc[t][0] + acc[t][1]) + (acc[t][2] + acc[t][3]);
            v += lane_xor<16>(v);
            v += lane_xor<32>(v);
            if (q == 0) part[wave * AD_ROWS * F::P + 16 * t + r] = v;
        } else {
            *reinterpret_cast<float4v*>(part + (wave * AD_ROWS + r) * F::P + 16 * t + 4 * q) = acc[t];
        }
    }
    __syncthreads();
    float4v s[RT] = {};
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
        for (int p = 0; p < AW_WAVES; ++p) s[i] += *reinterpret_cast<const float4v*>(part + (p * AD_ROWS + r) * F::P + 4 * RT * q + 4 * i);
        s[i] = 4 * RT * q + 4 * i < a.rank ? s[i] * sc : float4v{};
    }
#pragma unroll 1
    for (; u < c1; u += AW_WAVES * AD_UNIT) {
        float v[8];
        unpack<OT>(g.base, v);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float4v d = {v[4 * t], v[4 * t + 1], v[4 * t + 2], v[4 * t + 3]};
            float f[8];
            widen8<EL>(g.b[t], f);
#pragma unroll
            for (int e = 0; e < 4 * RT; ++e) d = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], s[e / 4][e % 4], d, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * t + i] = d[i];
        }
        if (o >= 0) store_eight<OT>(a.out, o * a.ldo + u + 8 * q, c1 - u - 8 * q, pack<OT>(v));
        g = request(u + AW_WAVES * AD_UNIT);
    }
}

template <Elem EL, bool X32, int RT, int OT>
__global__ void __launch_bounds__(AW_THREADS) k_adapter_mm(const AdapterArgs a) {
    extern __shared__ __align__(16) uint8_t lds_[];
    const Lds L = lds_of(lds_);
    const int slice = blockIdx.x % a.slices, tile = blockIdx.x / a.slices, j = tile / a.subs, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = threadIdx.x % 16, q = threadIdx.x % WAVE / 16;
    int m0 = tile % a.subs * AD_ROWS;
    // all of the job at once: the list holds njobs_cap of them
    const sfnx_bigjob& job = a.jobs[j];
    const int nj = *a.njobs, n = min(job.n, SFNX_PF_JOB), w = job.w;
    JobRow jr = job_row(job, n, m0 + r, a.rows);
    if (j >= nj || n <= m0) return;
    const int c0 = slice * a.units * AD_UNIT, c1 = min(a.n_out, c0 + a.units * AD_UNIT);
    const bool some = (unsigned) w < (unsigned) a.n;
    const uint8_t *Aw = some ? expert_at(a.A, a.sa, w) : nullptr, *Bw = some ? expert_at(a.B, a.sb, w) : nullptr;
    const float sc = some && a.scale ? a.scale[w] : 1.f;
    // one tile, but of a job with more entries than x has rows, some of which are none of its rows
#pragma unroll 1
    for (;;) {
        if (some) few_rows<EL, X32, RT, OT>(a, L, Aw, Bw, sc, jr, n - m0, c0, c1);
        else copy_base<OT>(a, jr.o, c0 + wave * AD_UNIT + 8 * q, c1, AW_WAVES * AD_UNIT);
        m0 += a.subs * AD_ROWS;
        if (m0 >= n) return;
        __syncthreads();   // the tile's s is read
        jr = job_row(job, n, m0 + r, a.rows);
    }
}

// ------------------------------------------------------------------------------------------------ two launches
// The first: a workgroup takes a job's rows and a part of the input columns, 128 columns a stage, stages in flight while one is multiplied;
// each wavefront takes 32 of a stage's columns, all rows and all ranks.  Bound by what a compute unit takes in, x and A for each 64 rows again: 4096
// rows, rank 64, 4096 columns, bf16, 34 MB of x and as much of A out of the L2, 14.5 us.
constexpr int A2_WAVES = 4, A2_THREADS = A2_WAVES * WAVE, A2_TILES = SFNX_PF_JOB / AD_ROWS, A2_KC = 128;
template <bool X32, int RT> struct Many {
    static constexpr int XROW = A2_KC * (X32 ? 4 : 2), AROW = A2_KC * 2;
    static constexpr int STAGE = SFNX_PF_JOB * XROW + 16 * RT * AROW;
    static constexpr int XI = SFNX_PF_JOB * XROW / 1024 / A2_WAVES, AI = 16 * RT * AROW / 1024 / A2_WAVES;   // copies of a wavefront for a stage
    static constexpr int STAGES = STAGE * 4 <= 144 * 1024 ? 4 : STAGE * 3 <= 144 * 1024 ? 3 : 2;
    static constexpr int P = 16 * RT + 4;
    static constexpr int SUM = 2 * SFNX_PF_JOB * P * 4;
    static constexpr int LDS = STAGES * STAGE > SUM ? STAGES * STAGE : SUM;
    static_assert(LDS <= 144 * 1024, "");
};

template <Elem EL, bool X32, int RT>
__global__ void __launch_bounds__(A2_THREADS) k_adapter_shrink(const AdapterArgs a) {
    typedef Many<X32, RT> M;
    extern __shared__ __align__(16) uint8_t lds_[];
    const Lds L = lds_of(lds_);
    const int part = blockIdx.x % a.parts, j = blockIdx.x / a.parts;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), r = lane % 16, q = lane / 16;
    const sfnx_bigjob& job = a.jobs[j];
    const int nj = *a.njobs, n = min(job.n, SFNX_PF_JOB), w = job.w;
    // the rows this lane copies from: lane_row of copy i
    int y[M::XI];
#pragma unroll
    for (int i = 0; i < M::XI; ++i) y[i] = job_row(job, n, lane_row<M::XROW>((i * A2_WAVES + wave) * (1024 / M::XROW), lane), a.rows).y;
    if (j >= nj || n <= 0 || (unsigned) w >= (unsigned) a.n) return;
    const uint8_t* Aw = expert_at(a.A, a.sa, w);
    const int k0 = part * a.steps * A2_KC, steps = min(a.steps, (a.n_in - k0 + A2_KC - 1) / A2_KC);
    const int turn = j % steps;   // the stage to begin with: jobs that run beside each other read other columns, other channels where rows lie a power of two apart
    const auto request = [&](int step) {
        uint8_t* xl = L.p + step % M::STAGES * M::STAGE;
        uint8_t* al = xl + SFNX_PF_JOB * M::XROW;
        int at = step + turn;
        at = at < steps ? at : at - steps;
        const int k = k0 + at * A2_KC, last = a.n_in - k;
#pragma unroll
        for (int i = 0; i < M::XI; ++i) {
            const int m = (i * A2_WAVES + wave) * (1024 / M::XROW), row = lane_row<M::XROW>(m, lane), c = lane_piece<M::XROW>(row, lane);
            const bool in = y[i] >= 0 && c * (X32 ? 4 : 8) < last;
            copy16(in ? a.x + (int64_t) y[i] * a.ldx + (size_t) k * (X32 ? 4 : 2) + 16 * c : (const uint8_t*) &ZERO16, L.at(xl + m * M::XROW));
        }
#pragma unroll
        for (int i = 0; i < M::AI; ++i) {
            const int m = (i * A2_WAVES + wave) * (1024 / M::AROW), row = lane_row<M::AROW>(m, lane), c = lane_piece<M::AROW>(row, lane);
            const bool in = row < a.rank && 8 * c < last;
            copy16(in ? Aw + 2 * ((size_t) row * a.n_in + k) + 16 * c : (const uint8_t*) &ZERO16, L.at(al + m * M::AROW));
        }
    };
    for (int t = 0; t < M::STAGES - 1 && t < steps; ++t) request(t);
    float4v acc[A2_TILES][RT] = {};
#pragma unroll 1
    for (int t = 0; t < steps; ++t) {
        if (t + M::STAGES - 2 < steps) vm_wait<(M::STAGES - 2) * (M::XI + M::AI)>();
        else vm_wait<0>();
        lds_barrier();   // the stage is there, and the one before it is read
        if (t + M::STAGES - 1 < steps) request(t + M::STAGES - 1);
        const uint8_t* xl = L.p + t % M::STAGES * M::STAGE;
        const uint8_t* al = xl + SFNX_PF_JOB * M::XROW;
        const int c = 4 * wave + q;
        uint4 av[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) av[i] = lds16(lds_piece<M::AROW>(al, 16 * i + r, c));
#pragma unroll
        for (int m = 0; m < A2_TILES; ++m) {   // of a short job's missing rows too: branches here cost more
            const uint4 xa = lds16(lds_piece<M::XROW>(xl, 16 * m + r, X32 ? 2 * c : c)), xb = X32 ? lds16(lds_piece<M::XROW>(xl, 16 * m + r, 2 * c + 1)) : xa;
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[m][i] = shrink_mma<EL, X32>(av[i], xa, xb, acc[m][i]);
        }
    }
    lds_barrier();
    // the wavefronts' sums of token 16 m + r, ranks 16 i + 4 q ..: the upper two hand theirs to the lower two, whose are added
    float* const mine = reinterpret_cast<float*>(L.p) + wave % 2 * SFNX_PF_JOB * M::P;
    if (wave >= 2)
#pragma unroll
        for (int m = 0; m < A2_TILES; ++m)
#pragma unroll
            for (int i = 0; i < RT; ++i) *reinterpret_cast<float4v*>(mine + (16 * m + r) * M::P + 16 * i + 4 * q) = acc[m][i];
    lds_barrier();
    if (wave < 2)
#pragma unroll
        for (int m = 0; m < A2_TILES; ++m)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                float4v* p = reinterpret_cast<float4v*>(mine + (16 * m + r) * M::P + 16 * i + 4 * q);
                *p = acc[m][i] + *p;
            }
    lds_barrier();
    const float* sum = reinterpret_cast<const float*>(L.p);
#pragma unroll 1
    for (int i = threadIdx.x; i < n * 4 * RT; i += A2_THREADS) {
        const int m = i / (4 * RT), c = i % (4 * RT) * 4, o = job_row(job, n, m, a.rows).o;
        if (o >= 0)
            *reinterpret_cast<float4v*>(a.part + ((int64_t) part * a.rows + o) * (16 * RT) + c) =
                *reinterpret_cast<const float4v*>(sum + m * M::P + c) + *reinterpret_cast<const float4v*>(sum + (SFNX_PF_JOB + m) * M::P + c);
    }
}

// The second: out = base + B s on bf16 matrix instructions, s as three bf16 parts whose sum it is: the upper 8 bits of its 24, the next, the
// last (truncated, so that none overflows).  Their products with B's values are exact; f16 values of B are two bf16 parts (the product of
// both lowest, 2^-25 of the whole, is left out).  A part that is 0 times an infinity would be NaN where the product is not, below 2^-110 the
// last part's bits would lie under bf16's smallest value, and f16's largest is 65536 in its first part, whose product with an s of 2^112 is
// infinite: jobs with an s outside [2^-102, 2^112) that is not 0 (above, no part is subnormal), and columns with a B that is not finite, are
// computed value by value, and the call takes as long as such a job does (4096 rows, rank 64, 4096 columns, one value of x infinite: 595 us for 40).
// The results pass through LDS, so that base and out go by whole rows' pieces.
// 4096 rows, rank 64, 4096 columns, bf16, 67 MB of base and out: 24.6 us, of which 6 pass before the first product (the job, then the parts of s, which
// every slice sums and splits for itself), and 2.6 for each unit of 128 columns: reads of LDS and products 1.5, the way out 1.
// the parts of two finite values, packed
__device__ __forceinline__ void split3(float f, float g, uint32_t (&p)[3]) {
    constexpr uint32_t HI = 0xffff0000u;
    const uint32_t a = __float_as_uint(f), b = __float_as_uint(g);
    const float f1 = f - __uint_as_float(a & HI), g1 = g - __uint_as_float(b & HI);
    const uint32_t c = __float_as_uint(f1), d = __float_as_uint(g1);
    const uint32_t x = __float_as_uint(f1 - __uint_as_float(c & HI)), y = __float_as_uint(g1 - __uint_as_float(d & HI));
    p[0] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    p[1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
    p[2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
}
// how far a size's bits lie above S_LOW's; of those below, but 0, more than any
constexpr uint32_t S_LOW = (127u - 102) << 23, S_HIGH = (127u + 112) << 23;
__device__ __forceinline__ uint32_t past_low(float f) {
    const uint32_t b = abs_bits(f);
    return b ? b - S_LOW : 0;
}
// the largest size of 16-bit values, in each half
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t top16(uint32_t top, const uint4& v) {
    ushort2v t = __builtin_bit_cast(ushort2v, top);
    const uint32_t g[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) t = __builtin_elementwise_max(t, __builtin_bit_cast(ushort2v, g[e] & 0x7fff7fffu));
    return __builtin_bit_cast(uint32_t, t);
}

template <int RT> struct Expand {
    static constexpr int KB = RT <= 2 ? 1 : RT / 2;                 // blocks of 32 ranks
    // two workgroups of four wavefronts a compute unit, or one of eight where s takes much of its LDS (4096 rows, 4096 -> 4096, us of the
    // call, four and eight: rank 64 43 and 47; rank 128, 2048 -> 2048, 48 and 39)
    static constexpr int WAVES = RT == 8 ? 8 : 4, EACH = 8 / WAVES, THREADS = WAVES * WAVE;
    static constexpr int COLS = 32 * WAVES, PITCH = COLS + 4;       // columns of a unit, 32 a wavefront; floats of a row of results in LDS
    static constexpr int SP = 32 * KB + 8;                          // values of a token's s in LDS
    static constexpr int S = 3 * SFNX_PF_JOB * SP * 2;
    static constexpr int LDS = S + SFNX_PF_JOB * PITCH * 4;
    static_assert(EACH * LDS <= 160 * 1024, "");
};
template <Elem EL, int RT, int OT>
__global__ void __launch_bounds__(Expand<RT>::THREADS) k_adapter_expand(const AdapterArgs a) {
    typedef Expand<RT> X;
    constexpr int AE_WAVES = X::WAVES, AE_COLS = X::COLS, AE_PITCH = X::PITCH;
    // a thread's rows are tid / LANES + 16 i: base and out 8 columns each, s RK ranks
    constexpr int KB = X::KB, RP = 16 * RT, LANES = AE_COLS / 8, PASSES = SFNX_PF_JOB * LANES / X::THREADS, RK = 32 * KB / LANES;
    static_assert(PASSES == SFNX_PF_JOB / 16, "");
    extern __shared__ __align__(16) uint8_t lds_[];
    uint16_t* const sp = reinterpret_cast<uint16_t*>(lds_);                  // [3][64][SP]
    float* const res = reinterpret_cast<float*>(lds_ + X::S);                // [64][AE_PITCH]
    const int slice = blockIdx.x % a.slices, j = blockIdx.x / a.slices;
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE, r = lane % 16, q = lane / 16, m0 = tid / LANES;
    const int c0 = slice * a.units * AE_COLS, c1 = min(a.n_out, c0 + a.units * AE_COLS), col = tid % LANES * 8, rk = tid % LANES * RK;
    const sfnx_bigjob& job = a.jobs[j];
    const int nj = *a.njobs, n = min(job.n, SFNX_PF_JOB), w = job.w;
    int o[PASSES];
    int64_t row[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        o[i] = job_row(job, n, 16 * i + m0, a.rows).o;
        row[i] = o[i] * a.ldo + col;
    }
    if (j >= nj || n <= 0) return;
    if ((unsigned) w >= (unsigned) a.n) {
#pragma unroll 1
        for (int i = 0; i < PASSES; ++i) copy_base<OT>(a, job_row(job, n, 16 * i + m0, a.rows).o, c0 + col, c1, AE_COLS);
        return;
    }
    const uint8_t* Bw = expert_at(a.B, a.sb, w);
    const float sc = a.scale ? a.scale[w] : 1.f;
    struct Unit {
        Eight<OT> base[PASSES];
        uint4 b[2][KB];   // of the column u + 32 wave + 16 t + r the ranks 32 k + 8 q ..
    };
    Unit g{};
    bool plain = true;
    // pass t multiplies unit t - 1 and writes it, with unit t's base and B on their way; the first makes s meanwhile
    const int units = (c1 - c0 + AE_COLS - 1) / AE_COLS, turn = j % units;   // the unit to begin with, as above
#pragma unroll 1
    for (int t = 0; t <= units; ++t) {
        int at = t - 1 + turn;
        at = at < units ? at : at - units;
        const int u = c0 + at * AE_COLS;   // the unit multiplied (t > 0)
        if (t > 0) {
            uint32_t top = 0;
            bf8v hi[2][KB], lo[2][KB];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    top = top16(top, g.b[h][k]);
                    if constexpr (EL == F16) {
                        float f[8];
                        widen8<F16>(g.b[h][k], f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            hi[h][k][e] = (__bf16) f[e];
                            lo[h][k][e] = (__bf16) (f[e] - (float) hi[h][k][e]);
                        }
                    } else {
                        hi[h][k] = __builtin_bit_cast(bf8v, g.b[h][k]);
                    }
                }
            constexpr uint32_t INF16 = EL == F16 ? 0x7c00u : 0x7f80u;
            const bool fin = __all(plain && (top & 0xffffu) < INF16 && top >> 16 < INF16);
            // tiles of 16 rows at once: all four, or the first of a job that has no more, without branches between them
            const auto tiles = [&](auto count) {
                constexpr int MT = decltype(count)::value;
                float4v d[MT][2] = {};
#pragma unroll
                for (int p = 2; p >= 0; --p)
#pragma unroll
                    for (int k = 0; k < KB; ++k)
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const bf8v s = __builtin_bit_cast(bf8v, lds16((const uint8_t*) (sp + (p * SFNX_PF_JOB + 16 * m + r) * X::SP + 32 * k + 8 * q)));
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if constexpr (EL == F16)
                                    if (p < 2) d[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo[h][k], s, d[m][h], 0, 0, 0);
                                d[m][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi[h][k], s, d[m][h], 0, 0, 0);
                            }
                        }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) *reinterpret_cast<float4v*>(res + (16 * m + r) * AE_PITCH + 32 * wave + 16 * h + 4 * q) = d[m][h];
            };
            if (fin && n <= 16) {
                tiles(std::integral_constant<int, 1>());
            } else if (fin) {
                tiles(std::integral_constant<int, A2_TILES>());
            } else {
#pragma unroll 1
                for (int m = 0; 16 * m < n; ++m) {
                    float4v d[2] = {};
                    const int om = job_row(job, n, 16 * m + r, a.rows).o;
#pragma unroll 1
                    for (int k = 0; k < a.rank; ++k) {
                        float f = 0.f;
                        for (int p = 0; om >= 0 && p < a.parts; ++p) f += a.part[((int64_t) p * a.rows + om) * RP + k];
                        f *= sc;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int c = min(u + 32 * wave + 16 * (e / 4) + 4 * q + e % 4, c1 - 1);
                            d[e / 4][e % 4] = fmaf(f, wide16(EL == F16, reinterpret_cast<const uint16_t*>(Bw)[(size_t) c * a.rank + k]), d[e / 4][e % 4]);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) *reinterpret_cast<float4v*>(res + (16 * m + r) * AE_PITCH + 32 * wave + 16 * h + 4 * q) = d[h];
                }
            }
            lds_barrier();
        }
        Unit next{};
        if (t < units) {
            int an = t + turn;
            an = an < units ? an : an - units;
            const int v = c0 + an * AE_COLS;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const int c = v + 32 * wave + 16 * h + r;
                    if (c < c1 && 32 * k + 8 * q < a.rank) next.b[h][k] = *reinterpret_cast<const uint4*>(Bw + 2 * ((size_t) c * a.rank + 32 * k + 8 * q));
                }
            if (a.base && v + col + 8 <= c1)
#pragma unroll
                for (int i = 0; i < PASSES; ++i)
                    if (o[i] >= 0) next.base[i] = load_eight<OT>(a.base, row[i] + v, 8);
        }
        if (t == 0) {   // s: the parts' sum times the scale, zeros for missing rows and beyond the rank
            constexpr int AT = KB == 1 ? 4 : 2;   // parts requested at once
            float s[PASSES][RK] = {};
            uint32_t size = 0;
            const int64_t step = (int64_t) a.rows * RP;
            const float* at = a.part + rk;
#pragma unroll 1
            for (int p = 0; p < a.parts; p += AT) {
                float x[AT][PASSES][RK] = {};
#pragma unroll
                for (int e = 0; e < AT; ++e)
#pragma unroll
                    for (int i = 0; i < PASSES; ++i)
                        if (p + e < a.parts && o[i] >= 0 && rk < a.rank)
                            __builtin_memcpy(x[e][i], __builtin_assume_aligned(at + (int64_t) (p + e) * step + (int64_t) o[i] * RP, 4 * (RK < 4 ? RK : 4)), 4 * RK);
#pragma unroll
                for (int e = 0; e < AT; ++e)
#pragma unroll
                    for (int i = 0; i < PASSES; ++i)
#pragma unroll
                        for (int c = 0; c < RK; ++c) s[i][c] += x[e][i][c];
            }
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
#pragma unroll
                for (int c = 0; c < RK; c += 2) {
                    const float f = s[i][c] * sc, h = s[i][c + 1] * sc;
                    size = max(size, max(past_low(f), past_low(h)));
                    uint32_t p[3];
                    split3(f, h, p);
#pragma unroll
                    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t*>(sp + (k * SFNX_PF_JOB + 16 * i + m0) * X::SP + rk + c) = p[k];
                }
            const int fin = __all(size < S_HIGH - S_LOW);
            if (lane == 0) reinterpret_cast<int*>(res)[wave * AE_PITCH + AE_COLS] = fin;   // beside the results
            lds_barrier();
#pragma unroll
            for (int k = 0; k < AE_WAVES; ++k) plain = plain && reinterpret_cast<const int*>(res)[k * AE_PITCH + AE_COLS];
        } else {
            if (u + col + 8 <= c1) {
#pragma unroll
                for (int i = 0; i < PASSES; ++i)
                    if (o[i] >= 0) {
                        float v[8];
                        unpack<OT>(g.base[i], v);
                        const float* p = res + (16 * i + m0) * AE_PITCH + col;
                        const float4v x = reinterpret_cast<const float4v*>(p)[0], y = reinterpret_cast<const float4v*>(p)[1];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += x[e], v[4 + e] += y[e];
                        store_eight<OT>(a.out, row[i] + u, 8, pack<OT>(v));
                    }
            } else {   // the row's last columns
#pragma unroll 1
                for (int i = 0; i < PASSES; ++i) {
                    const int om = job_row(job, n, 16 * i + m0, a.rows).o;
#pragma unroll 1
                    for (int c = u + col; om >= 0 && c < c1; ++c) {
                        const float b = a.base ? load_one<OT>(a.base, om * a.ldo + c) : 0.f;
                        store_one<OT>(a.out, om * a.ldo + c, b + res[(16 * i + m0) * AE_PITCH + c - u]);
                    }
                }
            }
            lds_barrier();
        }
        g = next;
    }
}

// ------------------------------------------------------------------------------------------------ launches
template <typename F> void by_type(uint32_t type, F&& f) {
    if (type == SFNX_F32) f(std::integral_constant<int, SFNX_F32>());
    else if (type == SFNX_F16) f(std::integral_constant<int, SFNX_F16>());
    else f(std::integral_constant<int, SFNX_BF16>());
}
int rank_up(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// Parts of the input columns, such that the workgroups of `jobs` jobs run in one round, one a compute unit; at most 8, whose sums the second
// launch reads in each of its slices.
void split_columns(int64_t jobs, int n_in, int& parts, int& steps) {
    const int all = (n_in + A2_KC - 1) / A2_KC;
    parts = (int) std::max<int64_t>(1, std::min<int64_t>({CUS / std::max<int64_t>(1, jobs), (int64_t) all, 8}));
    steps = (all + parts - 1) / parts;
    parts = (all + steps - 1) / steps;
}

// The form.  One launch computes s in each slice and holds 128 KB of LDS, two have a launch more and pass s through memory.  us in a graph, one
// and two launches, 4 adapters of a list of 8, 2048 -> 2048 columns, bf16:
//   rows                 1          16          128         512         1024        2048        4096
//   rank 16, bf16 x      4.7  8.0   6.3  8.2    6.9  9.5    8.3  10.9   10.0 12.3   17.0 16.9   32.5 22.1
//   rank 32, bf16 x      6.1  8.3   7.6  8.5    7.9  10.4   9.5  11.6   11.7 13.9   19.6 18.7   37.3 23.3
//   rank 16, f32 x       5.2  9.2   8.7  9.5    9.9  11.3   11.0 12.3   13.2 14.1   20.5 19.9   38.0 25.8
//   rank 32, f32 x       6.7  10.4  12.1 10.5   13.5 12.4   14.9 13.7   17.2 16.1   25.6 22.5   48.0 28.9
// A window's rows are mostly one to an adapter, which one launch multiplies as the first column does.  Ranks above 32 are two launches: each slice would
// read 256 KB of A for itself, of which a compute unit takes in about 35 KB/us.
bool two_launches(int rows, int rank, bool x32) { return rank > 32 || rows > 1024 || (x32 && rank > 16 && rows > SFNX_MAXT); }

// Jobs that are not full, as launches take them: one for each adapter, and for the rows without; of a long list a chunk's rows are taken to use a
// quarter.  More are a second round of workgroups, fewer leave compute units idle (4096 rows of 16 of 64 adapters, 2048 -> 2048, rank 32, f32:
// 38 us, with all 64 counted 71).  Long lists of which few are used leave them idle all the same: 4096 rows of 4 adapters, rank 64, 4096 columns,
// 39.6 us of a list of 8, 41.0 of 64, 108 of 1000.
int64_t short_jobs(const AdapterArgs& a) {
    const int most = std::min(a.rows, a.n + 1);
    return a.rows <= 256 ? most : (most + 3) / 4;
}

// more than 64 KB of LDS are asked for once a GPU
template <auto KERN, int LDS> void launch_lds(unsigned grid, int threads, const AdapterArgs& a, hipStream_t st) {
    if (LDS > 64 * 1024) {
        static std::atomic<uint64_t> asked{0};
        allow_lds((const void*) KERN, LDS, asked);
    }
    KERN<<<grid, threads, LDS, st>>>(a);
}

template <Elem EL, bool X32, int RT> void launch(AdapterArgs a, uint32_t out_type, int cap, hipStream_t st) {
    const auto slice = [&](int64_t want, int cols) {   // the outputs in about `want` slices of `cols` columns at least
        const int units = (a.n_out + cols - 1) / cols, n = (int) std::max<int64_t>(1, std::min<int64_t>(units, want));
        a.units = (units + n - 1) / n;
        a.slices = (units + a.units - 1) / a.units;
    };
    if (a.part == nullptr) {
        if constexpr (RT <= 2) {
            a.subs = std::min(SFNX_PF_JOB / AD_ROWS, (a.rows + AD_ROWS - 1) / AD_ROWS);
            const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>((int64_t) cap * a.subs, a.rows / AD_ROWS + short_jobs(a)));
            slice(std::max<int64_t>(1, CUS / tiles), AD_UNIT * AW_WAVES);   // one workgroup a compute unit runs at once
            a.units *= AW_WAVES;
            const unsigned grid = grid_of(a.slices * a.subs, cap, AW_THREADS);
            by_type(out_type, [&](auto ot) { launch_lds<k_adapter_mm<EL, X32, RT, decltype(ot)::value>, Few<X32, RT>::LDS>(grid, AW_THREADS, a, st); });
        }
        return;
    }
    const int64_t jobs = std::max<int64_t>(1, std::min<int64_t>(cap, a.rows / SFNX_PF_JOB + short_jobs(a)));
    split_columns(std::max<int64_t>(jobs, a.rows / SFNX_PF_JOB), a.n_in, a.parts, a.steps);   // a short list of many rows' jobs: the workspace goes by rows
    slice(std::max<int64_t>(1, Expand<RT>::EACH * CUS / jobs), Expand<RT>::COLS);
    launch_lds<k_adapter_shrink<EL, X32, RT>, Many<X32, RT>::LDS>(grid_of(a.parts, cap, A2_THREADS), A2_THREADS, a, st);
    const unsigned grid = grid_of(a.slices, cap, Expand<RT>::THREADS);
    by_type(out_type, [&](auto ot) { launch_lds<k_adapter_expand<EL, RT, decltype(ot)::value>, Expand<RT>::LDS>(grid, Expand<RT>::THREADS, a, st); });
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" size_t sfnx_adapter_workspace(int rows, int rank, int n_in, uint32_t x_type) {
    if (rows <= 0 || rank <= 0 || n_in <= 0 || !two_launches(rows, rank, x_type == SFNX_F32)) return 0;
    // Rows times parts, as more than the split gives for any number of jobs and not less for more rows: at most 8 parts, and with j >= 32 jobs 256 / j for fewer
    // than 64 (j + 1) rows
    const int64_t all = (n_in + A2_KC - 1) / A2_KC;
    const int64_t n = std::max<int64_t>(rows, std::min<int64_t>(std::min<int64_t>(8, all) * rows, (int64_t) CUS * SFNX_PF_JOB * 33 / 32));
    return (size_t) n * rank_up(rank) * sizeof(float);
}

extern "C" int sfnx_adapter_mm(const void* A, size_t sa, const void* B, size_t sb, uint32_t type, const float* scale, int n_adapters, int rank,
                               int n_in, int n_out, const sfnx_bigjob* jobs, const int* njobs, int njobs_cap, uint32_t x_type, const void* x,
                               int64_t ldx, const void* base, uint32_t out_type, void* out, int64_t ldo, int rows, void* ws,
                               size_t ws_bytes, void* st) {
    return guarded("sfnx_adapter_mm", [&] {
        require(type == SFNX_F16 || type == SFNX_BF16, "adapter type must be F16 (1) or BF16 (30)");
        require(x_type == SFNX_F32 || x_type == type, "x type must be F32 (0) or the adapters'");
        require(out_type_ok(out_type), "out type must be F32 (0), F16 (1) or BF16 (30)");
        require(n_adapters >= 1 && n_adapters <= (1 << 20), "n_adapters out of range");
        require(rank >= 8 && rank % 8 == 0 && rank <= 128, "rank must be a multiple of 8, at most 128");
        require(n_in > 0 && n_in % 8 == 0 && n_in <= (1 << 20), "input width must be a multiple of 8, at most 2^20");
        require(n_out > 0 && n_out <= (1 << 20), "n_out out of range");
        require(stride_ok(sa, 2 * (size_t) rank * n_in) && stride_ok(sb, 2 * (size_t) n_out * rank), "adapter stride smaller than a matrix");
        require(sa % 16 == 0 && sb % 16 == 0, "adapter stride must be a multiple of 16");
        require(rows >= 0, "rows out of range");
        require(njobs_cap >= 0 && njobs_cap <= (1 << 20), "njobs out of range");
        if (rows == 0 || njobs_cap == 0) return;
        require(A != nullptr && B != nullptr && jobs != nullptr && njobs != nullptr && x != nullptr && out != nullptr, "null pointer");
        require((((uintptr_t) A | (uintptr_t) B | (uintptr_t) x) & 15) == 0, "pointers must be 16-byte aligned");
        const int xs = out_size(x_type), os = out_size(out_type);
        require(ldx >= n_in && ldx <= ((int64_t) 1 << 40) && ldx * xs % 16 == 0, "ldx must be at least n_in, its rows 16-byte aligned");
        require(ldo >= n_out && ldo <= ((int64_t) 1 << 40), "ldo smaller than n_out");
        require((((uintptr_t) out | (uintptr_t) base) & (os - 1)) == 0, "out and base must be aligned to their type");
        require((((uintptr_t) scale | (uintptr_t) jobs | (uintptr_t) njobs) & 3) == 0, "scales and jobs must be 4-byte aligned");
        AdapterArgs a{(const uint8_t*) A, (const uint8_t*) B, sa, sb, scale, n_adapters, rank, n_in, n_out, jobs, njobs, (const uint8_t*) x,
                      ldx * xs, base, out, ldo, rows};
        const size_t need = sfnx_adapter_workspace(rows, rank, n_in, x_type);
        if (need != 0) {
            require(ws != nullptr && ws_bytes >= need, "workspace smaller than sfnx_adapter_workspace");
            require(((uintptr_t) ws & 15) == 0, "workspace must be 16-byte aligned");
            a.part = (float*) ws;
        }
        const auto go = [&](auto el, auto x32) {
            constexpr Elem EL = decltype(el)::value;
            constexpr bool X32 = decltype(x32)::value;
            hipStream_t s = stream_of(st);
            switch (rank_up(rank)) {
                case 16: return launch<EL, X32, 1>(a, out_type, njobs_cap, s);
                case 32: return launch<EL, X32, 2>(a, out_type, njobs_cap, s);
                case 64: return launch<EL, X32, 4>(a, out_type, njobs_cap, s);
                default: return launch<EL, X32, 8>(a, out_type, njobs_cap, s);
            }
        };
        const auto by_x = [&](auto el) {
            if (x_type == SFNX_F32) go(el, std::true_type());
            else go(el, std::false_type());
        };
        if (type == SFNX_F16) by_x(std::integral_constant<Elem, F16>());
        else by_x(std::integral_constant<Elem, BF16>());
    });
}
