// Low-rank adapters of many requests beside a shared projection: out = base + scale_a B_a (A_a x) for the rows of each job,
// whose adapter is a.
//
// A workgroup takes 16 rows of a job and a slice of the outputs.  Its wavefronts share the input columns for s = A_a x on the
// matrix cores (the adapter's rows are the A operand, the tokens the B operand), meet in LDS in wavefront order, and then take
// the outputs 32 columns at a time.  s stays in 32 bits: B_a is multiplied on v_mfma_f32_16x16x4_f32, so that the one rounding is
// that of the output.  Activations of 32 bits are multiplied so too; those of the adapters' type on 16x16x32, whose products are
// exact.
#include "mm.hpp"

namespace sfnx {
namespace {
using namespace mm;

constexpr int AD_WAVES = 4, AD_THREADS = AD_WAVES * WAVE, AD_ROWS = 16, AD_UNIT = 32;   // rows of a workgroup; columns of a unit of outputs
constexpr int AD_PITCH = AD_ROWS + 1;

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
    uint32_t out_type;
    int rows;                 // of x, base and out
    int slices, units;        // of the outputs: slices of `units` units
    int vec;                  // a lane's eight consecutive outputs are aligned to 16 bytes
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

// eight consecutive values of a row of base or out from column c on, those below `left`
__device__ __forceinline__ void load_base(const void* p, uint32_t type, int64_t i, int left, bool vec, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (p == nullptr) return;
    if (type == SFNX_F32) {
        const float* f = (const float*) p + i;
        if (vec && left >= 8) {
            const float4v a = reinterpret_cast<const float4v*>(f)[0], b = reinterpret_cast<const float4v*>(f)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) v[e] = f[e];
        }
        return;
    }
    const uint16_t* h = (const uint16_t*) p + i;
    if (vec && left >= 8) {
        const uint4 u = *reinterpret_cast<const uint4*>(h);
        if (type == SFNX_F16) widen8<F16>(u, v);
        else widen8<BF16>(u, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) v[e] = wide16(type == SFNX_F16, h[e]);
    }
}
__device__ __forceinline__ void store_out(void* p, uint32_t type, int64_t i, int left, bool vec, const float (&v)[8]) {
    if (vec && left >= 8 && type != SFNX_F32) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = half_bits(type, v[2 * k]) | half_bits(type, v[2 * k + 1]) << 16;
        *reinterpret_cast<uint4*>((uint16_t*) p + i) = uint4{w[0], w[1], w[2], w[3]};
        return;
    }
    store4(p, type, i, float4v{v[0], v[1], v[2], v[3]}, left, vec);
    store4(p, type, i + 4, float4v{v[4], v[5], v[6], v[7]}, left - 4, vec);
}

// RT: the rank in tiles of 16, rounded up to 1, 2, 4 or 8
template <Elem EL, bool X32, int RT>
__global__ void __launch_bounds__(AD_THREADS) k_adapter_mm(const AdapterArgs a) {
    __shared__ float part[AD_WAVES][RT * 16 * AD_PITCH];
    __shared__ int yrow[AD_ROWS], orow[AD_ROWS];
    const int slice = blockIdx.x % a.slices, sub = blockIdx.x / a.slices % (SFNX_PF_JOB / AD_ROWS);
    const int j = blockIdx.x / a.slices / (SFNX_PF_JOB / AD_ROWS), m0 = sub * AD_ROWS;
    const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE, r = lane % 16, q = lane / 16;
    if (j >= *a.njobs) return;
    const sfnx_bigjob& job = a.jobs[j];
    const int n = min(job.n, SFNX_PF_JOB) - m0, w = job.w;
    if (n <= 0) return;
    if (tid < AD_ROWS) {   // a row that is none of x's and out's counts as missing
        const int y = tid < n ? job.y[m0 + tid] : -1, o = tid < n ? job.out[m0 + tid] : -1;
        const bool ok = (unsigned) y < (unsigned) a.rows && (unsigned) o < (unsigned) a.rows;
        yrow[tid] = ok ? y : -1;
        orow[tid] = ok ? o : -1;
    }
    __syncthreads();
    const int c0 = slice * a.units * AD_UNIT, c1 = min(a.n_out, c0 + a.units * AD_UNIT);
    const int o = orow[r];
    if ((unsigned) w >= (unsigned) a.n) {   // no adapter
        if (a.base == a.out) return;
        for (int c = c0 + wave * AD_UNIT + 8 * q; c < c1; c += AD_WAVES * AD_UNIT)
            if (o >= 0) {
                float v[8];
                load_base(a.base, a.out_type, o * a.ldo + c, c1 - c, a.vec, v);
                store_out(a.out, a.out_type, o * a.ldo + c, c1 - c, a.vec, v);
            }
        return;
    }
    // ---- s = A x: rank rows 16 t + 4 q + i of token r, over this wavefront's steps of 64 columns
    float4v acc[RT] = {};
    const uint8_t* Aw = expert_at(a.A, a.sa, w);
    const int y = yrow[r];
    const uint8_t* xr = a.x + (int64_t) max(y, 0) * a.ldx;
    const uint4 zero = {0, 0, 0, 0};
    for (int k0 = wave * 64; k0 < a.n_in; k0 += AD_WAVES * 64) {
        const int k[2] = {k0 + 8 * q, k0 + 32 + 8 * q};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = k[h] < a.n_in, xin = in && y >= 0;
            uint4 wv[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int row = 16 * t + r;
                wv[t] = in && row < a.rank ? *reinterpret_cast<const uint4*>(Aw + 2 * ((size_t) row * a.n_in + k[h])) : zero;
            }
            if constexpr (X32) {
                const float4v *p = reinterpret_cast<const float4v*>(xr) + k[h] / 4;
                const float4v xa = xin ? p[0] : float4v{}, xb = xin ? p[1] : float4v{};
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float f[8];
                    widen8<EL>(wv[t], f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], e < 4 ? xa[e] : xb[e - 4], acc[t], 0, 0, 0);
                }
            } else {
                const uint4 xv = xin ? *reinterpret_cast<const uint4*>(xr + 2 * (size_t) k[h]) : zero;
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    if constexpr (EL == F16)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, wv[t]), __builtin_bit_cast(half8v, xv), acc[t], 0, 0, 0);
                    else
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, wv[t]), __builtin_bit_cast(bf8v, xv), acc[t], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][(16 * t + 4 * q + i) * AD_PITCH + r] = acc[t][i];
    __syncthreads();
    // ---- out = base + B (scale s): lane l holds s of token r for the 4 RT ranks from 4 RT q on
    float s[4 * RT];
    const float sc = a.scale ? a.scale[w] : 1.f;
#pragma unroll
    for (int i = 0; i < 4 * RT; ++i) {
        float v = 0.f;
#pragma unroll
        for (int p = 0; p < AD_WAVES; ++p) v += part[p][(4 * RT * q + i) * AD_PITCH + r];
        s[i] = 4 * RT * q + i < a.rank ? v * sc : 0.f;   // beyond the rank 0 x may be 0 inf
    }
    const uint8_t* Bw = expert_at(a.B, a.sb, w);
    for (int u = c0 + wave * AD_UNIT; u < c1; u += AD_WAVES * AD_UNIT) {
        // a tile's row r is column u + 8 (r / 4) + 4 t + r % 4, so that lane l's results are the columns u + 8 q .. u + 8 q + 7
        float v[8];
        load_base(o >= 0 ? a.base : nullptr, a.out_type, max(o, 0) * a.ldo + u + 8 * q, c1 - u - 8 * q, a.vec, v);
        float4v d[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = u + 8 * (r / 4) + 4 * t + r % 4;
            const uint8_t* b = Bw + 2 * ((size_t) c * a.rank + 4 * RT * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[t][i] = v[4 * t + i];
#pragma unroll
            for (int p = 0; p < 4 * RT; p += (RT == 1 ? 4 : 8)) {
                const bool in = c < c1 && 4 * RT * q + p < a.rank;   // rank is a multiple of 8
                float f[8];
                if constexpr (RT == 1) {
                    const uint2 g = in ? *reinterpret_cast<const uint2*>(b + 2 * p) : uint2{0, 0};
                    widen8<EL>(uint4{g.x, g.y, 0, 0}, f);
                } else {
                    widen8<EL>(in ? *reinterpret_cast<const uint4*>(b + 2 * p) : zero, f);
                }
#pragma unroll
                for (int e = 0; e < (RT == 1 ? 4 : 8); ++e) d[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(f[e], s[p + e], d[t], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * t + i] = d[t][i];
        }
        if (o >= 0) store_out(a.out, a.out_type, o * a.ldo + u + 8 * q, c1 - u - 8 * q, a.vec, v);
    }
}

template <Elem EL, bool X32> void launch(const AdapterArgs& a, unsigned grid, hipStream_t st) {
    if (a.rank <= 16) k_adapter_mm<EL, X32, 1><<<grid, AD_THREADS, 0, st>>>(a);
    else if (a.rank <= 32) k_adapter_mm<EL, X32, 2><<<grid, AD_THREADS, 0, st>>>(a);
    else if (a.rank <= 64) k_adapter_mm<EL, X32, 4><<<grid, AD_THREADS, 0, st>>>(a);
    else k_adapter_mm<EL, X32, 8><<<grid, AD_THREADS, 0, st>>>(a);
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" int sfnx_adapter_mm(const void* A, size_t sa, const void* B, size_t sb, uint32_t type, const float* scale, int n_adapters, int rank,
                               int n_in, int n_out, const sfnx_bigjob* jobs, const int* njobs, int njobs_cap, uint32_t x_type, const void* x,
                               int64_t ldx, const void* base, uint32_t out_type, void* out, int64_t ldo, int rows, void* st) {
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
        const int units = (n_out + AD_UNIT - 1) / AD_UNIT, subs = SFNX_PF_JOB / AD_ROWS;
        // slices of the outputs: enough workgroups to fill the chip, each with a unit a wavefront at least
        const int64_t tiles = std::min((int64_t) njobs_cap * subs, (int64_t) njobs_cap + rows / AD_ROWS);
        const int slices = (int) std::max<int64_t>(1, std::min<int64_t>((units + AD_WAVES - 1) / AD_WAVES, (4 * CUS + tiles - 1) / tiles));
        AdapterArgs a{(const uint8_t*) A, (const uint8_t*) B, sa, sb, scale, n_adapters, rank, n_in, n_out, jobs, njobs, (const uint8_t*) x,
                      ldx * xs, base, out, ldo, out_type, rows};
        a.units = (units + slices - 1) / slices;
        a.slices = (units + a.units - 1) / a.units;
        a.vec = (((uintptr_t) out | (uintptr_t) base) & 15) == 0 && ldo * os % 16 == 0;
        const unsigned grid = grid_of(a.slices * subs, njobs_cap, AD_THREADS);
        if (type == SFNX_F16) {
            if (x_type == SFNX_F32) launch<F16, true>(a, grid, stream_of(st));
            else launch<F16, false>(a, grid, stream_of(st));
        } else {
            if (x_type == SFNX_F32) launch<BF16, true>(a, grid, stream_of(st));
            else launch<BF16, false>(a, grid, stream_of(st));
        }
    });
}
