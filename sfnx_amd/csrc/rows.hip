// Rows grouped by a number each carries (an expert, an adapter), tokens' rows in the order of their experts and back with the
// router's weights, and the gradients of both.  No atomics on memory, sums in a fixed order: results repeat bit for bit.
#include "mm.hpp"

namespace sfnx {
namespace {
using namespace mm;

// ------------------------------------------------------------------------------------------------ group_rows
// A stable counting sort: pos[i] = offsets[g] + the rows of g = ids[i] before i.  A workgroup places 256 rows.  It counts the
// rows before its own and all others by group in LDS from a read of all of them, which gives every group's offset, its first
// job (the prefix over groups of ceil(cnt / 64)) and the rank its own rows start from.
constexpr int GR_THREADS = 256, GR_MAX = 4096;

// exclusive prefix sums of two counts over the workgroup's threads
__device__ __forceinline__ void block_prefix(int& a, int& b, int (&sums)[2][GR_THREADS / WAVE]) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
        const int pa = __shfl_up(a, o), pb = __shfl_up(b, o);
        if (lane >= o) a += pa, b += pb;
    }
    if (lane == WAVE - 1) sums[0][wave] = a, sums[1][wave] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GR_THREADS / WAVE; ++w)
        if (w < wave) a += sums[0][w], b += sums[1][w];
    a -= a0, b -= b0;
}

__global__ void __launch_bounds__(GR_THREADS) k_group_rows(const int* __restrict__ ids, int n, int G, int* __restrict__ offsets,
                                                          int* __restrict__ pos, int* __restrict__ order, sfnx_bigjob* __restrict__ jobs,
                                                          int* __restrict__ njobs, int in_place) {
    extern __shared__ int sh[];
    int *before = sh, *total = sh + G, *first = sh + 2 * G;   // first: a group's first job
    __shared__ int mine[GR_THREADS], sums[2][GR_THREADS / WAVE], all;   // all: rows that have a group
    const int tid = threadIdx.x, c0 = blockIdx.x * GR_THREADS, i = c0 + tid;
    for (int g = tid; g < G; g += GR_THREADS) before[g] = total[g] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += GR_THREADS) {
        const int g = ids[j];
        if ((unsigned) g < (unsigned) G) atomicAdd(j < c0 ? &before[g] : &total[g], 1);
    }
    const int g = i < n ? ids[i] : -1;
    const bool in = (unsigned) g < (unsigned) G;
    mine[tid] = in ? g : -1;
    __syncthreads();
    int rank = 0;
    for (int j = 0; j < tid; ++j) rank += mine[j] == g;
    // the prefix over groups, PER consecutive ones a thread
    const int per = (G + GR_THREADS - 1) / GR_THREADS;
    int rows = 0, nj = 0;
    for (int k = 0, h = tid * per; k < per && h < G; ++k, ++h) {
        const int c = before[h] + total[h];
        rows += c, nj += (c + SFNX_PF_JOB - 1) / SFNX_PF_JOB;
    }
    block_prefix(rows, nj, sums);
    for (int k = 0, h = tid * per; k < per && h < G; ++k, ++h) {
        const int c = before[h] + total[h];
        if (blockIdx.x == 0) offsets[h] = rows;
        first[h] = nj;
        total[h] = rows;   // its offset from here on
        rows += c, nj += (c + SFNX_PF_JOB - 1) / SFNX_PF_JOB;
        if (h == G - 1) {
            all = rows;
            if (blockIdx.x == 0) {
                offsets[G] = rows;
                if (njobs) njobs[0] = nj, njobs[1] = 0;
            }
        }
    }
    __syncthreads();
    if (i >= n) return;
    if (!in) {
        if (pos) pos[i] = -1;
        return;
    }
    const int r = before[g] + rank, p = total[g] + r;
    if (pos) pos[i] = p;
    if (order) order[p] = i;
    if (jobs) {
        sfnx_bigjob& j = jobs[first[g] + r / SFNX_PF_JOB];
        const int s = r % SFNX_PF_JOB, v = in_place ? i : p;
        j.y[s] = j.out[s] = v;
        if (s == 0) {
            j.w = g;
            j.n = min(SFNX_PF_JOB, (g + 1 < G ? total[g + 1] : all) - p);
        }
    }
}

// ------------------------------------------------------------------------------------------------ rows of 16- and 32-bit values
// E consecutive values of a row
template <int TYPE> struct ElemOf { typedef uint16_t type; };
template <> struct ElemOf<SFNX_F32> { typedef float type; };
template <int TYPE> __device__ __forceinline__ float to_float(typename ElemOf<TYPE>::type v) {
    if constexpr (TYPE == SFNX_F32) return v;
    else if constexpr (TYPE == SFNX_F16) return h2f(v);
    else return __uint_as_float((uint32_t) v << 16);
}
template <int TYPE> __device__ __forceinline__ typename ElemOf<TYPE>::type from_float(float f) {
    if constexpr (TYPE == SFNX_F32) return f;
    else return (uint16_t) half_bits(TYPE, f);
}
template <int TYPE, int E> struct alignas((TYPE == SFNX_F32 ? 4 : 2) * E < 16 ? (TYPE == SFNX_F32 ? 4 : 2) * E : 16) Pack {
    typename ElemOf<TYPE>::type v[E];
};
template <int TYPE, int E> __device__ __forceinline__ const Pack<TYPE, E>& pack_at(const void* p, int64_t i) {
    return *reinterpret_cast<const Pack<TYPE, E>*>((const typename ElemOf<TYPE>::type*) p + i);
}
template <int TYPE, int E> __device__ __forceinline__ void store_pack(void* p, int64_t i, const float (&v)[E]) {
    Pack<TYPE, E> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = from_float<TYPE>(v[e]);
    *reinterpret_cast<Pack<TYPE, E>*>((typename ElemOf<TYPE>::type*) p + i) = o;
}
constexpr int RW_THREADS = 256, RW_GROUP = 8;   // rows requested before the first is used

// ------------------------------------------------------------------------------------------------ sort_rows
// xs[pos[t][k]] = x[t]: a token's row is read once and written K times.  PIECE: the bytes a thread moves.
template <typename PIECE>
__global__ void __launch_bounds__(RW_THREADS) k_sort_rows(const uint8_t* __restrict__ x, int64_t ldx, int K, int pieces, int blocks,
                                                         const int* __restrict__ pos, uint8_t* __restrict__ xs, int64_t ldxs, int rows) {
    const int t = blockIdx.x / blocks, c = (blockIdx.x % blocks) * RW_THREADS + threadIdx.x;
    if (c >= pieces) return;
    const PIECE v = *(reinterpret_cast<const PIECE*>(x + (int64_t) t * ldx) + c);
    for (int k = 0; k < K; ++k) {
        const int p = pos[(int64_t) t * K + k];
        if ((unsigned) p < (unsigned) rows) *(reinterpret_cast<PIECE*>(xs + (int64_t) p * ldxs) + c) = v;
    }
}

// ------------------------------------------------------------------------------------------------ combine
// y[t] = sum_k w[t][k] ys[pos[t][k]] in k order, fmaf in 32 bits, one rounding to y's type; w null: 1 (the gradient of
// sort_rows).
template <int YS, int Y, int E>
__global__ void __launch_bounds__(RW_THREADS) k_combine_sorted(const void* __restrict__ ys, int64_t ldys, int rows, const float* __restrict__ w,
                                                              const int* __restrict__ pos, int K, int H, int blocks, void* __restrict__ y,
                                                              int64_t ldy) {
    const int t = blockIdx.x / blocks, c = ((blockIdx.x % blocks) * RW_THREADS + threadIdx.x) * E;
    if (c >= H) return;
    float s[E] = {};
    for (int k0 = 0; k0 < K; k0 += RW_GROUP) {
        Pack<YS, E> v[RW_GROUP];
        bool in[RW_GROUP];
#pragma unroll
        for (int k = 0; k < RW_GROUP; ++k) {
            const int p = k0 + k < K ? pos[(int64_t) t * K + k0 + k] : -1;
            in[k] = (unsigned) p < (unsigned) rows;
            if (in[k]) v[k] = pack_at<YS, E>(ys, p * ldys + c);
        }
#pragma unroll
        for (int k = 0; k < RW_GROUP; ++k)
            if (in[k]) {
                const float wk = w ? w[(int64_t) t * K + k0 + k] : 1.f;
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] = fmaf(wk, to_float<YS>(v[k].v[e]), s[e]);
            }
    }
    store_pack<Y, E>(y, t * ldy + c, s);
}

// dys[pos[t][k]] = w[t][k] dy[t], dw[t][k] = sum_h dy[t][h] ys[pos[t][k]][h]: a workgroup takes RW_GROUP picks of a token.  A
// thread's products of a row are summed in 32 bits in column order, then the threads by a tree.
template <int YS, int DY, int E>
__global__ void __launch_bounds__(RW_THREADS) k_combine_sorted_backward(const void* __restrict__ dy, int64_t lddy, const void* __restrict__ ys,
                                                                       int64_t ldys, int rows, const float* __restrict__ w,
                                                                       const int* __restrict__ pos, int K, int H, int groups,
                                                                       void* __restrict__ dys, int64_t lddys, float* __restrict__ dw) {
    const int t = blockIdx.x / groups, k0 = (blockIdx.x % groups) * RW_GROUP;
    __shared__ float part[RW_THREADS / WAVE][RW_GROUP];
    int p[RW_GROUP];
    float wk[RW_GROUP], s[RW_GROUP] = {};
#pragma unroll
    for (int k = 0; k < RW_GROUP; ++k) {
        p[k] = k0 + k < K ? pos[(int64_t) t * K + k0 + k] : -1;
        if ((unsigned) p[k] >= (unsigned) rows) p[k] = -1;
        wk[k] = dys && p[k] >= 0 ? w[(int64_t) t * K + k0 + k] : 0.f;
    }
    for (int c = threadIdx.x * E; c < H; c += RW_THREADS * E) {
        const Pack<DY, E> d = pack_at<DY, E>(dy, t * lddy + c);
        Pack<YS, E> v[RW_GROUP];
        if (dw) {
#pragma unroll
            for (int k = 0; k < RW_GROUP; ++k)
                if (p[k] >= 0) v[k] = pack_at<YS, E>(ys, p[k] * ldys + c);
        }
#pragma unroll
        for (int k = 0; k < RW_GROUP; ++k)
            if (p[k] >= 0) {
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float g = to_float<DY>(d.v[e]);
                    o[e] = wk[k] * g;
                    if (dw) s[k] = fmaf(g, to_float<YS>(v[k].v[e]), s[k]);
                }
                if (dys) store_pack<YS, E>(dys, p[k] * lddys + c, o);
            }
    }
    if (!dw) return;
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
#pragma unroll
    for (int k = 0; k < RW_GROUP; ++k) {
        const float v = group_sum<WAVE>(s[k]);
        if (lane == 0) part[wave][k] = v;
    }
    __syncthreads();
    if (threadIdx.x < RW_GROUP && k0 + (int) threadIdx.x < K) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < RW_THREADS / WAVE; ++q) v += part[q][threadIdx.x];
        dw[(int64_t) t * K + k0 + threadIdx.x] = v;
    }
}

// ------------------------------------------------------------------------------------------------ checks and launches
constexpr int RW_MAX_K = 64;
void check_picks(int T, int K, int H, int rows, const int* pos) {
    require(T >= 0, "T out of range");
    require(K >= 1 && K <= RW_MAX_K, "K out of range (1..64)");
    require(H >= 1 && H <= (1 << 20), "H out of range (1..2^20)");
    require(rows >= 0, "rows out of range");
    require(T == 0 || pos != nullptr, "null pointer");
    require(((uintptr_t) pos & 3) == 0, "pos must be 4-byte aligned");
}
void check_rows(const void* p, int64_t ld, int H, int size, bool used) {
    require(!used || p != nullptr, "null pointer");
    require(((uintptr_t) p & (size - 1)) == 0, "rows must be aligned to their type");
    require(ld >= H && ld <= ((int64_t) 1 << 40), "row stride out of range");
}
void check_type(uint32_t type) { require(out_type_ok(type), "type must be F32 (0), F16 (1) or BF16 (30)"); }
bool wide(const void* p, int64_t ld, int size, int bytes) { return ((uintptr_t) p & (bytes - 1)) == 0 && ld * size % bytes == 0; }
unsigned grid_rows(int T, int blocks) {
    require((int64_t) T * blocks * RW_THREADS < ((int64_t) 1 << 32), "too many rows for one launch");
    return (unsigned) (T * blocks);
}

template <typename F> void by_type(uint32_t type, F&& f) {
    if (type == SFNX_F32) f(std::integral_constant<int, SFNX_F32>());
    else if (type == SFNX_F16) f(std::integral_constant<int, SFNX_F16>());
    else f(std::integral_constant<int, SFNX_BF16>());
}
constexpr int wide_of(uint32_t type) { return type == SFNX_F32 ? 4 : 8; }   // values of 16 bytes

void combine_sorted(uint32_t ys_type, const void* ys, int64_t ldys, int rows, const float* w, const int* pos, int T, int K, int H,
                    uint32_t y_type, void* y, int64_t ldy, hipStream_t st) {
    check_type(ys_type);
    check_type(y_type);
    check_picks(T, K, H, rows, pos);
    check_rows(ys, ldys, H, out_size(ys_type), T > 0 && rows > 0);
    check_rows(y, ldy, H, out_size(y_type), T > 0);
    require(((uintptr_t) w & 3) == 0, "weights must be 4-byte aligned");
    if (T == 0) return;
    by_type(ys_type, [&](auto a) {
        by_type(y_type, [&](auto b) {
            constexpr int YS = decltype(a)::value, Y = decltype(b)::value, E = wide_of(YS);
            const int yb = E * out_size(Y) < 16 ? E * out_size(Y) : 16;
            if (H % E == 0 && wide(ys, ldys, out_size(YS), 16) && wide(y, ldy, out_size(Y), yb)) {
                const int blocks = (H / E + RW_THREADS - 1) / RW_THREADS;
                k_combine_sorted<YS, Y, E><<<grid_rows(T, blocks), RW_THREADS, 0, st>>>(ys, ldys, rows, w, pos, K, H, blocks, y, ldy);
            } else {
                const int blocks = (H + RW_THREADS - 1) / RW_THREADS;
                k_combine_sorted<YS, Y, 1><<<grid_rows(T, blocks), RW_THREADS, 0, st>>>(ys, ldys, rows, w, pos, K, H, blocks, y, ldy);
            }
        });
    });
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" int sfnx_group_rows(const int* ids, int n, int n_groups, int* offsets, int* pos, int* order, sfnx_bigjob* jobs, int* njobs,
                               int njobs_cap, int in_place, void* st) {
    return guarded("sfnx_group_rows", [&] {
        require(n >= 0 && n <= (1 << 20), "n out of range (0..2^20)");
        require(n_groups >= 1 && n_groups <= GR_MAX, "n_groups out of range (1..4096)");
        require((n == 0 || ids != nullptr) && offsets != nullptr, "null pointer");
        require((jobs == nullptr) == (njobs == nullptr), "jobs and njobs go together");
        require((((uintptr_t) ids | (uintptr_t) offsets | (uintptr_t) pos | (uintptr_t) order | (uintptr_t) jobs | (uintptr_t) njobs) & 3) == 0,
                "pointers must be 4-byte aligned");
        require(jobs == nullptr || njobs_cap >= n / SFNX_PF_JOB + std::min(n, n_groups), "njobs_cap smaller than n / 64 + min(n, n_groups)");
        const int blocks = std::max(1, (n + GR_THREADS - 1) / GR_THREADS);
        k_group_rows<<<blocks, GR_THREADS, 3 * n_groups * sizeof(int), stream_of(st)>>>(ids, n, n_groups, offsets, pos, order, jobs, njobs,
                                                                                       in_place);
    });
}

extern "C" int sfnx_moe_sort_rows(int elem, const void* x, int64_t ldx, int T, int K, int H, const int* pos, void* xs, int64_t ldxs, int rows,
                                  void* st) {
    return guarded("sfnx_moe_sort_rows", [&] {
        require(elem == 1 || elem == 2 || elem == 4, "values must be 1, 2 or 4 bytes");
        check_picks(T, K, H, rows, pos);
        check_rows(x, ldx, H, elem, T > 0);
        check_rows(xs, ldxs, H, elem, T > 0 && rows > 0);
        if (T == 0) return;
        const auto go = [&](auto piece) {
            typedef decltype(piece) P;
            const int pieces = (int) ((int64_t) H * elem / sizeof(P)), blocks = (pieces + RW_THREADS - 1) / RW_THREADS;
            k_sort_rows<P><<<grid_rows(T, blocks), RW_THREADS, 0, stream_of(st)>>>((const uint8_t*) x, ldx * elem, K, pieces, blocks, pos,
                                                                                  (uint8_t*) xs, ldxs * elem, rows);
        };
        if (H * elem % 16 == 0 && wide(x, ldx, elem, 16) && wide(xs, ldxs, elem, 16)) go(uint4{});
        else if (elem == 4) go(uint32_t{});
        else if (elem == 2) go(uint16_t{});
        else go(uint8_t{});
    });
}

extern "C" int sfnx_moe_sort_rows_backward(uint32_t dxs_type, const void* dxs, int64_t lddxs, int rows, const int* pos, int T, int K, int H,
                                           uint32_t dx_type, void* dx, int64_t lddx, void* st) {
    return guarded("sfnx_moe_sort_rows_backward", [&] {
        combine_sorted(dxs_type, dxs, lddxs, rows, nullptr, pos, T, K, H, dx_type, dx, lddx, stream_of(st));
    });
}

extern "C" int sfnx_moe_combine_sorted(uint32_t ys_type, const void* ys, int64_t ldys, int rows, const float* topw, const int* pos, int T,
                                       int K, int H, uint32_t y_type, void* y, int64_t ldy, void* st) {
    return guarded("sfnx_moe_combine_sorted", [&] {
        require(T <= 0 || topw != nullptr, "null pointer");
        combine_sorted(ys_type, ys, ldys, rows, topw, pos, T, K, H, y_type, y, ldy, stream_of(st));
    });
}

extern "C" int sfnx_moe_combine_sorted_backward(uint32_t dy_type, const void* dy, int64_t lddy, uint32_t ys_type, const void* ys,
                                                int64_t ldys, int rows, const float* topw, const int* pos, int T, int K, int H, void* dys,
                                                int64_t lddys, float* dw, void* st) {
    return guarded("sfnx_moe_combine_sorted_backward", [&] {
        check_type(dy_type);
        check_type(ys_type);
        check_picks(T, K, H, rows, pos);
        check_rows(dy, lddy, H, out_size(dy_type), T > 0);
        check_rows(ys, ldys, H, out_size(ys_type), T > 0 && rows > 0 && dw != nullptr);
        if (dys) check_rows(dys, lddys, H, out_size(ys_type), false);
        require(T <= 0 || topw != nullptr || dys == nullptr, "null pointer");
        require((((uintptr_t) topw | (uintptr_t) dw) & 3) == 0, "weights must be 4-byte aligned");
        if (T == 0 || (dys == nullptr && dw == nullptr)) return;
        by_type(ys_type, [&](auto a) {
            by_type(dy_type, [&](auto b) {
                constexpr int YS = decltype(a)::value, DY = decltype(b)::value, E = wide_of(YS);
                const int db = E * out_size(DY) < 16 ? E * out_size(DY) : 16, groups = (K + RW_GROUP - 1) / RW_GROUP;
                const unsigned grid = grid_rows(T, groups);
                if (H % E == 0 && wide(ys, ldys, out_size(YS), 16) && (!dys || wide(dys, lddys, out_size(YS), 16)) && wide(dy, lddy, out_size(DY), db))
                    k_combine_sorted_backward<YS, DY, E><<<grid, RW_THREADS, 0, stream_of(st)>>>(dy, lddy, ys, ldys, rows, topw, pos, K, H,
                                                                                               groups, dys, lddys, dw);
                else
                    k_combine_sorted_backward<YS, DY, 1><<<grid, RW_THREADS, 0, stream_of(st)>>>(dy, lddy, ys, ldys, rows, topw, pos, K, H,
                                                                                               groups, dys, lddys, dw);
            });
        });
    });
}
