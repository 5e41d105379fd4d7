// Rows grouped by a number each carries (an expert, an adapter), tokens' rows in the order of their experts and back with the
// router's weights, and the gradients of both.  No atomics on memory, sums in a fixed order: results repeat bit for bit.
#include "mm.hpp"

namespace sfnx {
namespace {
using namespace mm;

// ------------------------------------------------------------------------------------------------ group_rows
// A stable counting sort: pos[i] = offsets[g] + the rows of g = ids[i] before i.  A workgroup places a chunk of rows.  It needs how many rows
// of each group come before its chunk and how many there are: every group's offset and first job are prefixes over groups of the
// counts and of ceil(count / 64).  Few rows are one launch, whose workgroups count all rows for themselves; many are two, the first of
// which counts each chunk into a table.  Within a round of GR_THREADS rows a wavefront's lanes find those before them in the same group by
// ballots of the ids' bits, and the wavefronts before theirs from a byte each of the group's 16.
constexpr int GR_THREADS = 1024, GR_WAVES = GR_THREADS / WAVE, GR_MAX = 4096, GR_PER = GR_MAX / GR_THREADS, GR_CHUNKS = 128;
// Rows up to which one launch is used.  us of the kernels, 512 groups: 4096 rows 6.5 and (two launches) 2.2 + 6.5, 16384 8.0 and 2.4 + 7.1, 40960
// 10.6 and 2.4 + 8.9 and a launch more; 2^20 rows 5 + 38.
constexpr int GR_ALONE = 65536;

__global__ void __launch_bounds__(GR_THREADS) k_group_count(const int* __restrict__ ids, int n, int G, int chunk, int* __restrict__ table) {
    extern __shared__ int hist[];
    const int c0 = blockIdx.x * chunk, c1 = min(n, c0 + chunk);
    for (int g = threadIdx.x; g < G; g += GR_THREADS) hist[g] = 0;
    __syncthreads();
    for (int i = c0 + (int) threadIdx.x; i < c1; i += GR_THREADS) {
        const int g = ids[i];
        if ((unsigned) g < (unsigned) G) atomicAdd(&hist[g], 1);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < G; g += GR_THREADS) table[(size_t) blockIdx.x * G + g] = hist[g];
}

// exclusive prefix sums of two counts over the workgroup's threads
__device__ __forceinline__ void block_prefix(int& a, int& b, int (&sums)[2][GR_WAVES]) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) {
        const int pa = __shfl_up(a, o), pb = __shfl_up(b, o);
        if (lane >= o) a += pa, b += pb;
    }
    if (lane == WAVE - 1) sums[0][wave] = a, sums[1][wave] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GR_WAVES - 1; ++w) {
        a += w < wave ? sums[0][w] : 0;
        b += w < wave ? sums[1][w] : 0;
    }
    a -= a0, b -= b0;
}

constexpr int GR_FIXED = (2 * GR_WAVES + 1) * 4 + 12;   // LDS beside the 28 bytes a group: sums and all, to the next 16 bytes
// table: the chunks' counts, or null
__global__ void __launch_bounds__(GR_THREADS) k_group_rows(const int* __restrict__ ids, int n, int G, int chunk, const int* __restrict__ table,
                                                          int* __restrict__ offsets, int* __restrict__ pos, int* __restrict__ order,
                                                          sfnx_bigjob* __restrict__ jobs, int* __restrict__ njobs, int in_place) {
    extern __shared__ __align__(16) int sh[];
    uint4* const of_wave = reinterpret_cast<uint4*>(sh);                     // a group's rows of this round, a byte a wavefront
    int *run = sh + 4 * G, *off = sh + 5 * G, *first = sh + 6 * G;           // its rows so far, offset and first job
    __shared__ int sums[2][GR_WAVES], all;                // all: rows that have a group
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE, c0 = blockIdx.x * chunk, c1 = min(n, c0 + chunk);
    const int per = (G + GR_THREADS - 1) / GR_THREADS, g0 = tid * per;   // this thread's groups
    int before[GR_PER] = {}, total[GR_PER] = {};
    if (table) {
        constexpr int AT = 16;   // chunks requested at once
        const int nb = gridDim.x, mine = blockIdx.x;
#pragma unroll
        for (int k = 0; k < GR_PER; ++k)
            if (k < per && g0 + k < G)
                for (int b0 = 0; b0 < nb; b0 += AT) {
                    int c[AT];
#pragma unroll
                    for (int e = 0; e < AT; ++e) c[e] = b0 + e < nb ? table[(size_t) (b0 + e) * G + g0 + k] : 0;
#pragma unroll
                    for (int e = 0; e < AT; ++e) {
                        total[k] += c[e];
                        before[k] += b0 + e < mine ? c[e] : 0;
                    }
                }
    } else {
        for (int g = tid; g < G; g += GR_THREADS) run[g] = off[g] = 0;
        __syncthreads();
        for (int i0 = tid; i0 < n; i0 += 8 * GR_THREADS) {
            int g[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = i0 + e * GR_THREADS < n ? ids[i0 + e * GR_THREADS] : -1;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if ((unsigned) g[e] < (unsigned) G) atomicAdd(i0 + e * GR_THREADS < c0 ? &run[g[e]] : &off[g[e]], 1);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < GR_PER; ++k)
            if (k < per && g0 + k < G) {
                before[k] = run[g0 + k];
                total[k] = before[k] + off[g0 + k];
            }
        __syncthreads();
    }
    int rows = 0, nj = 0;
#pragma unroll
    for (int k = 0; k < GR_PER; ++k) rows += total[k], nj += (total[k] + SFNX_PF_JOB - 1) / SFNX_PF_JOB;
    block_prefix(rows, nj, sums);
#pragma unroll
    for (int k = 0; k < GR_PER; ++k)
        if (k < per && g0 + k < G) {
            const int g = g0 + k;
            if (blockIdx.x == 0) offsets[g] = rows;
            run[g] = before[k];
            of_wave[g] = uint4{0, 0, 0, 0};
            off[g] = rows;
            first[g] = nj;
            rows += total[k], nj += (total[k] + SFNX_PF_JOB - 1) / SFNX_PF_JOB;
            if (g == G - 1) {
                all = rows;
                if (blockIdx.x == 0) {
                    offsets[G] = rows;
                    if (njobs) njobs[0] = nj, njobs[1] = 0;
                }
            }
        }
    __syncthreads();
    const int bits = 32 - __clz(G - 1);   // of an id (G = 1: __clz(0) is 32)
    const auto bytes = [](const uint4& v) {
        unsigned n = 0;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) n = __builtin_amdgcn_udot4(w[e], 0x01010101u, n, false);
        return (int) n;
    };
    int next = c0 + tid < c1 ? ids[c0 + tid] : -1;
    for (int i0 = c0; i0 < c1; i0 += GR_THREADS) {
        const int i = i0 + tid, g = next;
        const bool in = (unsigned) g < (unsigned) G, more = i0 + GR_THREADS < c1;
        if (more) next = i + GR_THREADS < c1 ? ids[i + GR_THREADS] : -1;
        uint64_t same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot(g >> b & 1);
            same &= g >> b & 1 ? m : ~m;
        }
        const int mine = __popcll(same & ((1ull << lane) - 1));   // of the same group, before this lane
        if (in && mine == 0) reinterpret_cast<uint8_t*>(of_wave + g)[wave] = (uint8_t) __popcll(same);
        lds_barrier();
        int r = 0;
        if (in) {
            uint4 v = of_wave[g];   // of the wavefronts before this one
            const uint64_t lo = wave >= 8 ? ~0ull : (1ull << 8 * wave) - 1, hi = wave > 8 ? (1ull << 8 * (wave - 8)) - 1 : 0;
            v.x &= (uint32_t) lo, v.y &= (uint32_t) (lo >> 32), v.z &= (uint32_t) hi, v.w &= (uint32_t) (hi >> 32);
            r = run[g] + bytes(v) + mine;
        }
        if (more) {   // the round's rows join those before the next
            lds_barrier();
            for (int k = 0; k < per && g0 + k < G; ++k) {
                run[g0 + k] += bytes(of_wave[g0 + k]);
                of_wave[g0 + k] = uint4{0, 0, 0, 0};
            }
            lds_barrier();
        }
        if (i >= c1) continue;
        if (!in) {
            if (pos) pos[i] = -1;
            continue;
        }
        const int p = off[g] + r;
        if (pos) pos[i] = p;
        if (order) order[p] = i;
        if (jobs) {
            sfnx_bigjob& j = jobs[first[g] + r / SFNX_PF_JOB];
            const int s = r % SFNX_PF_JOB, v = in_place ? i : p;
            j.y[s] = j.out[s] = v;
            if (s == 0) {
                j.w = g;
                j.n = min(SFNX_PF_JOB, (g + 1 < G ? off[g + 1] : all) - p);
            }
        }
    }
}

// rows of a chunk, a multiple of GR_THREADS
int group_chunk(int n) { return (n + GR_THREADS * GR_CHUNKS - 1) / (GR_THREADS * GR_CHUNKS) * GR_THREADS; }

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
// ALIGNED: aligned to the piece's size (16 bytes at most); else to the type's, which is enough for wide accesses
template <int TYPE, int E, bool ALIGNED> __device__ __forceinline__ Pack<TYPE, E> load_pack(const void* p, int64_t i) {
    typedef typename ElemOf<TYPE>::type T;
    Pack<TYPE, E> r;
    __builtin_memcpy(&r, __builtin_assume_aligned((const T*) p + i, ALIGNED ? alignof(Pack<TYPE, E>) : sizeof(T)), E * sizeof(T));
    return r;
}
template <int TYPE, int E, bool ALIGNED> __device__ __forceinline__ void store_pack(void* p, int64_t i, const float (&v)[E]) {
    typedef typename ElemOf<TYPE>::type T;
    Pack<TYPE, E> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = from_float<TYPE>(v[e]);
    __builtin_memcpy(__builtin_assume_aligned((T*) p + i, ALIGNED ? alignof(Pack<TYPE, E>) : sizeof(T)), &o, E * sizeof(T));
}
// A row of n values is n / E pieces and, one by one, the values behind them (none of aligned rows).  us, 2047 and 2048 bf16 columns: 2048 tokens
// with 10 picks sorted 27.6, 18.7; 4096 tokens with 6 picks combined 31.4, 27.6, its gradient 57.7, 48.5.  All value by value 2047 columns took
// 40, 45 and 70.  2% more is written, 3 to 11% more read: the accesses across lines cost in the compute units.
template <int E> constexpr int pieces_of(int n) { return n / E + n % E; }
constexpr int RW_THREADS = 256, RW_GROUP = 8;   // rows requested before the first is used

// ------------------------------------------------------------------------------------------------ sort_rows
// xs[pos[t][k]] = x[t]: a token's row is read once and written K times, 16 bytes a thread (ELEM: the bytes of a value).  Bound by its writes: 2048
// tokens, 10 picks, 2048 bf16 columns, 92 MB, 18.7 us (4.9 TB/s).
template <int ELEM, bool ALIGNED>
__global__ void __launch_bounds__(RW_THREADS) k_sort_rows(const uint8_t* __restrict__ x, int64_t ldx, int K, int H, int blocks,
                                                         const int* __restrict__ pos, uint8_t* __restrict__ xs, int64_t ldxs, int rows) {
    constexpr int E = 16 / ELEM;
    const int t = blockIdx.x / blocks, i = (blockIdx.x % blocks) * blockDim.x + threadIdx.x, full = H / E;
    const auto move = [&](int64_t at, auto v) {
        constexpr int AL = ALIGNED ? 16 : ELEM;
        __builtin_memcpy(&v, __builtin_assume_aligned(x + t * ldx + at, AL), sizeof(v));
        for (int k = 0; k < K; ++k) {
            const int p = pos[(int64_t) t * K + k];
            if ((unsigned) p < (unsigned) rows) __builtin_memcpy(__builtin_assume_aligned(xs + p * ldxs + at, AL), &v, sizeof(v));
        }
    };
    typedef typename std::conditional<ELEM == 4, uint32_t, typename std::conditional<ELEM == 2, uint16_t, uint8_t>::type>::type One;
    if (i < full) move(i * 16, uint4{});
    else if (!ALIGNED && i < pieces_of<E>(H)) move((full * E + i - full) * ELEM, One{});
}

// ------------------------------------------------------------------------------------------------ combine
// y[t] = sum_k w[t][k] ys[pos[t][k]] in k order, fmaf in 32 bits, one rounding to y's type; w null: 1 (the gradient of
// sort_rows).  Bound by its reads: 4096 tokens, 10 picks, 2048 bf16 columns, 185 MB, 40.6 us (4.6 TB/s; 12 rows requested at once 44.5).
template <int YS, int Y, int E, bool ALIGNED>
__global__ void __launch_bounds__(RW_THREADS) k_combine_sorted(const void* __restrict__ ys, int64_t ldys, int rows, const float* __restrict__ w,
                                                              const int* __restrict__ pos, int K, int H, int blocks, void* __restrict__ y,
                                                              int64_t ldy) {
    const int t = blockIdx.x / blocks, i = (blockIdx.x % blocks) * blockDim.x + threadIdx.x, full = H / E;
    const auto sum = [&](int c, auto size) {
        constexpr int N = decltype(size)::value;
        float s[N] = {};
        for (int k0 = 0; k0 < K; k0 += RW_GROUP) {
            Pack<YS, N> v[RW_GROUP];
            bool in[RW_GROUP];
#pragma unroll
            for (int k = 0; k < RW_GROUP; ++k) {
                const int p = k0 + k < K ? pos[(int64_t) t * K + k0 + k] : -1;
                in[k] = (unsigned) p < (unsigned) rows;
                if (in[k]) v[k] = load_pack<YS, N, ALIGNED>(ys, p * ldys + c);
            }
#pragma unroll
            for (int k = 0; k < RW_GROUP; ++k)
                if (in[k]) {
                    const float wk = w ? w[(int64_t) t * K + k0 + k] : 1.f;
#pragma unroll
                    for (int e = 0; e < N; ++e) s[e] = fmaf(wk, to_float<YS>(v[k].v[e]), s[e]);
                }
        }
        store_pack<Y, N, ALIGNED>(y, t * ldy + c, s);
    };
    if (i < full) sum(i * E, std::integral_constant<int, E>());
    else if (!ALIGNED && i < pieces_of<E>(H)) sum(full * E + i - full, std::integral_constant<int, 1>());
}

// dys[pos[t][k]] = w[t][k] dy[t], dw[t][k] = sum_h dy[t][h] ys[pos[t][k]][h]: a workgroup a token, a wavefront a pick (the 17th on go to
// the first again), so that dy's row is in the L1 for all but the first and a pick's sum stays in its wavefront: a lane's products in column
// order by fmaf, then the lanes by a tree.  Bound by memory: 4096 tokens, 6 picks, 2048 bf16 columns, 218 MB, 48.7 us (4.5 TB/s; 42 at a large copy's
// rate); 10 picks of 1024 columns 42 us, where four pieces at once leave room for fewer wavefronts: 56.  With all of a token's
// picks in one thread's registers and their sums joined in LDS 52 and 84.
constexpr int CB_WAVES = 16, CB_AT = 2;   // pieces of a row requested at once
template <int YS, int DY, int E, bool ALIGNED>
__global__ void __launch_bounds__(CB_WAVES * WAVE) k_combine_sorted_backward(const void* __restrict__ dy, int64_t lddy, const void* ys, int64_t ldys,
                                                                            int rows, const float* __restrict__ w, const int* __restrict__ pos,
                                                                            int K, int H, void* dys, int64_t lddys, float* __restrict__ dw) {
    const int t = blockIdx.x, lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), nw = blockDim.x / WAVE;
    for (int k = wave; k < K; k += nw) {
        const int64_t at = (int64_t) t * K + k;
        const int p = pos[at];
        float s = 0.f;
        if ((unsigned) p < (unsigned) rows) {
            const float wk = dys ? w[at] : 0.f;
            const int full = H / E * E;
            for (int c0 = lane * E; c0 < full; c0 += CB_AT * WAVE * E) {
                Pack<DY, E> d[CB_AT];
                Pack<YS, E> v[CB_AT];
#pragma unroll
                for (int u = 0; u < CB_AT; ++u) {
                    const int c = c0 + u * WAVE * E;
                    if (c < full) {
                        d[u] = load_pack<DY, E, ALIGNED>(dy, t * lddy + c);
                        if (dw) v[u] = load_pack<YS, E, ALIGNED>(ys, p * ldys + c);
                    }
                }
#pragma unroll
                for (int u = 0; u < CB_AT; ++u) {
                    const int c = c0 + u * WAVE * E;
                    if (c >= full) continue;
                    float o[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float g = to_float<DY>(d[u].v[e]);
                        o[e] = wk * g;
                        if (dw) s = fmaf(g, to_float<YS>(v[u].v[e]), s);
                    }
                    if (dys) store_pack<YS, E, ALIGNED>(dys, p * lddys + c, o);
                }
            }
            if (!ALIGNED && full + lane < H) {   // the values behind the pieces
                const int c = full + lane;
                const float g = to_float<DY>(load_pack<DY, 1, false>(dy, t * lddy + c).v[0]), o[1] = {wk * g};
                if (dw) s = fmaf(g, to_float<YS>(load_pack<YS, 1, false>(ys, p * ldys + c).v[0]), s);
                if (dys) store_pack<YS, 1, false>(dys, p * lddys + c, o);
            }
            s = group_sum<WAVE>(s);
        }
        if (dw && lane == 0) dw[at] = s;
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
unsigned grid_rows(int T, int blocks, int threads) {
    require((int64_t) T * blocks * threads < ((int64_t) 1 << 32), "too many rows for one launch");
    return (unsigned) T * (unsigned) blocks;
}
// a row's pieces over workgroups of at most RW_THREADS, about the same for each
struct RowSplit {
    int blocks, threads;
};
RowSplit row_split(int pieces) {
    const int blocks = (pieces + RW_THREADS - 1) / RW_THREADS, each = (pieces + blocks - 1) / blocks;
    return RowSplit{blocks, (each + WAVE - 1) / WAVE * WAVE};
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
            const RowSplit r = row_split(pieces_of<E>(H));
            const unsigned grid = grid_rows(T, r.blocks, r.threads);
            if (H % E == 0 && wide(ys, ldys, out_size(YS), 16) && wide(y, ldy, out_size(Y), yb))
                k_combine_sorted<YS, Y, E, true><<<grid, r.threads, 0, st>>>(ys, ldys, rows, w, pos, K, H, r.blocks, y, ldy);
            else
                k_combine_sorted<YS, Y, E, false><<<grid, r.threads, 0, st>>>(ys, ldys, rows, w, pos, K, H, r.blocks, y, ldy);
        });
    });
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" size_t sfnx_group_rows_workspace(int n, int n_groups) {
    if (n <= GR_ALONE || n_groups <= 0) return 0;
    return (size_t) GR_CHUNKS * n_groups * sizeof(int);   // a table of all chunks: for more rows never less
}

extern "C" int sfnx_group_rows(const int* ids, int n, int n_groups, int* offsets, int* pos, int* order, sfnx_bigjob* jobs, int* njobs,
                               int njobs_cap, int in_place, void* ws, size_t ws_bytes, void* st) {
    return guarded("sfnx_group_rows", [&] {
        require(n >= 0 && n <= (1 << 24), "n out of range (0..2^24)");
        require(n_groups >= 1 && n_groups <= GR_MAX, "n_groups out of range (1..4096)");
        require((n == 0 || ids != nullptr) && offsets != nullptr, "null pointer");
        require((jobs == nullptr) == (njobs == nullptr), "jobs and njobs go together");
        require((((uintptr_t) ids | (uintptr_t) offsets | (uintptr_t) pos | (uintptr_t) order | (uintptr_t) jobs | (uintptr_t) njobs | (uintptr_t) ws) & 3) == 0,
                "pointers must be 4-byte aligned");
        require(jobs == nullptr || njobs_cap >= n / SFNX_PF_JOB + std::min(n, n_groups), "njobs_cap smaller than n / 64 + min(n, n_groups)");
        const size_t need = sfnx_group_rows_workspace(n, n_groups);
        require(need == 0 || (ws != nullptr && ws_bytes >= need), "workspace smaller than sfnx_group_rows_workspace");
        const int chunk = need ? group_chunk(n) : GR_THREADS, blocks = std::max(1, (n + chunk - 1) / chunk);
        int* const table = need ? (int*) ws : nullptr;
        if (table) k_group_count<<<blocks, GR_THREADS, n_groups * sizeof(int), stream_of(st)>>>(ids, n, n_groups, chunk, table);
        static std::atomic<uint64_t> asked{0};
        const int lds = 28 * n_groups;
        if (lds + GR_FIXED > 64 * 1024) allow_lds((const void*) k_group_rows, 28 * GR_MAX, asked);
        k_group_rows<<<blocks, GR_THREADS, lds, stream_of(st)>>>(ids, n, n_groups, chunk, table, offsets, pos, order, jobs, njobs, in_place);
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
        const bool aligned = H * elem % 16 == 0 && wide(x, ldx, elem, 16) && wide(xs, ldxs, elem, 16);
        const auto go = [&](auto size) {
            constexpr int ELEM = decltype(size)::value;
            const RowSplit r = row_split(pieces_of<16 / ELEM>(H));
            const unsigned grid = grid_rows(T, r.blocks, r.threads);
            const auto kern = aligned ? k_sort_rows<ELEM, true> : k_sort_rows<ELEM, false>;
            kern<<<grid, r.threads, 0, stream_of(st)>>>((const uint8_t*) x, ldx * elem, K, H, r.blocks, pos, (uint8_t*) xs, ldxs * elem, rows);
        };
        if (elem == 4) go(std::integral_constant<int, 4>());
        else if (elem == 2) go(std::integral_constant<int, 2>());
        else go(std::integral_constant<int, 1>());
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
        const unsigned grid = grid_rows(T, 1, CB_WAVES * WAVE);
        by_type(ys_type, [&](auto a) {
            by_type(dy_type, [&](auto b) {
                constexpr int YS = decltype(a)::value, DY = decltype(b)::value, E = wide_of(YS);
                const int db = E * out_size(DY) < 16 ? E * out_size(DY) : 16, threads = std::min(K, CB_WAVES) * WAVE;
                if (H % E == 0 && wide(ys, ldys, out_size(YS), 16) && (!dys || wide(dys, lddys, out_size(YS), 16)) && wide(dy, lddy, out_size(DY), db))
                    k_combine_sorted_backward<YS, DY, E, true><<<grid, threads, 0, stream_of(st)>>>(dy, lddy, ys, ldys, rows, topw, pos, K, H, dys, lddys, dw);
                else
                    k_combine_sorted_backward<YS, DY, E, false><<<grid, threads, 0, stream_of(st)>>>(dy, lddy, ys, ldys, rows, topw, pos, K, H, dys, lddys, dw);
            });
        });
    });
}
