// Experts that are not quantized: f16 or bf16 matrices [n_out][n_in] over the routers' jobs, activations of the same type.
// Few rows are bound by the weights (5 tokens over 65 experts of 1024 x 1024, 53 MB, 11 us, 4.8 TB/s), thousands by the matrix cores
// and what feeds them (4096 tokens over 65 of 2048 x 2048, 282 us, 0.85 PFLOP/s).
#include "mm_few.hpp"
#include "mm_tiles.hpp"

namespace sfnx {
namespace {
using namespace mm;

Args mm16_args(const void* A, size_t sa, uint32_t type, int n_in, int n_out, const void* jobs, const int* njobs, int cap,
               const uint16_t* x, uint32_t out_type, void* out) {
    require(type == SFNX_F16 || type == SFNX_BF16, "expert type must be F16 (1) or BF16 (30)");
    require(out_type_ok(out_type), "out type must be F32 (0), F16 (1) or BF16 (30)");
    require(n_in > 0 && n_in % 8 == 0 && n_in <= (1 << 20), "input width must be a multiple of 8, at most 2^20");
    require(n_out > 0 && n_out <= (1 << 20), "n_out out of range");
    require(2 * (uint64_t) n_out * n_in < ((uint64_t) 1 << 32), "a matrix must be smaller than 4 GiB");
    require(stride_ok(sa, 2 * (size_t) n_out * n_in), "expert stride smaller than a matrix");
    require(sa % 16 == 0, "expert stride must be a multiple of 16");
    require(cap >= 0 && cap <= (1 << 20), "njobs out of range");
    require(A != nullptr && (cap == 0 || (jobs != nullptr && njobs != nullptr && x != nullptr && out != nullptr)), "null pointer");
    require((((uintptr_t) A | (uintptr_t) x) & 15) == 0, "pointers must be 16-byte aligned");
    require(((uintptr_t) out & (out_size(out_type) - 1)) == 0, "out must be aligned to its type");
    const int vec = ((uintptr_t) out & (4 * out_size(out_type) - 1)) == 0 && n_out % 4 == 0;
    return Args{(const uint8_t*) A, sa, n_in, n_out, jobs, njobs, 0, (const uint8_t*) x, nullptr, out, nullptr, out_type, n_out, vec};
}

}  // namespace
}  // namespace sfnx

using namespace sfnx;

extern "C" int sfnx_moe_mm_16(const void* A, size_t sa, uint32_t type, int n_in, int n_out, const sfnx_job* jobs, const int* njobs,
                              int njobs_max, const uint16_t* x, uint32_t out_type, void* out, void* st) {
    return guarded("sfnx_moe_mm_16", [&] {
        const Args a = mm16_args(A, sa, type, n_in, n_out, jobs, njobs, njobs_max, x, out_type, out);
        if (njobs_max == 0) return;
        if (type == SFNX_F16) launch_few<F16, STORE, false>(a, njobs_max, stream_of(st));
        else launch_few<BF16, STORE, false>(a, njobs_max, stream_of(st));
    });
}

extern "C" int sfnx_moe_mm_16_big(const void* A, size_t sa, uint32_t type, int n_in, int n_out, const sfnx_bigjob* jobs,
                                  const int* njobs, int njobs_cap, const uint16_t* x, uint32_t out_type, void* out, void* st) {
    return guarded("sfnx_moe_mm_16_big", [&] {
        const Args a = mm16_args(A, sa, type, n_in, n_out, jobs, njobs, njobs_cap, x, out_type, out);
        if (njobs_cap == 0) return;
        if (type == SFNX_F16) launch_experts<F16>(a, njobs_cap, stream_of(st));
        else launch_experts<BF16>(a, njobs_cap, stream_of(st));
    });
}
