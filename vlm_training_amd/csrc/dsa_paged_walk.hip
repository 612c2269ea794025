// Attention of a chunk of new tokens over a paged cache as a launch of its own (dsa_paged_walk.h).
#include "dsa_paged_walk.h"

namespace {

template <int D, bool E4M3, bool AGPR>
__global__ __launch_bounds__(WALK_WAVES * 64, D <= 128 ? 2 : 1) void dsa_paged_walk_kernel(dsa_cache_args c, PagePlan plan, const bf16_t *__restrict__ q, int64_t q_tok, int64_t q_head,
                                                                                           int Hq, int gshift, int pshift, float scale_log2, uint32_t flip, int slots, int tail,
                                                                                           bf16_t *__restrict__ out, float *__restrict__ lse, float *__restrict__ part_o,
                                                                                           float *__restrict__ part_ml) {
    paged_walk<D, E4M3, AGPR>(c, plan, q, q_tok, q_head, Hq, gshift, pshift, scale_log2, flip, slots, tail, out, lse, part_o, part_ml, blockIdx.x / c.Hkv, blockIdx.x % c.Hkv);
}

template <int D, bool E4M3>
hipError_t launch_walk(const dsa_cache_args &c, const PagePlan &plan, const void *q, int64_t q_tok, int64_t q_head, int Hq, int gshift, int pshift, float scale, int slots, int tail,
                       void *out, float *lse, float *part_o, float *part_ml, hipStream_t stream) {
    constexpr int lds = walk_lds_bytes<D>();
    const auto kernel = &dsa_paged_walk_kernel<D, E4M3, (D > 128)>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)slots * c.Hkv), dim3(WALK_WAVES * 64), lds, stream, c, plan, (const bf16_t *)q, q_tok, q_head, Hq, gshift, pshift, fabsf(scale) * LOG2E_F,
                       scale < 0.f ? 0x80008000u : 0u, slots, tail, (bf16_t *)out, lse, part_o, part_ml);
    return hipGetLastError();
}

}  // namespace

// plan.qb: 128 rows' queries.  The file is compiled twice, the second time (WALK_256) for head_dim 256, with results of MFMA builtins in vector registers: the sums have the
// accumulation registers.
#define WALK_ARGS const dsa_cache_args *c, const PagePlan *plan, const void *q, int64_t q_tok, int64_t q_head, int Hq, float scale, int slots, int tail, void *out, float *lse, \
    float *part_o, float *part_ml, hipStream_t stream
#define WALK_CASE(D_, E_) return launch_walk<D_, E_>(*c, *plan, q, q_tok, q_head, Hq, gshift, pshift, logit_scale(scale), slots, tail, out, lse, part_o, part_ml, stream)
extern "C" hipError_t dsa_launch_paged_walk_256(WALK_ARGS);
#if WALK_256
extern "C" hipError_t dsa_launch_paged_walk_256(WALK_ARGS) {
    const int gshift = group_shift(Hq, c->Hkv), pshift = __builtin_ctz((unsigned)c->page);
    if (c->kind == DSA_CACHE_E4M3) WALK_CASE(256, true);
    WALK_CASE(256, false);
}
#else
extern "C" hipError_t dsa_launch_paged_walk(WALK_ARGS) {
    const int gshift = group_shift(Hq, c->Hkv), pshift = __builtin_ctz((unsigned)c->page);
    if (plan->qb << gshift != 128 || c->D > 256) return hipErrorInvalidValue;
    if (c->D > 128) return dsa_launch_paged_walk_256(c, plan, q, q_tok, q_head, Hq, scale, slots, tail, out, lse, part_o, part_ml, stream);
    if (c->kind == DSA_CACHE_E4M3) {
        if (c->D <= 64) WALK_CASE(64, true);
        WALK_CASE(128, true);
    }
    if (c->D <= 64) WALK_CASE(64, false);
    WALK_CASE(128, false);
}
#endif
