// A batch of chunks and of single tokens over a paged cache in one launch: the walks of many rows (dsa_paged_walk.h) beside the shares of a few (dsa_paged_step.h).
//
// The shares come first: they are bound by memory, end first, and a compute unit whose first one has ended takes a walk beside the other, which is bound by its instructions and what they
// wait for.  8-bit caches: as many shares as run at once (512 workgroups); bf16: one to a unit, whose waves' tiles of 16 KB keep its memory busy.  us, a launch each -> both in one: a
// chunk of 512 behind 7680, a prompt of 333 and 40 tokens over 200 to 4000 keys, 8-bit 128 -> 117, bf16 143 -> 117; a chunk of 64 and 200 tokens over 4000 keys, 8-bit 337 -> 317 (with 256
// shares 460); a prompt of 2000 and 8 tokens over 3000, 8-bit 86 -> 87; two chunks and 64 tokens over 500 71 -> 60; 1000 behind 29 000 and 60 tokens over 8000 731 -> 703.  256 walks in
// front of the shares: from 3 % less to 19 % more.
#include "dsa_paged_step.h"
#include "dsa_paged_walk.h"

namespace {

constexpr int STEP_RING = 1;                             // (two workgroups to a unit, of four waves each)
template <int D, bool E4M3>
constexpr int both_lds_bytes() {
    const int step = WALK_WAVES * step_wave_bytes<D, E4M3, 1, STEP_RING>();
    return step > walk_lds_bytes<D>() ? step : walk_lds_bytes<D>();
}

template <int D, bool E4M3>
__global__ __launch_bounds__(WALK_WAVES * 64, 2) void dsa_paged_both_kernel(dsa_cache_args c, PagedPart many, PagedPart few, const bf16_t *__restrict__ q, int64_t q_tok, int64_t q_head,
                                                                            int Hq, int gshift, int pshift, float walk_scale, uint32_t flip, float step_scale, int slots,
                                                                            bf16_t *__restrict__ out, float *__restrict__ lse) {
    const int at = blockIdx.x / c.Hkv, kvh = blockIdx.x % c.Hkv, shares = few.plan.target;
    if (at < shares)
        paged_step<D, E4M3, 1, WALK_WAVES, STEP_RING>(c, few.plan, q, q_tok, q_head, Hq, gshift, pshift, step_scale, 0, out, lse, few.part_o, few.part_ml, at, kvh);
    else
        // (8-bit at head_dim 128: with four operands of V ahead beside the shares' code the loop read spilled registers, and the mixed batch took 145 us)
        paged_walk<D, E4M3, false, E4M3 && D == 128 ? 2 : 4>(c, many.plan, q, q_tok, q_head, Hq, gshift, pshift, walk_scale, flip, slots, 1, out, lse, many.part_o, many.part_ml, at - shares, kvh);
}

template <int D, bool E4M3>
hipError_t launch_both(const dsa_cache_args &c, const PagedPart &many, const PagedPart &few, const void *q, int64_t q_tok, int64_t q_head, int Hq, int gshift, int pshift, float scale,
                       int slots, void *out, float *lse, hipStream_t stream) {
    constexpr int lds = both_lds_bytes<D, E4M3>();
    const auto kernel = &dsa_paged_both_kernel<D, E4M3>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    const float walk = logit_scale(scale);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(slots + few.plan.target) * c.Hkv), dim3(WALK_WAVES * 64), lds, stream, c, many, few, (const bf16_t *)q, q_tok, q_head, Hq, gshift, pshift,
                       fabsf(walk) * LOG2E_F, walk < 0.f ? 0x80008000u : 0u, scale * LOG2E_F, slots, (bf16_t *)out, lse);
    return hipGetLastError();
}

}  // namespace

// many.plan.qb: 128 rows' queries, few.plan.qb: up to 16 rows'; head_dim up to 128.  slots: of the walks, for each kv head
extern "C" hipError_t dsa_launch_paged_both(const dsa_cache_args *c, const PagedPart *many, const PagedPart *few, const void *q, int64_t q_tok, int64_t q_head, int Hq, float scale, int slots,
                                            void *out, float *lse, hipStream_t stream) {
    const int gshift = group_shift(Hq, c->Hkv), pshift = __builtin_ctz((unsigned)c->page);
    if (many->plan.qb << gshift != 128 || few->plan.qb << gshift > 16 || c->D > 128) return hipErrorInvalidValue;
#define BOTH_CASE(D_, E_) return launch_both<D_, E_>(*c, *many, *few, q, q_tok, q_head, Hq, gshift, pshift, scale, slots, out, lse, stream)
    if (c->kind == DSA_CACHE_E4M3) {
        if (c->D <= 64) BOTH_CASE(64, true);
        BOTH_CASE(128, true);
    }
    if (c->D <= 64) BOTH_CASE(64, false);
    BOTH_CASE(128, false);
}
