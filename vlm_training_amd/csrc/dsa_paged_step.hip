// Attention of a few rows over a paged cache as a launch of its own (dsa_paged_step.h), and the joining of pieces.
#include "dsa_paged_step.h"
#include <algorithm>

namespace {

// The pieces of a block: out = sum of 2^(m_i - m) O_i over sum of 2^(m_i - m) l_i, in a fixed order.  A workgroup takes ITEMS of the block's rows' four columns at a time and
// has 256 / ITEMS threads for each, which take every so many-th piece: 8 or 32 where a few blocks have many pieces (a long request by itself), 256 elsewhere.
template <int ITEMS>
__global__ __launch_bounds__(256) void dsa_paged_join_kernel(dsa_cache_args c, PagedPart many, PagedPart few, int Hq, int gshift,
                                                             bf16_t *__restrict__ out, float *__restrict__ lse) {
    constexpr int GROUPS = 256 / ITEMS;
    const int Hkv = c.Hkv, G = Hq / Hkv, d_real = c.D, kvh = blockIdx.x % Hkv, at_ = blockIdx.x / Hkv;
    const bool shares = at_ >= many.blocks;
    const PagePlan plan = shares ? few.plan : many.plan;
    const float *const part_o = shares ? few.part_o : many.part_o, *const part_ml = shares ? few.part_ml : many.part_ml;
    const int rows = plan.qb << gshift, cols = d_real / 4;
    PagePiece pc;
    int spare;
    if (!(shares ? locate_share_block(plan, at_ - many.blocks, pc) : locate_piece<true>(plan, at_, pc, spare)) || pc.pieces <= 1) return;
    auto slot_of = [&](int i) { return (int64_t)(shares && i ? 2 * i - 1 : i); };            // of piece i, from the first one's
    __shared__ f32x4 sums[GROUPS > 1 ? 256 : 1];
    __shared__ f32x2 stats[GROUPS > 1 ? 256 : 1];
    const int tid = threadIdx.x, group = tid / ITEMS, live = min(pc.m - pc.first, plan.qb) << gshift;
    const int64_t first = (int64_t)pc.slot * Hkv + kvh;
    for (int base = blockIdx.y * ITEMS; base < live * cols; base += gridDim.y * ITEMS) {
        const int item = base + tid % ITEMS, row = item / cols, d = item % cols * 4, head = row & ((1 << gshift) - 1);
        const bool mine = item < live * cols && head < G;
        float m = -INFINITY, l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        if (mine) {
            const int64_t at = first * rows + row, step = (int64_t)Hkv * rows;
#pragma unroll 4
            for (int i = group; i < pc.pieces; i += GROUPS) {
                const f32x2 ml = *reinterpret_cast<const f32x2 *>(part_ml + 2 * (at + slot_of(i) * step));
                const f32x4 x = *reinterpret_cast<const f32x4 *>(part_o + (at + slot_of(i) * step) * d_real + d);
                // (sums against the largest so far: no load waits for another piece's)
                const float most = fmaxf(m, ml[0]), old = m == -INFINITY ? 0.f : fast_exp2(m - most), w = ml[0] == -INFINITY ? 0.f : fast_exp2(ml[0] - most);
                l = fmaf(w, ml[1], l * old);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] *= old;
                    o[e] = ml[0] == -INFINITY ? o[e] : fmaf(w, x[e], o[e]);
                }
                m = most;
            }
        }
        if constexpr (GROUPS > 1) {
            __syncthreads();
            sums[tid] = o;
            stats[tid] = f32x2{m, l};
            __syncthreads();
            if (group == 0) {
                float most = m;
#pragma unroll
                for (int k = 1; k < GROUPS; ++k) most = fmaxf(most, stats[k * ITEMS + tid][0]);
                l = 0.f;
                o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < GROUPS; ++k) {
                    const f32x2 ml = stats[k * ITEMS + tid];
                    const f32x4 x = sums[k * ITEMS + tid];
                    const float w = ml[0] == -INFINITY ? 0.f : fast_exp2(ml[0] - most);
                    l = fmaf(w, ml[1], l);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = ml[0] == -INFINITY ? o[e] : fmaf(w, x[e], o[e]);
                }
                m = most;
            }
        }
        if (mine && group == 0) {
            const int64_t t = pc.row0 + pc.first + (row >> gshift), hq = kvh * G + head;
            const float inv = m == -INFINITY ? 0.f : 1.f / l;
            *reinterpret_cast<u32x2 *>(out + (t * Hq + hq) * d_real + d) = u32x2{pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)};
            if (lse && d == 0) lse[hq * plan.T + t] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * LN2_F;
        }
    }
}

template <int D, bool E4M3, int RG, int NW>
__global__ __launch_bounds__(NW * 64, 1) void dsa_paged_step_kernel(dsa_cache_args c, PagePlan plan, const bf16_t *__restrict__ q, int64_t q_tok, int64_t q_head, int Hq, int gshift,
                                                                    int pshift, float scale_log2, int tail, bf16_t *__restrict__ out, float *__restrict__ lse,
                                                                    float *__restrict__ part_o, float *__restrict__ part_ml) {
    paged_step<D, E4M3, RG, NW>(c, plan, q, q_tok, q_head, Hq, gshift, pshift, scale_log2, tail, out, lse, part_o, part_ml, blockIdx.x / c.Hkv, blockIdx.x % c.Hkv);
}

template <int D, bool E4M3, int RG, int NW>
hipError_t launch_step(const dsa_cache_args &c, const PagePlan &plan, const void *q, int64_t q_tok, int64_t q_head, int Hq, int gshift, int pshift, float scale, int tail, void *out, float *lse, float *part_o, float *part_ml, hipStream_t stream) {
    constexpr int lds = NW * step_wave_bytes<D, E4M3, RG>();
    const auto kernel = &dsa_paged_step_kernel<D, E4M3, RG, NW>;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)plan.target * c.Hkv), dim3(NW * 64), lds, stream, c, plan, (const bf16_t *)q, q_tok, q_head, Hq, gshift, pshift, scale * LOG2E_F,
                       tail, (bf16_t *)out, lse, part_o, part_ml);
    return hipGetLastError();
}

}  // namespace

// waves: 4 at head_dim 65 to 128 in a bf16 cache (else 2 there): a workgroup to a compute unit, for launches in which single pieces count
extern "C" hipError_t dsa_launch_paged_step(const dsa_cache_args *c, const PagePlan *plan, const void *q, int64_t q_tok, int64_t q_head, int Hq, float scale, int waves, int tail,
                                            void *out, float *lse, float *part_o, float *part_ml, hipStream_t stream) {
    const int gshift = group_shift(Hq, c->Hkv), pshift = __builtin_ctz((unsigned)c->page), rows = plan->qb << gshift;
    const bool e = c->kind == DSA_CACHE_E4M3;
    // waves: two workgroups to a compute unit (head_dim 256: one of 132 KB)
#define STEP_ROWS(D_, E_, NW_) return rows <= 16 ? launch_step<D_, E_, 1, NW_>(*c, *plan, q, q_tok, q_head, Hq, gshift, pshift, scale, tail, out, lse, part_o, part_ml, stream) \
                                                 : launch_step<D_, E_, 2, NW_>(*c, *plan, q, q_tok, q_head, Hq, gshift, pshift, scale, tail, out, lse, part_o, part_ml, stream)
    if (rows > 32 || c->D > 256) return hipErrorInvalidValue;
    if (c->D <= 64) {
        if (e) STEP_ROWS(64, true, 4);
        STEP_ROWS(64, false, 4);
    }
    if (c->D <= 128) {
        if (e) STEP_ROWS(128, true, 4);
        if (waves == 4) STEP_ROWS(128, false, 4);
        STEP_ROWS(128, false, 2);
    }
    if (e) STEP_ROWS(256, true, 4);
    STEP_ROWS(256, false, 2);
}
// many: of the walk of many rows (blocks 0: none), few: of this file's
extern "C" hipError_t dsa_launch_paged_join(const dsa_cache_args *c, const PagedPart *many, const PagedPart *few, int Hq, void *out, float *lse, hipStream_t stream) {
    const int gshift = group_shift(Hq, c->Hkv), rows = std::max(many->blocks ? many->plan.qb : 0, few->blocks ? few->plan.qb : 0) << gshift, items = rows * c->D / 4;
    const int wg = (many->blocks + few->blocks) * c->Hkv;
    // workgroups enough for the card where the blocks alone are not
    const bool very = std::max(many->blocks ? many->pieces : 0, few->blocks ? few->pieces : 0) > 16 && (int64_t)wg * ((items + 31) / 32) < 256, some = (int64_t)wg * ((items + 255) / 256) < 256;
    const int y = very ? (items + 7) / 8 : some ? (items + 31) / 32 : std::max(1, std::min((items + 255) / 256, 4096 / wg));
    const auto kernel = very ? &dsa_paged_join_kernel<8> : some ? &dsa_paged_join_kernel<32> : &dsa_paged_join_kernel<256>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wg, (unsigned)y), dim3(256), 0, stream, *c, *many, *few, Hq, gshift, (bf16_t *)out, lse);
    return hipGetLastError();
}
