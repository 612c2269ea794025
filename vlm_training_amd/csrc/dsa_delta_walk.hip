// Gated delta rule: the walks of the state, forward and backward (dsa_delta.h and dsa_delta_bwd.hip have the formulas), where there are many of heads of 128.
//
// One workgroup of eight waves per sequence and value head.  A wave has 16 columns of the state and all of its rows, in registers (fp32) from the first chunk to
// the last, so the chain of a chunk's products - forward K S0, T R, K^T N - never leaves its registers: a result of mfma16 has rows 16 t + 4 (l/16) + v of column
// l%16 in lane l, and two such tiles are an operand of the next product whose contraction runs over rows 32 s + 4 (l/16) + 0..3 and 16 further.  The other
// operand is read to match: K and Q in two pieces of eight bytes, K^T with its rows so, T and P laid out so by the kernel that forms them.  What is
// written (O, and N, dR for the gradients) is formed transposed from the same registers, so that a lane has four neighbours of a row.
// K, Q, V, T and P come into LDS once per workgroup, the next chunk's while this one is worked on; one barrier a chunk.
#include "dsa_delta.h"

enum { WALK_D = 128, WALK_W = 8, WALK_KB = WALK_D / 32, WALK_KS = WALK_D + 8 };
enum { WALK_LANES = WALK_D / 8, WALK_ROWS = 64 * WALK_W / WALK_LANES };      // lanes to a row of K, Q or V, rows to a load
struct DeltaTiles {
    bf16_t k[64 * WALK_KS], q[64 * WALK_KS], v[64 * WALK_KS], tp[24 * 512];  // v: V, backward dO; tp: T hi, lo, P hi, lo, six blocks of 16 rows x 32 columns each
    float f[5 * 64];                                     // the rows' factors, DELTA_EG to DELTA_RQ
};
struct DeltaAhead {
    u32x4 k[2], q[2], v[2], m[3], f;
};
static_assert(2 * WALK_ROWS == 64 && 3 * WALK_W == 24, "a thread's loads of a chunk");
// Where a workgroup's threads find their part of a chunk.  BACK: T and P transposed, from the last chunk to the first.
template <bool BACK> struct DeltaLoader {
    const char *pk, *pq, *pv, *pm;
    int64_t step_m;
    int at_k, at_q, at_v, k_tok, q_tok, v_tok, Dk, v_width, rows_all, mats_bytes, planes, chunks;
    __device__ __forceinline__ void start(const DeltaArgs &a, const bf16_t *v, int64_t vtok, int64_t vhead, int h, int hk, int s0, int L, int slot0, int n) {
        const dsa_delta_args &in = a.in;
        const int tid = threadIdx.x;
        chunks = n;
        const int64_t first = BACK ? n - 1 : 0, t0 = s0 + 64 * first;
        k_tok = (int)in.k_tok;
        q_tok = (int)in.q_tok;
        v_tok = (int)vtok;
        Dk = in.Dk;
        v_width = in.Dv;
        rows_all = min(L, in.T - s0);
        mats_bytes = a.mats_bytes;
        planes = a.planes;
        const int row = tid / WALK_LANES, col = tid % WALK_LANES * 8;
        at_k = col < Dk ? (row * k_tok + col) * 2 : NOWHERE;
        at_q = col < Dk ? (row * q_tok + col) * 2 : NOWHERE;
        at_v = col < v_width ? (row * v_tok + col) * 2 : NOWHERE;
        pk = (const char *)in.k + (t0 * in.k_tok + hk * in.k_head) * 2;
        pq = (const char *)in.q + (t0 * in.q_tok + hk * in.q_head) * 2;
        pv = (const char *)v + (t0 * vtok + h * vhead) * 2;
        pm = a.mats + ((slot0 + first) * in.Hv + h) * a.mats_bytes;
        step_m = (BACK ? -1 : 1) * (int64_t)in.Hv * a.mats_bytes;
    }
    // chunk i; the last one of the walk is fetched again and again (behind a branch, waits would be for every load in flight)
    __device__ __forceinline__ void fetch(int i, DeltaAhead &x) {
        const int n = min(64, rows_all - 64 * i), lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const buffer_t k = rows_buffer(pk, k_tok, n, Dk), q = rows_buffer(pq, q_tok, n, Dk), v = rows_buffer(pv, v_tok, n, v_width), m = buffer_of(pm, mats_bytes);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            x.k[e] = __builtin_bit_cast(u32x4, buf16(k, further(at_k, e * WALK_ROWS * k_tok * 2)));
            x.q[e] = __builtin_bit_cast(u32x4, buf16(q, further(at_q, e * WALK_ROWS * q_tok * 2)));
            x.v[e] = __builtin_bit_cast(u32x4, buf16(v, further(at_v, e * WALK_ROWS * v_tok * 2)));
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) {
            const int b = wv + WALK_W * e, plane = b / 6, j = b % 6;
            // block j: 16 rows, then which half of the columns (upper rows have the first alone, transposed lower ones the second)
            const int block = BACK ? (j < 4 ? j : 2 * j - 3) : (j < 2 ? 2 * j : j + 2);
            const int where = DELTA_T + ((plane & 2 ? planes : 0) + (BACK ? 2 : 0) + (plane & 1)) * DELTA_PLANE + block * 1024;
            x.m[e] = __builtin_bit_cast(u32x4, buf16(m, lane * 16, where));
        }
        x.f = __builtin_bit_cast(u32x4, buf16(m, threadIdx.x * 16));
        const int go = BACK ? (i > 0 ? -64 : 0) : i + 1 < chunks ? 64 : 0;
        pk += (int64_t)go * k_tok * 2;
        pq += (int64_t)go * q_tok * 2;
        pv += (int64_t)go * v_tok * 2;
        pm += go ? step_m : 0;
    }
    __device__ __forceinline__ void put(const DeltaAhead &x, DeltaTiles &t) {
        const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, at = tid / WALK_LANES * WALK_KS + tid % WALK_LANES * 8;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<u32x4_any *>(t.k + at + e * WALK_ROWS * WALK_KS) = x.k[e];
            *reinterpret_cast<u32x4_any *>(t.q + at + e * WALK_ROWS * WALK_KS) = x.q[e];
            *reinterpret_cast<u32x4_any *>(t.v + at + e * WALK_ROWS * WALK_KS) = x.v[e];
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) *reinterpret_cast<u32x4_any *>(t.tp + (wv + WALK_W * e) * 512 + lane * 8) = x.m[e];
        if (tid < 80) *reinterpret_cast<u32x4_any *>(t.f + tid * 4) = x.f;
    }
};
// rows r0 + l%16, columns c0 + 4 (l/16) + 0..3 and 16 further
__device__ __forceinline__ bf16x8 frag_rows(const bf16_t *t, int stride, int r0, int c0) {
    const int l = threadIdx.x & 63;
    const bf16_t *const p = t + (r0 + (l & 15)) * stride + c0 + 4 * (l >> 4);
    const u32x2 a = *reinterpret_cast<const u32x2_any *>(p), b = *reinterpret_cast<const u32x2_any *>(p + 16);
    return __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
}
// two tiles as an operand: hi, and what it leaves
__device__ __forceinline__ void split8(f32x4 x, f32x4 y, bf16x8 &hi, bf16x8 &lo) {
    const u32x2 a = hi4(x), b = hi4(y), c = lo4(x, a), d = lo4(y, b);
    hi = __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
    lo = __builtin_bit_cast(bf16x8, u32x4{c[0], c[1], d[0], d[1]});
}
__device__ __forceinline__ f32x4 row_factors(const float *f, int which, int r0) { return *reinterpret_cast<const f32x4 *>(f + which * 64 + r0); }
__device__ __forceinline__ f32x4 lower4(bf16x8 x) { const u32x4 w = __builtin_bit_cast(u32x4, x); return up4(u32x2{w[0], w[1]}); }
__device__ __forceinline__ f32x4 upper4(bf16x8 x) { const u32x4 w = __builtin_bit_cast(u32x4, x); return up4(u32x2{w[2], w[3]}); }
// block (16 rows t, 32 columns s) of plane p: transposed rows begin at the diagonal, the others end there
template <bool BACK> __device__ __forceinline__ bf16x8 plane_block(const bf16_t *tp, int p, int t, int s) {
    const int j = BACK ? (t < 2 ? 2 * t + s : t + 2) : (t < 2 ? t : 2 * t - 2 + s);
    return *reinterpret_cast<const bf16x8 *>(tp + (p * 6 + j) * 512 + (threadIdx.x & 63) * 8);
}
enum { PLANE_TH, PLANE_TL, PLANE_PH, PLANE_PL };

// the state of a walk, from or to memory: st[s][hh] has rows 32 s + 16 hh + 4 (l/16) + v of column l%16
template <typename F> __device__ __forceinline__ void each_state(F f) {
    const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < WALK_KB; ++s)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int v = 0; v < 4; ++v) f(s, hh, v, 32 * s + 16 * hh + 4 * g4 + v);
}
template <bool SAVE>
__global__ __launch_bounds__(64 * WALK_W, 2) void dsa_delta_walk_kernel(DeltaArgs a) {
    constexpr int KB = WALK_KB, KS = WALK_KS, VS = WALK_KS;
    __shared__ __align__(16) DeltaTiles tiles[2];
    const dsa_delta_args &in = a.in;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    int64_t unit;
    int block, slot0, chunks, s0, L;
    if (a.choose && delta_form(a) != DELTA_HEAD) return;
    if (!delta_walk_unit(blockIdx.x, 1, (int64_t)in.N * in.Hv, unit, block)) return;
    const int h = (int)(unit % in.Hv), seg = delta_longest(in.cu, in.N, (int)(unit / in.Hv)), hk = h / (in.Hv / in.Hk), dv0 = 16 * wv;
    delta_segment(in.cu, in.N, seg, slot0, chunks, s0, L);
    chunks = min(chunks, a.slots - slot0);
    s0 = max(s0, 0);
    f32x4 st[KB][2];
    const int64_t cell = ((int64_t)seg * in.Hv + h) * in.Dk * in.Dv + dv0 + l16;
    each_state([&](int s, int hh, int v, int k) {
        st[s][hh][v] = a.initial && k < in.Dk && dv0 + l16 < in.Dv ? a.initial[cell + (int64_t)k * in.Dv] : 0.f;
    });
    loads_done();
    DeltaLoader<false> loader;
    DeltaAhead x;
    char *ps = a.saved + ((int64_t)slot0 * in.Hv + h) * a.saved_bytes, *po = (char *)(a.out + ((int64_t)s0 * in.Hv + h) * in.Dv);
    const int64_t step_s = (int64_t)in.Hv * a.saved_bytes;
    const int o_tok = in.Hv * in.Dv, rows_all = min(L, in.T - s0);
    const int orow = lane / 2, ocol = lane % 2 * 8, at_o = dv0 + ocol < in.Dv ? (orow * o_tok + dv0 + ocol) * 2 : NOWHERE;
    const int at_s = (wv * KB * 64 + lane) * 16, at_n = WALK_D * WALK_D * 2 + (wv * 256 + lane) * 16;
    if (chunks > 0) {
        loader.start(a, (const bf16_t *)in.v, in.v_tok, in.v_head, h, hk, s0, L, slot0, chunks);
        loader.fetch(0, x);
        loader.put(x, tiles[0]);
        __syncthreads();
    }
#pragma unroll 1
    for (int i = 0; i < chunks; ++i) {
        DeltaTiles &t = tiles[i & 1];
        loader.fetch(min(i + 1, chunks - 1), x);
        const buffer_t save = buffer_of(ps, a.saved_bytes);
        // K S0, and S0^T Q^T
        f32x4 r[4], o[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) r[m] = o[m] = zero4();
#pragma unroll
        for (int s = 0; s < KB; ++s) {
            bf16x8 sh, sl;
            split8(st[s][0], st[s][1], sh, sl);
            if (SAVE) buf_put16_past(save, at_s + s * 1024, __builtin_bit_cast(u32x4, sh));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const bf16x8 kf = frag_rows(t.k, KS, 16 * m, 32 * s), qf = frag_rows(t.q, KS, 16 * m, 32 * s);
                r[m] = mfma16(kf, sl, r[m]);
                o[m] = mfma16(sl, qf, o[m]);
                r[m] = mfma16(kf, sh, r[m]);
                o[m] = mfma16(sh, qf, o[m]);
            }
        }
        // R = beta (V - e^G K S0)
        bf16x8 rh[2], rl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 beta[2], f[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r0 = 32 * s + 16 * hh + 4 * g4;
                beta[hh] = row_factors(t.f, DELTA_BETA, r0);
                f[hh] = row_factors(t.f, DELTA_EG, r0) * row_factors(t.f, DELTA_RK, r0);
            }
            const bf16x8 v = frag_column(t.v, VS, 32 * s, dv0);
            split8((lower4(v) - r[2 * s] * f[0]) * beta[0], (upper4(v) - r[2 * s + 1] * f[1]) * beta[1], rh[s], rl[s]);
        }
        // N = T R
        f32x4 n[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 across;
            n[m] = across = zero4();
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const bf16x8 th = plane_block<false>(t.tp, PLANE_TH, m, s), tl = plane_block<false>(t.tp, PLANE_TL, m, s);
                n[m] = mfma16(th, rl[s], n[m]);
                n[m] = mfma16(tl, rh[s], n[m]);
                n[m] = mfma16(th, rh[s], n[m]);
                if (SAVE) {
                    across = mfma16(rl[s], th, across);
                    across = mfma16(rh[s], tl, across);
                    across = mfma16(rh[s], th, across);
                }
            }
            if (SAVE) {
                const u32x2 yh = hi4(across), yl = lo4(across, yh);
                buf_put16_past(save, at_n + m * 1024, u32x4{yh[0], yh[1], yl[0], yl[1]});
            }
        }
        // S1 = e^G_63 S0 + K^T e^(G_63 - G) N
        bf16x8 nh[2], nl[2], mh[2], ml[2];
        const float end = t.f[DELTA_EG * 64 + 63];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 f[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) f[hh] = row_factors(t.f, DELTA_EC, 32 * s + 16 * hh + 4 * g4) * row_factors(t.f, DELTA_RK, 32 * s + 16 * hh + 4 * g4);
            split8(n[2 * s], n[2 * s + 1], nh[s], nl[s]);
            split8(n[2 * s] * f[0], n[2 * s + 1] * f[1], mh[s], ml[s]);
        }
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                st[k][hh] *= end;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 kt = frag_column(t.k, KS, 32 * s, 32 * k + 16 * hh);
                    st[k][hh] = mfma16(kt, ml[s], st[k][hh]);
                    st[k][hh] = mfma16(kt, mh[s], st[k][hh]);
                }
            }
        // O^T = scale e^G S0^T Q^T + N^T P^T, through V's place (the wave's own columns)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float f = t.f[DELTA_EG * 64 + 16 * m + l16] * t.f[DELTA_RQ * 64 + 16 * m + l16];
            o[m] *= f;
#pragma unroll
            for (int s = 0; s <= m / 2; ++s) {
                const bf16x8 ph = plane_block<false>(t.tp, PLANE_PH, m, s), pl = plane_block<false>(t.tp, PLANE_PL, m, s);
                o[m] = mfma16(nl[s], ph, o[m]);
                o[m] = mfma16(nh[s], pl, o[m]);
                o[m] = mfma16(nh[s], ph, o[m]);
            }
            put4(t.v + (16 * m + l16) * VS + dv0 + 4 * g4, hi4(o[m]));
        }
        wave_sync();
        const buffer_t out = rows_buffer(po, o_tok, min(64, rows_all - 64 * i), in.Dv);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            buf_put16(out, further(at_o, e * 32 * o_tok * 2), *reinterpret_cast<const u32x4_any *>(t.v + (orow + e * 32) * VS + dv0 + ocol));
        ps += SAVE ? step_s : 0;
        po += (int64_t)o_tok * 128;
        loader.put(x, tiles[(i + 1) & 1]);
        __syncthreads();
    }
    if (a.final)
        each_state([&](int s, int hh, int v, int k) {
            if (k < in.Dk && dv0 + l16 < in.Dv) a.final[cell + (int64_t)k * in.Dv] = st[s][hh][v];
        });
}

__global__ __launch_bounds__(64 * WALK_W, 2) void dsa_delta_back_kernel(DeltaArgs a) {
    constexpr int KB = WALK_KB, KS = WALK_KS, VS = WALK_KS;
    __shared__ __align__(16) DeltaTiles tiles[2];
    const dsa_delta_args &in = a.in;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
    int64_t unit;
    int block, slot0, chunks, s0, L;
    if (a.choose && delta_form(a) != DELTA_HEAD) return;
    if (!delta_walk_unit(blockIdx.x, 1, (int64_t)in.N * in.Hv, unit, block)) return;
    const int h = (int)(unit % in.Hv), seg = delta_longest(in.cu, in.N, (int)(unit / in.Hv)), hk = h / (in.Hv / in.Hk), dv0 = 16 * wv;
    delta_segment(in.cu, in.N, seg, slot0, chunks, s0, L);
    chunks = min(chunks, a.slots - slot0);
    s0 = max(s0, 0);
    f32x4 st[KB][2];                                 // dS
    const int64_t cell = ((int64_t)seg * in.Hv + h) * in.Dk * in.Dv + dv0 + l16;
    each_state([&](int s, int hh, int v, int k) {
        st[s][hh][v] = a.dfinal && k < in.Dk && dv0 + l16 < in.Dv ? a.dfinal[cell + (int64_t)k * in.Dv] : 0.f;
    });
    loads_done();
    DeltaLoader<true> loader;
    DeltaAhead x;
    const int64_t last = slot0 + chunks - 1;
    char *pb = a.back + (last * in.Hv + h) * a.back_bytes, *pv = (char *)(a.dv + ((s0 + 64 * (int64_t)(chunks - 1)) * in.Hv + h) * in.Dv);
    const int64_t step_b = (int64_t)in.Hv * a.back_bytes;
    const int o_tok = in.Hv * in.Dv, rows_all = min(L, in.T - s0);
    const int orow = lane / 2, ocol = lane % 2 * 8, at_o = dv0 + ocol < in.Dv ? (orow * o_tok + dv0 + ocol) * 2 : NOWHERE;
    const int at_s = (wv * KB * 64 + lane) * 16, at_n = WALK_D * WALK_D * 2 + (wv * 256 + lane) * 16;
    if (chunks > 0) {
        loader.start(a, a.dout, o_tok, in.Dv, h, hk, s0, L, slot0, chunks);
        loader.fetch(chunks - 1, x);
        loader.put(x, tiles[(chunks - 1) & 1]);
        __syncthreads();
    }
#pragma unroll 1
    for (int i = chunks - 1; i >= 0; --i) {
        DeltaTiles &t = tiles[i & 1];
        loader.fetch(max(i - 1, 0), x);
        const buffer_t back = buffer_of(pb, a.back_bytes);
        // dN = e^(G_63 - G) K dS1 + P^T dO
        f32x4 r[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) r[m] = zero4();
#pragma unroll
        for (int s = 0; s < KB; ++s) {
            bf16x8 sh, sl;
            split8(st[s][0], st[s][1], sh, sl);
            buf_put16_past(back, at_s + s * 1024, __builtin_bit_cast(u32x4, sh));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const bf16x8 kf = frag_rows(t.k, KS, 16 * m, 32 * s);
                r[m] = mfma16(kf, sl, r[m]);
                r[m] = mfma16(kf, sh, r[m]);
            }
        }
        bf16x8 of[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) of[s] = frag_column(t.v, VS, 32 * s, dv0);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x4 f = row_factors(t.f, DELTA_EC, 16 * m + 4 * g4) * row_factors(t.f, DELTA_RK, 16 * m + 4 * g4);
            r[m] *= f;
#pragma unroll
            for (int s = m / 2; s < 2; ++s) {
                const bf16x8 ph = plane_block<true>(t.tp, PLANE_PH, m, s), pl = plane_block<true>(t.tp, PLANE_PL, m, s);
                r[m] = mfma16(pl, of[s], r[m]);
                r[m] = mfma16(ph, of[s], r[m]);
            }
        }
        bf16x8 nh[2], nl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) split8(r[2 * s], r[2 * s + 1], nh[s], nl[s]);
        // dR = T^T dN, and transposed; dV = beta dR through dO's place (the wave's own columns)
        f32x4 y[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 across;
            y[m] = across = zero4();
#pragma unroll
            for (int s = m / 2; s < 2; ++s) {
                const bf16x8 th = plane_block<true>(t.tp, PLANE_TH, m, s), tl = plane_block<true>(t.tp, PLANE_TL, m, s);
                y[m] = mfma16(th, nl[s], y[m]);
                across = mfma16(nl[s], th, across);
                y[m] = mfma16(tl, nh[s], y[m]);
                across = mfma16(nh[s], tl, across);
                y[m] = mfma16(th, nh[s], y[m]);
                across = mfma16(nh[s], th, across);
            }
            const float beta = t.f[DELTA_BETA * 64 + 16 * m + l16];
            const u32x2 yh = hi4(across), yl = lo4(across, yh);
            buf_put16_past(back, at_n + m * 1024, u32x4{yh[0], yh[1], yl[0], yl[1]});
            put4(t.v + (16 * m + l16) * VS + dv0 + 4 * g4, hi4(across * beta));
        }
        wave_sync();
        const buffer_t dvs = rows_buffer(pv, o_tok, min(64, rows_all - 64 * i), in.Dv);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            buf_put16(dvs, further(at_o, e * 32 * o_tok * 2), *reinterpret_cast<const u32x4_any *>(t.v + (orow + e * 32) * VS + dv0 + ocol));
        // dS0 = e^G_63 dS1 + Q^T scale e^G dO - K^T beta e^G dR
        bf16x8 uh[2], ul[2], wh[2], wl[2];
        const float end = t.f[DELTA_EG * 64 + 63];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 fk[2], fq[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r0 = 32 * s + 16 * hh + 4 * g4;
                const f32x4 eg = row_factors(t.f, DELTA_EG, r0);
                fk[hh] = -(eg * row_factors(t.f, DELTA_BETA, r0) * row_factors(t.f, DELTA_RK, r0));
                fq[hh] = eg * row_factors(t.f, DELTA_RQ, r0);
            }
            split8(y[2 * s] * fk[0], y[2 * s + 1] * fk[1], uh[s], ul[s]);
            split8(lower4(of[s]) * fq[0], upper4(of[s]) * fq[1], wh[s], wl[s]);
        }
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                st[k][hh] *= end;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 kt = frag_column(t.k, KS, 32 * s, 32 * k + 16 * hh), qt = frag_column(t.q, KS, 32 * s, 32 * k + 16 * hh);
                    st[k][hh] = mfma16(kt, ul[s], st[k][hh]);
                    st[k][hh] = mfma16(qt, wl[s], st[k][hh]);
                    st[k][hh] = mfma16(kt, uh[s], st[k][hh]);
                    st[k][hh] = mfma16(qt, wh[s], st[k][hh]);
                }
            }
        pb -= step_b;
        pv -= (int64_t)o_tok * 128;
        loader.put(x, tiles[(i + 1) & 1]);
        __syncthreads();
    }
    if (a.dinitial)
        each_state([&](int s, int hh, int v, int k) {
            if (k < in.Dk && dv0 + l16 < in.Dv) a.dinitial[cell + (int64_t)k * in.Dv] = st[s][hh][v];
        });
}

extern "C" void dsa_launch_delta_chain(const DeltaArgs *a, int form, int save, hipStream_t stream);
extern "C" void dsa_launch_delta_chain_back(const DeltaArgs *a, int form, hipStream_t stream);
// The forms that lengths unknown to the host leave: all chunks are those of one longest sequence at the least, of N at the most.  Short batches take one that may not be
// the best rather than launches for nothing; batches of 512 walks leave DELTA_ONE out, and of 1024 all but DELTA_HEAD (33 sequences: 8 us a launch of 310 for nothing).  That goes by
// the numbers alone, and loses where one sequence outlasts the rest: forward and backward, 32 heads, one of 8192 rows beside 32 of 64 takes 1911 us where the long one alone takes
// 749, one of 2048 among 63 empty ones 469 where it takes 200.
static int delta_forms(DeltaArgs &a, int (&forms)[3]) {
    const int64_t least = a.in.Hv, most = (int64_t)a.in.N * a.in.Hv;
    const int low = delta_form_of(a, least, 1), high = delta_form_of(a, most, 1), many = a.Dkp == 128 && a.Dvp == 128 && most >= 512;
    int n = 0;
    a.maybe_one = low == DELTA_ONE && (high == DELTA_ONE || most < 512);
    if ((a.in.T < 2048 || (many && most >= 1024)) && low != high) forms[n++] = many ? DELTA_HEAD : DELTA_TWO;
    else
        for (int f = low == DELTA_ONE && !a.maybe_one ? DELTA_TWO : low; f <= high; ++f) forms[n++] = f;
    a.choose = n > 1;
    return n;
}
extern "C" void dsa_launch_delta_walk(const DeltaArgs *args, int save, hipStream_t stream) {
    DeltaArgs a = *args;
    int forms[3];
    const int n = delta_forms(a, forms);
    const dim3 walks((unsigned)(((int64_t)a.in.N * a.in.Hv + 7) / 8 * 8));
    for (int i = 0; i < n; ++i) {
        if (forms[i] != DELTA_HEAD) dsa_launch_delta_chain(&a, forms[i], save, stream);
        else if (save) hipLaunchKernelGGL(dsa_delta_walk_kernel<true>, walks, dim3(64 * WALK_W), 0, stream, a);
        else hipLaunchKernelGGL(dsa_delta_walk_kernel<false>, walks, dim3(64 * WALK_W), 0, stream, a);
    }
}
extern "C" void dsa_launch_delta_back(const DeltaArgs *args, hipStream_t stream) {
    DeltaArgs a = *args;
    int forms[3];
    const int n = delta_forms(a, forms);
    for (int i = 0; i < n; ++i) {
        if (forms[i] != DELTA_HEAD) dsa_launch_delta_chain_back(&a, forms[i], stream);
        else hipLaunchKernelGGL(dsa_delta_back_kernel, dim3((unsigned)(((int64_t)a.in.N * a.in.Hv + 7) / 8 * 8)), dim3(64 * WALK_W), 0, stream, a);
    }
}
