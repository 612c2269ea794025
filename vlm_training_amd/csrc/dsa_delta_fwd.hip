// Gated delta rule, chunked forward: the chunks' own matrices, then the walk of the state (see dsa_delta.h for the formulas).
#include "dsa_delta.h"

// ---- T and P of every chunk; one workgroup per chunk and key head, its value heads in turn --------------------------------------------------
// The products of q and k rows are shared by the key head's value heads and stay in registers (wave w: columns 16 w .. of the transposed
// products, so that a lane holds four neighbours of a row of P and A).  T by blocks of 16 rows: the diagonal blocks by substitution, a wave
// each, then T_ij = -T_ii sum_k A_ik T_kj from the diagonal outwards, in fp32 (mfma of 16x16x4): a run of equal keys, whose A is a full triangle of
// ones, has a T of ones and minus ones that powers of A would lose in cancellation.
template <int DK>
__global__ __launch_bounds__(256, 4) void dsa_delta_prep_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, FS = 68;
    __shared__ __align__(16) float am[64 * FS], tm[64 * FS], ms[4][16 * 17], rk[64], rq[64], gh[64], gl[64], bt[64];
    bf16_t *const ks = (bf16_t *)am, *const qs = (bf16_t *)tm;               // K and Q, before their products are there
    static_assert(64 * KS * 2 <= 64 * FS * 4, "a tile of K lies in A's place");
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = tid & 15, g4 = (tid & 63) >> 4;
    const int slot = blockIdx.x, hk = blockIdx.y, rep = in.Hv / in.Hk;
    DeltaChunk c;
    if (!delta_locate(in.cu, in.N, in.T, slot, c)) {
        // rows behind the last sequence: zeros
        const int64_t r0 = (int64_t)max(in.cu[in.N], 0) + 64 * (int64_t)c.index;
        for (int r = 0; r < 64 && r0 + r < in.T; ++r)
            for (int i = tid; i < rep * in.Dv; i += 256) a.out[((r0 + r) * in.Hv + hk * rep) * in.Dv + i] = (bf16_t)0.f;
        return;
    }
    tile_copy<DK>(ks, KS, (const bf16_t *)in.k + c.row0 * in.k_tok + hk * in.k_head, in.k_tok, c.rows, in.Dk);
    tile_copy<DK>(qs, KS, (const bf16_t *)in.q + c.row0 * in.q_tok + hk * in.q_head, in.q_tok, c.rows, in.Dk);
    __syncthreads();
    {   // 1/|k|, scale/|q|: four threads per row
        const int r = tid >> 2, c0 = (tid & 3) * (DK / 4);
        float sk = 0.f, sq = 0.f;
        for (int i = 0; i < DK / 4; ++i) {
            const float x = (float)ks[r * KS + c0 + i], y = (float)qs[r * KS + c0 + i];
            sk += x * x;
            sq += y * y;
        }
        sk += __shfl_xor(sk, 1, 64); sk += __shfl_xor(sk, 2, 64);
        sq += __shfl_xor(sq, 1, 64); sq += __shfl_xor(sq, 2, 64);
        if ((tid & 3) == 0) {
            rk[r] = in.l2_norm ? rsqrtf(sk + 1e-6f) : 1.f;
            rq[r] = in.l2_norm ? in.scale * rsqrtf(sq + 1e-6f) : in.scale;
        }
    }
    f32x4 kk[4], qk[4];                                  // [tile of 16 rows j][j = 4 g4 + v], row i = 16 wv + l16
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        kk[t] = qk[t] = zero4();
        if (t <= wv) {
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) {
                const bf16x8 kj = frag_n(ks, KS, 16 * t, 32 * s);
                kk[t] = mfma16(kj, frag_n(ks, KS, 16 * wv, 32 * s), kk[t]);
                qk[t] = mfma16(kj, frag_n(qs, KS, 16 * wv, 32 * s), qk[t]);
            }
        }
    }
    for (int u = 0; u < rep; ++u) {
        const int lane = fresh_lane(), l16 = lane & 15, g4 = lane >> 4, tid = 64 * wv + lane, i = 16 * wv + l16;
        const int h = hk * rep + u;
        const int64_t p = (int64_t)slot * in.Hv + h;
        __syncthreads();                                 // (the previous head's LDS has been read)
        float *const rows = (float *)(a.mats + p * a.mats_bytes);
        if (wv == 0) {
            const bool live = lane < c.rows;
            const int64_t t = c.row0 + (live ? lane : 0);
            double g = live ? (double)delta_gate(in, t, h) : 0.;
            const float beta = live ? delta_beta(in, t, h) : 0.f;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const double x = __shfl_up(g, m, 64);
                if (lane >= m) g += x;
            }
            const double end = __shfl(g, 63, 64);
            const float h0 = (float)g;
            gh[lane] = h0;
            gl[lane] = (float)(g - (double)h0);
            bt[lane] = beta;
            rows[DELTA_EG * 64 + lane] = expf((float)g);
            rows[DELTA_EC * 64 + lane] = expf((float)(end - g));
            rows[DELTA_BETA * 64 + lane] = beta;
            rows[DELTA_RK * 64 + lane] = rk[lane];
            rows[DELTA_RQ * 64 + lane] = rq[lane];
            rows[DELTA_GH * 64 + lane] = h0;
            rows[DELTA_GL * 64 + lane] = gl[lane];
        }
        __syncthreads();
        bf16_t *const tg = (bf16_t *)(a.mats + p * a.mats_bytes + DELTA_T), *const pm = tg + a.planes * 4096;
        f32x4 px[4];
        const float gi = gh[i], gi_lo = gl[i], fx = rq[i], fy = bt[i] * rk[i];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 x = zero4(), y = zero4();
            if (t <= wv) {
                const int j0 = 16 * t + 4 * g4;
                const f32x4 dh = gi - *reinterpret_cast<const f32x4 *>(gh + j0), dl = gi_lo - *reinterpret_cast<const f32x4 *>(gl + j0), r = *reinterpret_cast<const f32x4 *>(rk + j0);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float e = delta_decay(dh[v] + dl[v]) * r[v];
                    x[v] = j0 + v <= i ? e * fx * qk[t][v] : 0.f;
                    y[v] = j0 + v < i ? e * fy * kk[t][v] : 0.f;
                }
            }
            px[t] = x;
            *reinterpret_cast<f32x4 *>(am + i * FS + 16 * t + 4 * g4) = y;
            if (t > wv) *reinterpret_cast<f32x4 *>(tm + i * FS + 16 * t + 4 * g4) = zero4();
        }
        wave_sync();                                     // (a diagonal block is its own wave's)
        {
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float s = r == l16 ? 1.f : 0.f;
#pragma unroll
                for (int k = 0; k < r; k += 4) {
                    const f32x4 y = *reinterpret_cast<const f32x4 *>(am + (16 * wv + r) * FS + 16 * wv + k);
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (k + v < r) s -= y[v] * x[k + v];
                }
                x[r] = s;
            }
            if (g4 == 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r) tm[(16 * wv + r) * FS + 16 * wv + l16] = x[r];
            }
        }
        for (int d = 1; d < 4; ++d) {
            __syncthreads();
            if (wv + d < 4) {                            // block (bi, bj)
                const int bi = wv + d, bj = wv;
                f32x4 m = zero4();
                for (int b = bj; b < bi; ++b)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        m = __builtin_amdgcn_mfma_f32_16x16x4f32(am[(16 * bi + l16) * FS + 16 * b + 4 * s + g4], tm[(16 * b + 4 * s + g4) * FS + 16 * bj + l16], m, 0, 0, 0);
#pragma unroll
                for (int v = 0; v < 4; ++v) ms[wv][(4 * g4 + v) * 17 + l16] = m[v];
                wave_sync();
                f32x4 r = zero4();
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    r = __builtin_amdgcn_mfma_f32_16x16x4f32(tm[(16 * bi + l16) * FS + 16 * bi + 4 * s + g4], ms[wv][(4 * s + g4) * 17 + l16], r, 0, 0, 0);
#pragma unroll
                for (int v = 0; v < 4; ++v) tm[(16 * bi + 4 * g4 + v) * FS + 16 * bj + l16] = -r[v];
            }
        }
        __syncthreads();
        // P through A's place, then the planes in the order of their fragments
#pragma unroll
        for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4 *>(am + i * FS + 16 * t + 4 * g4) = px[t];
        __syncthreads();
        auto plane = [&](bf16_t *to, int at, f32x4 x, f32x4 y) __attribute__((always_inline)) {
            const u32x2 xh = hi4(x), yh = hi4(y), xl = lo4(x, xh), yl = lo4(y, yh);
            *reinterpret_cast<u32x4_any *>(to + at) = u32x4{xh[0], xh[1], yh[0], yh[1]};
            *reinterpret_cast<u32x4_any *>(to + 4096 + at) = u32x4{xl[0], xl[1], yl[0], yl[1]};
        };
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int at = tid + 256 * e, r = at / 128 * 16 + l16, c0 = at / 64 % 2 * 32 + 8 * g4;
            // (the quarter that is all zeros is neither written nor read)
            if (r < 32 && c0 >= 32) {}
            else {
                plane(tg, at * 8, *reinterpret_cast<const f32x4 *>(tm + r * FS + c0), *reinterpret_cast<const f32x4 *>(tm + r * FS + c0 + 4));
                plane(pm, at * 8, *reinterpret_cast<const f32x4 *>(am + r * FS + c0), *reinterpret_cast<const f32x4 *>(am + r * FS + c0 + 4));
            }
            if (a.planes > 2 && !(r >= 32 && c0 < 32)) { // transposed
                f32x4 x[2], y[2];
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    x[v / 4][v % 4] = tm[(c0 + v) * FS + r];
                    y[v / 4][v % 4] = am[(c0 + v) * FS + r];
                }
                plane(tg + 2 * 4096, at * 8, x[0], x[1]);
                plane(pm + 2 * 4096, at * 8, y[0], y[1]);
            }
        }
    }
}

// ---- the walk: one workgroup per sequence, value head and 16 NC columns of the state -------------------------------------------------------
// Wave w has rows 16 w .. of the chunk and rows Dk/4 w .. of the state, which stay in registers (fp32) from the first chunk to the last.  A chunk is a chain
// of three products over the same columns - K S0 (and Q S0), T R, K^T N (and P N) - so their results go through LDS to the other waves, a barrier each; they are
// formed transposed (lane: its row, four neighbouring columns), which makes every factor of a row one register and every access 8 or 16 bytes.
// Rows of K, Q, T and P are needed by their own wave alone (K by all of them as K^T): T and P come as fragments straight into registers, rows of K, Q and V
// 16 bytes a lane through the wave's own part of LDS.  The next chunk's loads go out as soon as a register has been read.  (With waves side by side over the columns instead, each of them read all of K, Q, T, P from LDS: 5.3 us per chunk.)
template <int DK, int NC> struct WalkRows {
    bf16x8 k[DK / 32], q[DK / 32], th[2], tl[2], ph[2], pl[2];
    Piece<4 * NC> v;
    float eg, ec, beta, rk, rq, end;
};
template <int DK, int NC, bool SAVE>
__global__ __launch_bounds__(256, 2) void dsa_delta_walk_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, RS = DELTA_RS, NT = DK / 64;
    __shared__ bf16_t ks[2][64 * KS], sh[16 * NC * KS], sl[16 * NC * KS], rh[64 * RS], rl[64 * RS], pool[4 * 64 * RS];
    // N and e^(G_63 - G)/|k| N as hi, lo; Q before they are there
    bf16_t *const nh = pool, *const nl = pool + 64 * RS, *const mh = pool + 128 * RS, *const ml = pool + 192 * RS, *const qt = pool;
    static_assert(KS <= 4 * RS, "Q lies in N's place");
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g4 = lane >> 4, row = 16 * wv + l16;
    int64_t unit;
    int block, slot0, chunks, s0, L;
    if (!delta_walk_unit(blockIdx.x, a.Dvp / (16 * NC), (int64_t)in.N * in.Hv, unit, block)) return;
    const int h = (int)(unit % in.Hv), seg = (int)(unit / in.Hv), hk = h / (in.Hv / in.Hk), dv0 = 16 * NC * block;
    delta_segment(in.cu, in.N, seg, slot0, chunks, s0, L);
    chunks = min(chunks, a.slots - slot0);
    s0 = max(s0, 0);
    f32x4 st[NT][NC];                                    // S[dk = 16 (NT wv + t) + 4 g4 + v][dv0 + 16 c + l16]
    const int64_t cell = ((int64_t)seg * in.Hv + h) * in.Dk * in.Dv + dv0 + l16;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int k = 16 * (NT * wv + t) + 4 * g4 + v;
                st[t][c][v] = a.initial && k < in.Dk && dv0 + 16 * c + l16 < in.Dv ? a.initial[cell + (int64_t)k * in.Dv + 16 * c] : 0.f;
            }
    loads_done();
    // offsets of this lane, in bytes
    constexpr int LPR = DK / 8, RPI = 64 / LPR;          // lanes to a row of K or Q, rows to a load
    const int rrow = 16 * wv + lane / LPR, rcol = lane % LPR * 8, vrow = 16 * wv + lane / 4, vcol = lane % 4 * 4 * NC;
    const int at_k = rcol < in.Dk ? (rrow * (int)in.k_tok + rcol) * 2 : NOWHERE, at_q = rcol < in.Dk ? (rrow * (int)in.q_tok + rcol) * 2 : NOWHERE;
    const int at_v = dv0 + vcol < in.Dv ? (vrow * (int)in.v_tok + dv0 + vcol) * 2 : NOWHERE, at_o = dv0 + vcol < in.Dv ? (vrow * in.Hv * in.Dv + dv0 + vcol) * 2 : NOWHERE;
    const int at_t = wv * 2048 + lane * 16, at_t1 = wv >= 2 ? at_t + 1024 : NOWHERE;       // (rows of T and P end at the diagonal)
    const int at_s = (dv0 * DK + (wv * 64 + lane) * 4 * NT) * 2, at_n = a.Dvp * DK * 2 + (dv0 / 16 * 256 + wv * 64 + lane) * 16;
    // where the next chunk to be fetched, and the one at hand, lie; a chunk further they are a fixed number of bytes on
    const int64_t first = (int64_t)slot0 * in.Hv + h;
    const char *pk = (const char *)in.k + (s0 * in.k_tok + hk * in.k_head) * 2, *pq = (const char *)in.q + (s0 * in.q_tok + hk * in.q_head) * 2;
    const char *pv = (const char *)in.v + (s0 * in.v_tok + h * in.v_head) * 2, *pm = a.mats + first * a.mats_bytes;
    char *ps = a.saved + first * a.saved_bytes, *po = (char *)(a.out + ((int64_t)s0 * in.Hv + h) * in.Dv);
    const int64_t step_m = (int64_t)in.Hv * a.mats_bytes, step_s = (int64_t)in.Hv * a.saved_bytes;
    const int step_k = (int)in.k_tok * 128, step_q = (int)in.q_tok * 128, step_v = (int)in.v_tok * 128, step_o = in.Hv * in.Dv * 128;
    const int rows_all = min(L, in.T - s0);              // (one chunk after the other takes its 64 of them)
    typedef WalkRows<DK, NC> Rows;
    auto fetch_rows = [&](int i, Rows &w) __attribute__((always_inline)) {
        const int n = min(64, rows_all - 64 * i);
        const buffer_t k = rows_buffer(pk, (int)in.k_tok, n, in.Dk), q = rows_buffer(pq, (int)in.q_tok, n, in.Dk), v = rows_buffer(pv, (int)in.v_tok, n, in.Dv);
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) {              
            w.k[s] = buf16(k, further(at_k, s * RPI * (int)in.k_tok * 2));
            w.q[s] = buf16(q, further(at_q, s * RPI * (int)in.q_tok * 2));
        }
        w.v = buf_piece<4 * NC>(v, at_v);
        const bool on = i + 1 < chunks;                  // (the last one is fetched again: behind a branch, waits would be for every load in flight)
        pk += on ? step_k : 0;
        pq += on ? step_q : 0;
        pv += on ? step_v : 0;
    };
    auto fetch_t = [&](Rows &w) __attribute__((always_inline)) {
        const buffer_t m = buffer_of(pm, a.mats_bytes);
        w.th[0] = buf16(m, at_t, DELTA_T);
        w.tl[0] = buf16(m, at_t, DELTA_T + DELTA_PLANE);
        w.th[1] = buf16(m, at_t1, DELTA_T);
        w.tl[1] = buf16(m, at_t1, DELTA_T + DELTA_PLANE);
    };
    auto fetch_p = [&](int i, Rows &w) __attribute__((always_inline)) {
        const buffer_t m = buffer_of(pm, a.mats_bytes);
        const int p = DELTA_T + a.planes * DELTA_PLANE;
        w.ph[0] = buf16(m, at_t, p);
        w.pl[0] = buf16(m, at_t, p + DELTA_PLANE);
        w.ph[1] = buf16(m, at_t1, p);
        w.pl[1] = buf16(m, at_t1, p + DELTA_PLANE);
        w.eg = buf4(m, DELTA_EG * 256 + row * 4);
        w.ec = buf4(m, DELTA_EC * 256 + row * 4);
        w.beta = buf4(m, DELTA_BETA * 256 + row * 4);
        w.rk = buf4(m, DELTA_RK * 256 + row * 4);
        w.rq = buf4(m, DELTA_RQ * 256 + row * 4);
        w.end = buf4(m, DELTA_EG * 256 + 252);
        pm += i + 1 < chunks ? step_m : 0;
    };
    auto chunk = [&](int i, Rows &x, bf16_t *kt) __attribute__((always_inline)) {
        const int ahead = min(i + 1, chunks - 1);
        // S0 as [dv][dk], K as it is
        const buffer_t save = buffer_of(ps, a.saved_bytes);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            Piece<4 * NT> all;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int at = (16 * c + l16) * KS + 16 * (NT * wv + t) + 4 * g4;
                const u32x2 y = hi4(st[t][c]);
                put4(sh + at, y);
                put4(sl + at, lo4(st[t][c], y));
                all.x[2 * t] = y[0];
                all.x[2 * t + 1] = y[1];
            }
            if (SAVE) buf_put_piece<4 * NT>(save, at_s + c * 32 * DK, all);
        }
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) *reinterpret_cast<bf16x8 *>(kt + (rrow + s * RPI) * KS + rcol) = x.k[s];
        __syncthreads();
        // Q and V: the wave's own rows
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) *reinterpret_cast<bf16x8 *>(qt + (rrow + s * RPI) * KS + rcol) = x.q[s];
        put_piece<4 * NC>(rh + vrow * RS + vcol, x.v);
        fetch_rows(ahead, x);
        wave_sync();
        f32x4 o[NC], r[NC];                              // [dv = 16 c + 4 g4 + v][row]
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] = r[c] = zero4();
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) {
            const bf16x8 kb = frag_n(kt, KS, 16 * wv, 32 * s), qb = frag_n(qt, KS, 16 * wv, 32 * s);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bf16x8 ah = frag_n(sh, KS, 16 * c, 32 * s), al = frag_n(sl, KS, 16 * c, 32 * s);
                r[c] = mfma16(al, kb, r[c]);
                o[c] = mfma16(al, qb, o[c]);
                r[c] = mfma16(ah, kb, r[c]);
                o[c] = mfma16(ah, qb, o[c]);
            }
        }
        const float f = x.eg * x.rk;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = row * RS + 16 * c + 4 * g4;
            put_split4(rh + at, rl + at, (up4(*reinterpret_cast<const u32x2_any *>(rh + at)) - r[c] * f) * x.beta);
        }
        __syncthreads();
        // N^T = R^T T^T
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            f32x4 y = zero4();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s == 1 && wv < 2) continue;
                const bf16x8 ah = frag_t(rh, RS, 32 * s, 16 * c), al = frag_t(rl, RS, 32 * s, 16 * c);
                y = mfma16(al, x.th[s], y);
                y = mfma16(ah, x.tl[s], y);
                y = mfma16(ah, x.th[s], y);
            }
            const int at = row * RS + 16 * c + 4 * g4;
            const u32x2 yh = hi4(y), yl = lo4(y, yh);
            put4(nh + at, yh);
            put4(nl + at, yl);
            put_split4(mh + at, ml + at, y * (x.ec * x.rk));
            if (SAVE) buf_put16(save, at_n + c * 4096, u32x4{yh[0], yh[1], yl[0], yl[1]});
        }
        fetch_t(x);
        __syncthreads();
        // S1 = e^G_63 S0 + K^T e^(G_63 - G) N
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c) st[t][c] *= x.end;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 bh[NC], bl[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                bh[c] = frag_t(mh, RS, 32 * s, 16 * c);
                bl[c] = frag_t(ml, RS, 32 * s, 16 * c);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bf16x8 ka = frag_t(kt, KS, 32 * s, 16 * (NT * wv + t));
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    st[t][c] = mfma16(ka, bl[c], st[t][c]);
                    st[t][c] = mfma16(ka, bh[c], st[t][c]);
                }
            }
        }
        // O^T = scale e^G S0^T Q^T + N^T P^T
        const buffer_t out = rows_buffer(po, in.Hv * in.Dv, min(64, rows_all - 64 * i), in.Dv);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            o[c] *= x.eg * x.rq;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s == 1 && wv < 2) continue;
                const bf16x8 ah = frag_t(nh, RS, 32 * s, 16 * c), al = frag_t(nl, RS, 32 * s, 16 * c);
                o[c] = mfma16(al, x.ph[s], o[c]);
                o[c] = mfma16(ah, x.pl[s], o[c]);
                o[c] = mfma16(ah, x.ph[s], o[c]);
            }
            put4(rh + row * RS + 16 * c + 4 * g4, hi4(o[c]));
        }
        wave_sync();
        buf_put_piece<4 * NC>(out, at_o, get_piece<4 * NC>(rh + vrow * RS + vcol));
        fetch_p(ahead, x);
        po += step_o;
        if (SAVE) ps += step_s;
    };
    Rows x;
    if (chunks > 0) {
        fetch_rows(0, x);
        fetch_t(x);
        fetch_p(0, x);
        for (int i = 0; i < chunks; ++i) chunk(i, x, ks[i & 1]);
    }
    if (a.final) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int k = 16 * (NT * wv + t) + 4 * g4 + v;
                    if (k < in.Dk && dv0 + 16 * c + l16 < in.Dv) a.final[cell + (int64_t)k * in.Dv + 16 * c] = st[t][c][v];
                }
    }
}

// ---- one token for each of B requests: the state passes through registers once ----------------------------------------------------------------
// o = scale (e^g S^T q + (k.q) d), S += k d^T with d = beta (v - e^g S^T k): both sums over Dk come from the state as it was read, so it is read
// and written once.  A workgroup takes 32 columns of one head's state (a row of them is 128 bytes, 8 lanes of 16), 32 rows at a time.
// Bound by memory.
template <int DK>
__global__ __launch_bounds__(256) void dsa_delta_step_kernel(dsa_delta_args in, float *state, int64_t state_req, bf16_t *out) {
    constexpr int RPT = DK / 32;                         // rows of the state per thread
    __shared__ float kq[2][DK], sums[2][4][32], ends[3];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int blocks = (in.Dv + 31) / 32;
    const int64_t req = blockIdx.x / blocks / in.Hv;
    const int h = blockIdx.x / blocks % in.Hv, hk = h / (in.Hv / in.Hk), d0 = blockIdx.x % blocks * 32 + tid % 8 * 4, k0 = tid / 8;
    float *const cell = state + req * state_req + (int64_t)h * in.Dk * in.Dv + d0;
    const bool in_d = d0 < in.Dv;
    f32x4 s[RPT];
#pragma unroll
    for (int u = 0; u < RPT; ++u) {
        const int k = k0 + 32 * u;
        s[u] = in_d && k < in.Dk ? *reinterpret_cast<const f32x4 *>(cell + (int64_t)k * in.Dv) : zero4();
    }
    if (wv == 0) {
        float x[DK / 64], y[DK / 64], kk = 0.f, qq = 0.f, dot = 0.f;
#pragma unroll
        for (int u = 0; u < DK / 64; ++u) {
            const int k = lane + 64 * u;
            x[u] = k < in.Dk ? (float)((const bf16_t *)in.k)[req * in.k_tok + hk * in.k_head + k] : 0.f;
            y[u] = k < in.Dk ? (float)((const bf16_t *)in.q)[req * in.q_tok + hk * in.q_head + k] : 0.f;
            kk += x[u] * x[u];
            qq += y[u] * y[u];
            dot += x[u] * y[u];
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            kk += __shfl_xor(kk, m, 64);
            qq += __shfl_xor(qq, m, 64);
            dot += __shfl_xor(dot, m, 64);
        }
        const float rk = in.l2_norm ? rsqrtf(kk + 1e-6f) : 1.f, rq = (in.l2_norm ? rsqrtf(qq + 1e-6f) : 1.f) * in.scale;
#pragma unroll
        for (int u = 0; u < DK / 64; ++u) {
            kq[0][lane + 64 * u] = x[u] * rk;
            kq[1][lane + 64 * u] = y[u] * rq;
        }
        if (lane == 0) {
            ends[0] = dot * rk * rq;
            ends[1] = expf(delta_gate(in, req, h));
            ends[2] = delta_beta(in, req, h);
        }
    }
    __syncthreads();
    f32x4 sk = zero4(), sq = zero4();
#pragma unroll
    for (int u = 0; u < RPT; ++u) {
        sk += s[u] * kq[0][k0 + 32 * u];
        sq += s[u] * kq[1][k0 + 32 * u];
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int m = 8; m < 64; m <<= 1) {
            sk[v] += __shfl_xor(sk[v], m, 64);
            sq[v] += __shfl_xor(sq[v], m, 64);
        }
    if (lane < 8) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            sums[0][wv][lane * 4 + v] = sk[v];
            sums[1][wv][lane * 4 + v] = sq[v];
        }
    }
    __syncthreads();
    const float e = ends[1], beta = ends[2];
    f32x4 d = zero4(), o = zero4();
    if (in_d) {
        const int64_t vi = req * in.v_tok + h * in.v_head + d0;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int col = tid % 8 * 4 + v;
            const float a = (sums[0][0][col] + sums[0][1][col]) + (sums[0][2][col] + sums[0][3][col]);
            const float b = (sums[1][0][col] + sums[1][1][col]) + (sums[1][2][col] + sums[1][3][col]);
            d[v] = beta * ((float)((const bf16_t *)in.v)[vi + v] - e * a);
            o[v] = e * b + ends[0] * d[v];
        }
        if (tid < 8) put4(out + (req * in.Hv + h) * in.Dv + d0, hi4(o));
    }
#pragma unroll
    for (int u = 0; u < RPT; ++u) {
        const int k = k0 + 32 * u;
        if (in_d && k < in.Dk) *reinterpret_cast<f32x4 *>(cell + (int64_t)k * in.Dv) = s[u] * e + d * kq[0][k];
    }
}

// Groups of 16 columns per walk: one where the launch leaves compute units without a walk of two
extern "C" int dsa_delta_columns(const DeltaArgs *a) { return (int64_t)a->in.N * a->in.Hv * (a->Dvp / 32) < 256 ? 1 : 2; }
extern "C" hipError_t dsa_launch_delta_fwd(const DeltaArgs *a, int save, hipStream_t stream) {
    if (a->in.T > 0) {
        const dim3 grid(a->slots, a->in.Hk);
        if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_prep_kernel<64>), grid, dim3(256), 0, stream, *a);
        else hipLaunchKernelGGL((dsa_delta_prep_kernel<128>), grid, dim3(256), 0, stream, *a);
    }
    if (a->in.T > 0 || a->final) {
        const int nc = dsa_delta_columns(a);
        const dim3 walks((unsigned)(((int64_t)a->in.N * a->in.Hv + 7) / 8 * 8 * (a->Dvp / (16 * nc))));
#define DELTA_WALK(DK, NC)                                                                                                    \
    if (save) hipLaunchKernelGGL((dsa_delta_walk_kernel<DK, NC, true>), walks, dim3(256), 0, stream, *a);                      \
    else hipLaunchKernelGGL((dsa_delta_walk_kernel<DK, NC, false>), walks, dim3(256), 0, stream, *a);
        if (a->Dkp == 64 && nc == 1) { DELTA_WALK(64, 1) }
        else if (a->Dkp == 64) { DELTA_WALK(64, 2) }
        else if (nc == 1) { DELTA_WALK(128, 1) }
        else { DELTA_WALK(128, 2) }
    }
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_delta_step(const dsa_delta_args *in, float *state, int64_t state_req, void *out, hipStream_t stream) {
    const int64_t grid = (int64_t)in->T * in->Hv * ((in->Dv + 31) / 32);
    if (grid == 0) return hipSuccess;
    if (in->Dk <= 64) hipLaunchKernelGGL((dsa_delta_step_kernel<64>), dim3((unsigned)grid), dim3(256), 0, stream, *in, state, state_req, (bf16_t *)out);
    else hipLaunchKernelGGL((dsa_delta_step_kernel<128>), dim3((unsigned)grid), dim3(256), 0, stream, *in, state, state_req, (bf16_t *)out);
    return hipGetLastError();
}
