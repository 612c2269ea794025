// Gated delta rule, backward: what the walks (dsa_delta_walk.hip, dsa_delta_chain.hip) leave to do.
// With N = T R, R = beta (V - e^G K S0) of a chunk (dsa_delta.h), from its last chunk to its first:
//     dN = P^T dO + e^(G_63 - G) K dS1      dR = T^T dN      dS0 = e^G_63 dS1 + scale Q^T e^G dO - K^T beta e^G dR
// (the walk, which leaves dS1 and dR of every chunk and dV = beta dR), then all chunks at once
//     dP = dO N^T   dA = -dR N^T   X = scale E dP   Z = beta E dA (below the diagonal)
//     dQ = X K + scale e^G dO S0^T          dK = X^T Q + (Z + Z^T) K + e^(G_63 - G) N dS1^T - beta e^G dR S0^T
//     db = (1 - beta) dR.N                  (dR.N = beta dbeta: both of beta's places, in R and in A, at once)
//     dG_i = q.(X K + scale e^G S0 dO) + k.(Z K - beta e^G S0 dR) - k.(X^T Q + Z^T K + e^(G_63 - G) dS1 N)
//     dG_63 also + all k.(e^(G_63 - G) dS1 N) + e^G_63 <dS1, S0>
// dg is the sum of dG from its row on.  What a pair of rows behind t adds comes in twice with opposite signs, from one X and Z: it leaves 2^-18 of itself.
#include "dsa_delta.h"

// ---- everything that needs one chunk alone: one workgroup per chunk and key head, its value heads in turn --------------------------------
// Wave w has rows 16 w ..; N, dR, X and Z go into their products as hi + lo (where keys repeat, a row of X K is a sum that cancels).  S0 and dS1 go in as one bf16,
// off by 2^-9: dq and dk of 16 384 rows of 32 heads are off by 1.97e-3 of their 2-norm, where rounding them to bf16 makes 1.66e-3 (with N and dR, too, as one bf16
// dk 2.25e-3).  Their low halves would be 64 KB more a chunk and head, 0.57 GB of these rows to write and to read, beside 128 KB that this kernel waits for.  Everything is formed
// transposed (lane: its row, four neighbouring columns), so that a row's factor is one register and its sums stay in four lanes.  dq and dk of the key head
// are summed over its value heads in registers, in that order.  The columns of the values are taken 64 at a time, so that two workgroups share a compute
// unit's LDS and one's loads pass under the other's products; dO and dR are read by their own rows' wave alone.
// 16 384 rows of 32 heads: 0.50 ms for 1.2 GB.  Neither memory (2.4 TB/s) nor the matrix units (a fifth) nor LDS (two fifths) is full: a workgroup waits for its columns'
// loads twice a head, and registers (219 of 256) have no room for them a step earlier (there they spill: 0.6 ms; in phases that leave room, with dO, dR and N
// read twice: 0.73 ms where this form takes 0.49).
template <int DK, int DV>
__global__ __launch_bounds__(256, 2) void dsa_delta_grad_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, TS = DELTA_TS, NT = DK / 16;
    __shared__ bf16_t ks[64 * KS], qs[64 * KS], pool[4 * 64 * TS];
    __shared__ __align__(16) float rows[DELTA_ROWS * 64], dg_row[64], dg_s[64], dots[4];
    bf16_t *const ns = pool, *const ss = pool + 2 * 64 * TS;                                              // N as hi, lo; S0, then dS1: 64 columns of the values
    bf16_t *const xs = pool, *const zs = pool + 2 * 64 * TS;                                              // in their place X and Z as hi, lo
    static_assert(64 * KS <= 2 * 64 * TS, "64 rows of the state lie in two tiles");
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g4 = lane >> 4, row = 16 * wv + l16;
    const int slot = blockIdx.x, hk = blockIdx.y, rep = in.Hv / in.Hk;
    DeltaChunk c;
    if (!delta_locate(in.cu, in.N, in.T, slot, c)) {
        // rows behind the last sequence: zeros; the sums of a chunk that is none: zeros
        const int64_t r0 = (int64_t)max(in.cu[in.N], 0) + 64 * (int64_t)c.index;
        for (int r = 0; r < 64 && r0 + r < in.T; ++r) {
            for (int i = tid; i < in.Dk; i += 256) a.dq[((r0 + r) * in.Hk + hk) * in.Dk + i] = a.dk[((r0 + r) * in.Hk + hk) * in.Dk + i] = (bf16_t)0.f;
            for (int i = tid; i < rep * in.Dv; i += 256) a.dv[((r0 + r) * in.Hv + hk * rep) * in.Dv + i] = (bf16_t)0.f;
            for (int u = tid; u < rep; u += 256) {
                store_any(a.da, (r0 + r) * in.Hv + hk * rep + u, in.a_f32, 0.f);
                store_any(a.db, (r0 + r) * in.Hv + hk * rep + u, in.b_f32, 0.f);
            }
        }
        for (int u = tid; u < rep; u += 256) a.part[(int64_t)(hk * rep + u) * a.slots + slot] = a.part[((int64_t)in.Hv + hk * rep + u) * a.slots + slot] = 0.f;
        return;
    }
    tile_copy<DK>(ks, KS, (const bf16_t *)in.k + c.row0 * in.k_tok + hk * in.k_head, in.k_tok, c.rows, in.Dk);
    tile_copy<DK>(qs, KS, (const bf16_t *)in.q + c.row0 * in.q_tok + hk * in.q_head, in.q_tok, c.rows, in.Dk);
    f32x4 dq[NT], dk[NT];                                // [16 t + 4 g4 + v][row], times scale/|q| and 1/|k|
#pragma unroll
    for (int t = 0; t < NT; ++t) dq[t] = dk[t] = zero4();
    float sum_q = 0.f, sum_k = 0.f;                      // q.dQ and k.dK over the heads, this lane's columns
    const bool live = row < c.rows;
    const bf16_t *const krow = ks + row * KS + 4 * g4, *const qrow = qs + row * KS + 4 * g4;
    auto four = [](const bf16_t *p) __attribute__((always_inline)) { return up4(*reinterpret_cast<const u32x2_any *>(p)); };
    auto dot4 = [](f32x4 x, f32x4 y, float s) __attribute__((always_inline)) { return s + ((x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3])); };
    auto dot8 = [](u32x4 x, u32x4 y, float s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t xi = x[i], yi = y[i];         // (a bit cast of a vector's element itself is compiled as one of element 0)
            s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, xi), __builtin_bit_cast(bf16x2, yi), s, false);
        }
        return s;
    };
    auto over_row = [](float x) __attribute__((always_inline)) { x += __shfl_xor(x, 16, 64); return x + __shfl_xor(x, 32, 64); };
#pragma unroll 1
    for (int u = 0; u < rep; ++u) {
        const int h = hk * rep + u;
        const int64_t p = (int64_t)slot * in.Hv + h;
        const bf16_t *const state = (const bf16_t *)(a.saved + p * a.saved_bytes), *const news = state + DV * DK;
        const bf16_t *const dstate = (const bf16_t *)(a.back + p * a.back_bytes), *const drs = dstate + DV * DK;
        f32x4 x[4], z[4];
        // this head's own parts of q.dQ and k.dK: dG is formed of these alone, so that a head neither loses bits to its neighbours nor takes over their NaN.  own_k: what counts
        // for dG with a plus; dots_, kx: through dS1 and from X^T Q + Z^T K, with a minus
        float own_q = 0.f, own_k = 0.f, dots_ = 0.f, kx = 0.f, dot = 0.f, db = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = z[t] = zero4();
        __syncthreads();                                 // (the previous head's LDS has been read)
        for (int e = tid; e < DELTA_ROWS * 64; e += 256) rows[e] = ((const float *)(a.mats + p * a.mats_bytes))[e];
        const int halves = __builtin_amdgcn_readfirstlane(a.Dvp) / 64;       // (DV / 64, unknown to the compiler: a single turn drawn into what is around it spills)
#pragma unroll 1
        for (int b = 0; b < halves; ++b) {
            const int ln = fresh_lane(), l16 = ln & 15, g4 = ln >> 4, row = 16 * wv + l16, tid = 64 * wv + ln;
            const bf16_t *const krow = ks + row * KS + 4 * g4, *const qrow = qs + row * KS + 4 * g4;
            const bf16_t *const orow = a.dout + ((int64_t)(c.row0 + row) * in.Hv + h) * in.Dv + 64 * b;
            bf16x8 of[2], rf[2], rl[2];                  // the wave's rows of dO, and of dR as hi, lo
            u32x4 tn[4], ts[DK / 32];                    // (read once: past the caches, 750 -> 738 us for 32 768 rows)
#pragma unroll
            for (int e = 0; e < 4; ++e) tn[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(news + (64 * b * 16 + tid + 256 * e) * 8));
#pragma unroll
            for (int e = 0; e < DK / 32; ++e) ts[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(state + 64 * b * DK + (tid + 256 * e) * 8));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                of[s] = row_frag(orow, 32 * s + 8 * g4, row < c.rows && 64 * b + 32 * s + 8 * g4 < in.Dv);
                // eight columns of dR: two lanes' four
                const bf16_t *const r4 = drs + ((4 * b + 2 * s + (g4 >> 1)) * 256 + wv * 64 + (g4 & 1) * 32 + l16) * 8;
                const u32x4 r0 = *reinterpret_cast<const u32x4_any *>(r4), r1 = *reinterpret_cast<const u32x4_any *>(r4 + 128);
                rf[s] = __builtin_bit_cast(bf16x8, u32x4{r0[0], r0[1], r1[0], r1[1]});
                rl[s] = __builtin_bit_cast(bf16x8, u32x4{r0[2], r0[3], r1[2], r1[3]});
            }
            if (b) __syncthreads();                      // (the columns before have been read)
#pragma unroll
            for (int e = 0; e < 4; ++e) {                // N: 16 columns e, wave wv, this lane
                bf16_t *const to = ns + row * TS + 16 * e + 4 * g4;
                put4(to, u32x2{tn[e][0], tn[e][1]});
                put4(to + 64 * TS, u32x2{tn[e][2], tn[e][3]});
            }
            // the state's pieces: 16 columns, 32 rows, lane, two fours 16 rows apart
            auto place = [&](int e, int half) __attribute__((always_inline)) {
                constexpr int KB = DK / 32;
                const int piece = tid + 256 * e, l = piece % 64;
                return ss + (piece / (KB * 64) * 16 + l % 16) * KS + piece / 64 % KB * 32 + half * 16 + l / 16 * 4;
            };
#pragma unroll
            for (int e = 0; e < DK / 32; ++e) {
                put4(place(e, 0), u32x2{ts[e][0], ts[e][1]});
                put4(place(e, 1), u32x2{ts[e][2], ts[e][3]});
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < DK / 32; ++e) ts[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(dstate + 64 * b * DK + (tid + 256 * e) * 8));
            // dO N^T and dR N^T
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (t > wv) continue;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 nj = frag_n(ns, TS, 16 * t, 32 * s, ln), lj = frag_n(ns + 64 * TS, TS, 16 * t, 32 * s, ln);
                    x[t] = mfma16(lj, of[s], x[t]);
                    z[t] = mfma16(lj, rf[s], z[t]);
                    z[t] = mfma16(nj, rl[s], z[t]);
                    x[t] = mfma16(nj, of[s], x[t]);
                    z[t] = mfma16(nj, rf[s], z[t]);
                }
            }
            const float rk = rows[DELTA_RK * 64 + row], eg = rows[DELTA_EG * 64 + row];
            const float fq = eg * rows[DELTA_RQ * 64 + row], fk = -rows[DELTA_BETA * 64 + row] * eg * rk, fs = rows[DELTA_EC * 64 + row] * rk;
            bf16x8 nf[2], nl[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                nf[s] = frag_n(ns, TS, 16 * wv, 32 * s, ln);
                nl[s] = frag_n(ns + 64 * TS, TS, 16 * wv, 32 * s, ln);
            }
            // through S0: scale e^G dO S0^T into dQ, -beta e^G dR S0^T into dK
            float part_q = 0.f, part_k = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 y = zero4(), w = zero4();
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 m = frag_t(ss, KS, 32 * s, 16 * t, ln);
                    w = mfma16(m, rl[s], w);
                    y = mfma16(m, of[s], y);
                    w = mfma16(m, rf[s], w);
                }
                dq[t] += y * fq;
                dk[t] += w * fk;
                part_q = dot4(y, four(qrow + 16 * t), part_q);
                part_k = dot4(w, four(krow + 16 * t), part_k);
                if (t % 2) __builtin_amdgcn_sched_barrier(0);        // (the products' operands of all t at once are more than the registers hold)
            }
            own_q += part_q * fq;
            own_k += part_k * fk;
            __syncthreads();
            // dS1 in the place of S0, their product summed on the way
#pragma unroll
            for (int e = 0; e < DK / 32; ++e) {
                bf16_t *const q0 = place(e, 0), *const q1 = place(e, 1);
                const u32x2 lo = *reinterpret_cast<const u32x2_any *>(q0), hi = *reinterpret_cast<const u32x2_any *>(q1);
                dot = dot8(u32x4{lo[0], lo[1], hi[0], hi[1]}, ts[e], dot);
                put4(q0, u32x2{ts[e][0], ts[e][1]});
                put4(q1, u32x2{ts[e][2], ts[e][3]});
            }
            __syncthreads();
            // through dS1: e^(G_63 - G) N dS1^T into dK
            float part = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 y = zero4();
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const bf16x8 m = frag_t(ss, KS, 32 * s, 16 * t, ln);
                    y = mfma16(m, nl[s], y);
                    y = mfma16(m, nf[s], y);
                }
                dk[t] += y * fs;
                part = dot4(y, four(krow + 16 * t), part);
                if (t % 2) __builtin_amdgcn_sched_barrier(0);
            }
            dots_ += part * fs;
        }
        __syncthreads();
        // X and Z
        const int ln = fresh_lane(), l16 = ln & 15, g4 = ln >> 4, row = 16 * wv + l16;
        const bf16_t *const krow = ks + row * KS + 4 * g4, *const qrow = qs + row * KS + 4 * g4;
        const int diagonal = l16 - 4 * g4;               // (the lane that has the row's own element, and which)
        const float rk = rows[DELTA_RK * 64 + row], fx = rows[DELTA_RQ * 64 + row], fz = -rows[DELTA_BETA * 64 + row] * rk;
        const float gi = rows[DELTA_GH * 64 + row], gi_lo = rows[DELTA_GL * 64 + row];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 xv = zero4(), zv = zero4();
            if (t <= wv) {
                const int j0 = 16 * t + 4 * g4;
                const f32x4 dh = gi - *reinterpret_cast<const f32x4 *>(rows + DELTA_GH * 64 + j0), dl = gi_lo - *reinterpret_cast<const f32x4 *>(rows + DELTA_GL * 64 + j0);
                const f32x4 rj = *reinterpret_cast<const f32x4 *>(rows + DELTA_RK * 64 + j0);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float e = delta_decay(dh[v] + dl[v]) * rj[v];
                    xv[v] = j0 + v <= row ? x[t][v] * e * fx : 0.f;
                    zv[v] = j0 + v < row ? z[t][v] * e * fz : 0.f;
                    if (t == wv && v == diagonal) db = z[t][v];      // dR.N
                }
            }
            const int at = row * TS + 16 * t + 4 * g4;
            const u32x2 xh = hi4(xv), zh = hi4(zv), xl = lo4(xv, xh), zl = lo4(zv, zh);
            put4(xs + at, xh);
            put4(xs + 64 * TS + at, xl);
            put4(zs + at, zh);
            put4(zs + 64 * TS + at, zl);
            if (t <= wv) {
                // q.(X K) and k.(Z K) of the row, from X and Z as the products below take them (accumulators of X K and Z K for this head alone have no registers: with
                // them 23 spill)
                f32x4 qk = zero4(), kk = zero4();
#pragma unroll
                for (int s = 0; s < DK / 32; ++s) {
                    const bf16x8 kj = frag_n(ks, KS, 16 * t, 32 * s, ln);
                    qk = mfma16(kj, frag_n(qs, KS, 16 * wv, 32 * s, ln), qk);
                    kk = mfma16(kj, frag_n(ks, KS, 16 * wv, 32 * s, ln), kk);
                }
                own_q = dot4(qk, up4(xh) + up4(xl), own_q);
                own_k = dot4(kk, up4(zh) + up4(zl), own_k);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) dot += __shfl_xor(dot, m, 64);
        if (lane == 0) dots[wv] = dot;
        __syncthreads();
        // X K, X^T Q, (Z + Z^T) K: zeros and all (left out by wave, their branches cost more)
        bf16x8 xa[2][2], za[2][2], xt[2][2], zt[2][2];   // [hi, lo][32 columns or rows]
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                bf16_t *const xh = xs + half * 64 * TS, *const zh = zs + half * 64 * TS;
                xa[half][s] = frag_n(xh, TS, 16 * wv, 32 * s, ln);
                za[half][s] = frag_n(zh, TS, 16 * wv, 32 * s, ln);
                xt[half][s] = frag_t(xh, TS, 32 * s, 16 * wv, ln);
                zt[half][s] = frag_t(zh, TS, 32 * s, 16 * wv, ln);
            }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 y = dq[t], w = dk[t], u1 = zero4();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 kb = frag_t(ks, KS, 32 * s, 16 * t, ln), qb = frag_t(qs, KS, 32 * s, 16 * t, ln);
#pragma unroll
                for (int half = 1; half >= 0; --half) {
                    y = mfma16(kb, xa[half][s], y);
                    w = mfma16(kb, za[half][s], w);
                    u1 = mfma16(kb, zt[half][s], u1);
                    u1 = mfma16(qb, xt[half][s], u1);
                }
            }
            const f32x4 kr = four(krow + 16 * t);
            dq[t] = y;
            dk[t] = w + u1;
            kx = dot4(u1, kr, kx);
            if (t % 2) __builtin_amdgcn_sched_barrier(0);
        }
        const float sum = over_row((own_q + own_k) - (kx + dots_));
        sum_q += own_q;
        sum_k += own_k + (kx + dots_);
        dots_ = over_row(dots_);
        db = over_row(db);
        if (g4 == 0) {
            dg_row[row] = sum;
            dg_s[row] = dots_;
            if (row < c.rows) store_any(a.db, (int64_t)(c.row0 + row) * in.Hv + h, in.b_f32, (1.f - rows[DELTA_BETA * 64 + row]) * db);
        }
        __syncthreads();
        if (wv == 0) {                                   // lane: its row
            float ends = dg_s[lane];
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) ends += __shfl_xor(ends, m, 64);
            ends += rows[DELTA_EG * 64 + 63] * ((dots[0] + dots[1]) + (dots[2] + dots[3]));
            float dg = dg_row[lane];
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const float y = __shfl_down(dg, m, 64);
                if (lane + m < 64) dg += y;
            }
            dg += ends;
            float da = 0.f, dlog = 0.f;
            if (lane < c.rows) {
                const int64_t t = c.row0 + lane;
                const float g = delta_gate(in, t, h), y = load_any(in.a, t * in.a_tok + h, in.a_f32) + load_any(in.dt_bias, h, in.param_f32);
                da = -expf(load_any(in.a_log, h, in.param_f32)) / (1.f + expf(-y)) * dg;
                dlog = g * dg;
                if (g == -1e4f) da = dlog = 0.f;
                store_any(a.da, t * in.Hv + h, in.a_f32, da);
            }
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                da += __shfl_xor(da, m, 64);
                dlog += __shfl_xor(dlog, m, 64);
            }
            if (lane == 0) {
                a.part[(int64_t)h * a.slots + slot] = dlog;
                a.part[((int64_t)in.Hv + h) * a.slots + slot] = da;
            }
        }
    }
    // back through the unit length: with x = r q (r = 1/|q|), dq = r dx - q r^2 (q . r dx); the accumulators hold r dx
    const float rq = rows[DELTA_RQ * 64 + row] / in.scale, rk = rows[DELTA_RK * 64 + row];
    const float pq = in.l2_norm ? over_row(sum_q) * rq * rq : 0.f;
    const float pk = in.l2_norm ? over_row(sum_k) * rk * rk : 0.f;
    bf16_t *const dq_row = a.dq + ((int64_t)(c.row0 + row) * in.Hk + hk) * in.Dk, *const dk_row = a.dk + ((int64_t)(c.row0 + row) * in.Hk + hk) * in.Dk;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int d = 16 * t + 4 * g4;
        if (live && d < in.Dk) {
            put4(dq_row + d, hi4(dq[t] - four(qrow + 16 * t) * pq));
            put4(dk_row + d, hi4(dk[t] - four(krow + 16 * t) * pk));
        }
    }
}

// da_log and ddt_bias: a workgroup per value head and sum adds its chunks' parts, each thread every 256th, then the threads' in a fixed order
__global__ __launch_bounds__(256) void dsa_delta_param_kernel(DeltaArgs a) {
    __shared__ float red[4];
    const int h = blockIdx.x % a.in.Hv, which = blockIdx.x / a.in.Hv;    // (part: all heads' sums for da_log, then for ddt_bias)
    float s = 0.f;
    for (int c = threadIdx.x; c < a.slots; c += 256) s += a.part[(int64_t)blockIdx.x * a.slots + c];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) store_any(which ? a.ddt : a.da_log, h, a.in.param_f32, (red[0] + red[1]) + (red[2] + red[3]));
}

extern "C" void dsa_launch_delta_back(const DeltaArgs *a, hipStream_t stream);
extern "C" hipError_t dsa_launch_delta_bwd(const DeltaArgs *a, hipStream_t stream) {
    const dim3 grid(a->slots, a->in.Hk);
    dsa_launch_delta_back(a, stream);
    if (a->Dkp == 64 && a->Dvp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<64, 64>), grid, dim3(256), 0, stream, *a);
    else if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<64, 128>), grid, dim3(256), 0, stream, *a);
    else if (a->Dvp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<128, 64>), grid, dim3(256), 0, stream, *a);
    else hipLaunchKernelGGL((dsa_delta_grad_kernel<128, 128>), grid, dim3(256), 0, stream, *a);
    hipLaunchKernelGGL(dsa_delta_param_kernel, dim3(2 * a->in.Hv), dim3(256), 0, stream, *a);
    return hipGetLastError();
}
