// Gated delta rule, backward.  With N = T R, R = beta (V - e^G K S0) of a chunk (dsa_delta.h), from its last chunk to its first:
//     dN = P^T dO + e^(G_63 - G) K dS1      dR = T^T dN      dS0 = e^G_63 dS1 + scale Q^T e^G dO - K^T beta e^G dR
// (the walk, which leaves dS1 and dR of every chunk and dV = beta dR), then all chunks at once
//     dP = dO N^T   dA = -dR N^T   X = scale E dP   Z = beta E dA (below the diagonal)
//     dQ = X K + scale e^G dO S0^T          dK = X^T Q + (Z + Z^T) K + e^(G_63 - G) N dS1^T - beta e^G dR S0^T
//     db = (1 - beta) dR.N                  (dR.N = beta dbeta: both of beta's places, in R and in A, at once)
//     dG_i = rows of (X QK + Z KK) - columns of it + q.(scale e^G S0 dO) - k.(beta e^G S0 dR) - k.(e^(G_63 - G) dS1 N)
//     dG_63 also + all k.(e^(G_63 - G) dS1 N) + e^G_63 <dS1, S0>
// dg is the sum of dG from its row on.  Rows and columns of X QK come from one rounding, so that a pair of rows behind t leaves nothing in dg_t.
#include "dsa_delta.h"

// ---- the walk: as the forward's, from the last chunk to the first ------------------------------------------------------------------------
template <int DK>
__global__ __launch_bounds__(256) void dsa_delta_back_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, TS = DELTA_TS, NS = 20, SS = 16 * KS > 64 * NS ? 16 * KS : 64 * NS;     // dR takes the place of dS in the wave's LDS
    __shared__ bf16_t ks[64 * KS], qs[64 * KS], th[64 * TS], tl[64 * TS], ps[64 * TS], ds[64 * TS];
    __shared__ bf16_t wsh[4][SS], wsl[4][SS], wrh[4][16 * TS], wrl[4][16 * TS], wo[4][2][64 * NS];
    __shared__ float rows[5 * 64];
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, l16 = lane & 15, g4 = lane >> 4;
    const int blocks = a.Dvp / 64, h = blockIdx.x / blocks % in.Hv, seg = blockIdx.x / blocks / in.Hv, dv0 = blockIdx.x % blocks * 64;
    const int hk = h / (in.Hv / in.Hk), dv = dv0 + 16 * wv + l16;
    int slot0, chunks, s0, L;
    delta_segment(in.cu, in.N, seg, slot0, chunks, s0, L);
    chunks = min(chunks, a.slots - slot0);
    s0 = max(s0, 0);
    bf16_t *const sh = wsh[wv], *const sl = wsl[wv], *const rh = wrh[wv], *const rl = wrl[wv], *const oh = wo[wv][0], *const ol = wo[wv][1];
    f32x4 st[DK / 16];                                   // dS[dk = 16 t + 4 g4 + v][dv]
    const int64_t cell = ((int64_t)seg * in.Hv + h) * in.Dk * in.Dv + dv;
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int k = 16 * t + 4 * g4 + v;
            st[t][v] = a.dfinal && k < in.Dk && dv < in.Dv ? a.dfinal[cell + (int64_t)k * in.Dv] : 0.f;
        }
    Tile64<DK> tk, tq;
    Tile64<64> tth, ttl, tp, td;
    float tr[2];
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const int row0 = s0 + 64 * c, n = min(min(64, L - 64 * c), in.T - row0);
        const int64_t p = (int64_t)(slot0 + c) * in.Hv + h;
        tile_load<DK>(tk, (const bf16_t *)in.k + row0 * in.k_tok + hk * in.k_head, in.k_tok, n, in.Dk);
        tile_load<DK>(tq, (const bf16_t *)in.q + row0 * in.q_tok + hk * in.q_head, in.q_tok, n, in.Dk);
        tile_load<64>(tth, a.tmat + p * 8192, 64, 64, 64);
        tile_load<64>(ttl, a.tmat + p * 8192 + 4096, 64, 64, 64);
        tile_load<64>(tp, a.pmat + p * 4096, 64, 64, 64);
        tile_load<64>(td, a.dout + ((int64_t)row0 * in.Hv + h) * in.Dv + dv0, (int64_t)in.Hv * in.Dv, n, in.Dv - dv0);
        tr[0] = a.rows[p * DELTA_ROWS * 64 + tid];
        tr[1] = tid < 64 ? a.rows[p * DELTA_ROWS * 64 + 256 + tid] : 0.f;
    };
    if (chunks > 0) fetch(chunks - 1);
    for (int c = chunks - 1; c >= 0; --c) {
        const int row0 = s0 + 64 * c, n = min(min(64, L - 64 * c), in.T - row0);
        const int64_t p = (int64_t)(slot0 + c) * in.Hv + h;
        tile_put<DK>(tk, ks, KS);
        tile_put<DK>(tq, qs, KS);
        tile_put<64>(tth, th, TS);
        tile_put<64>(ttl, tl, TS);
        tile_put<64>(tp, ps, TS);
        tile_put<64>(td, ds, TS);
        rows[tid] = tr[0];
        if (tid < 64) rows[256 + tid] = tr[1];
        __syncthreads();
        if (c > 0) fetch(c - 1);
        const float *const eg = rows + DELTA_EG * 64, *const ec = rows + DELTA_EC * 64, *const beta = rows + DELTA_BETA * 64, *const rk = rows + DELTA_RK * 64,
                    *const rq = rows + DELTA_RQ * 64;
        // dS1 as [dv][dk], and e^G scale/|q| dO as [row][dv] (lane: its row)
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            const u32x2 x = hi4(st[t]);
            put4(sh + l16 * KS + 16 * t + 4 * g4, x);
            put4(sl + l16 * KS + 16 * t + 4 * g4, lo4(st[t], x));
            put4(a.dstate + (p * a.Dvp + dv) * DK + 16 * t + 4 * g4, x);
        }
        const float fo = eg[lane] * rq[lane];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            f32x4 x;
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = (float)ds[lane * TS + 16 * wv + 4 * u + v] * fo;
            put_split4(oh + lane * NS + 4 * u, ol + lane * NS + 4 * u, x);
        }
        wave_sync();
        f32x4 r[4];                                      // [row 16 m + 4 g4 + v][dv = l16]
#pragma unroll
        for (int m = 0; m < 4; ++m) r[m] = zero4();
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) {
            const bf16x8 bh = frag_n(sh, KS, 0, 32 * s), bl = frag_n(sl, KS, 0, 32 * s);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const bf16x8 ka = frag_n(ks, KS, 16 * m, 32 * s);
                r[m] = mfma16(ka, bl, r[m]);
                r[m] = mfma16(ka, bh, r[m]);
            }
        }
        bf16x8 db[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) db[s] = frag_t(ds, TS, 32 * s, 16 * wv);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int v = 0; v < 4; ++v) r[m][v] *= ec[16 * m + 4 * g4 + v] * rk[16 * m + 4 * g4 + v];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (32 * s + 31 >= 16 * m) r[m] = mfma16(frag_t(ps, TS, 32 * s, 16 * m), db[s], r[m]);
            put_split4(rh + l16 * TS + 16 * m + 4 * g4, rl + l16 * TS + 16 * m + 4 * g4, r[m]);
        }
        wave_sync();
        // dR^T = dN^T T: [dv = 4 g4 + v][row 16 m + l16]; columns of T begin at the diagonal
        bf16x8 ah[2], al[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            ah[s] = frag_n(rh, TS, 0, 32 * s);
            al[s] = frag_n(rl, TS, 0, 32 * s);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 x = zero4();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (32 * s + 31 < 16 * m) continue;
                const bf16x8 bh = frag_t(th, TS, 32 * s, 16 * m), bl = frag_t(tl, TS, 32 * s, 16 * m);
                x = mfma16(al[s], bh, x);
                x = mfma16(ah[s], bl, x);
                x = mfma16(ah[s], bh, x);
            }
            const int i = 16 * m + l16, d = dv0 + 16 * wv + 4 * g4;
            put4(a.drs + (p * 64 + i) * a.Dvp + d, hi4(x));
            if (i < n && d < in.Dv) put4(a.dv + ((int64_t)(row0 + i) * in.Hv + h) * in.Dv + d, hi4(x * beta[i]));
            put_split4(sh + i * NS + 4 * g4, sl + i * NS + 4 * g4, x * (-beta[i] * eg[i] * rk[i]));
        }
        wave_sync();
        // dS0 = e^G_63 dS1 + Q^T (..) + K^T (..)
        const float e = eg[63];
        bf16x8 bh[2], bl[2], qh[2], ql[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bh[s] = frag_t(sh, NS, 32 * s, 0);
            bl[s] = frag_t(sl, NS, 32 * s, 0);
            qh[s] = frag_t(oh, NS, 32 * s, 0);
            ql[s] = frag_t(ol, NS, 32 * s, 0);
        }
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            st[t] *= e;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 ka = frag_t(ks, KS, 32 * s, 16 * t), qa = frag_t(qs, KS, 32 * s, 16 * t);
                st[t] = mfma16(ka, bl[s], st[t]);
                st[t] = mfma16(ka, bh[s], st[t]);
                st[t] = mfma16(qa, ql[s], st[t]);
                st[t] = mfma16(qa, qh[s], st[t]);
            }
        }
        __syncthreads();
    }
    if (a.dinitial) {
#pragma unroll
        for (int t = 0; t < DK / 16; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int k = 16 * t + 4 * g4 + v;
                if (k < in.Dk && dv < in.Dv) a.dinitial[cell + (int64_t)k * in.Dv] = st[t][v];
            }
    }
}

// ---- everything that needs one chunk alone: one workgroup per chunk and key head, its value heads in turn --------------------------------
// dq and dk of the key head are summed over its value heads in registers (wave w: rows 16 w ..), in that order.  The matrices of 64 x 64 are formed
// transposed (lane: one row i, four neighbours j), so that they go to LDS in row order.
template <int DK, int DV>
__global__ __launch_bounds__(256) void dsa_delta_grad_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, VS = DV + 8, TS = DELTA_TS, NT = DK / 16;
    __shared__ bf16_t ks[64 * KS], qs[64 * KS], os[64 * VS], rs[64 * VS], ns[64 * VS], ss[DV * KS], xs[64 * TS], zs[64 * TS];
    __shared__ float rows[DELTA_ROWS * 64], dg_row[64], dg_col[4][64], dg_q[64], dg_k[64], dg_s[64], dbeta[64], dots[4];
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, l16 = lane & 15, g4 = lane >> 4;
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
    __syncthreads();
    f32x4 kk[4], qk[4];                                  // [j = 16 t + 4 g4 + v], row i = 16 wv + l16
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
    f32x4 dq[NT], dk[NT];                                // [row 16 wv + 4 g4 + v][16 t + l16], times scale/|q| and 1/|k|
#pragma unroll
    for (int t = 0; t < NT; ++t) dq[t] = dk[t] = zero4();
    const float *const eg = rows + DELTA_EG * 64, *const ec = rows + DELTA_EC * 64, *const beta = rows + DELTA_BETA * 64, *const rk = rows + DELTA_RK * 64,
                *const rq = rows + DELTA_RQ * 64, *const gh = rows + DELTA_GH * 64, *const gl = rows + DELTA_GL * 64;
    const int i = 16 * wv + l16;
    for (int u = 0; u < rep; ++u) {
        const int h = hk * rep + u;
        const int64_t p = (int64_t)slot * in.Hv + h;
        __syncthreads();                                 // (the previous head's LDS has been read)
        tile_copy<DV>(os, VS, a.dout + ((int64_t)c.row0 * in.Hv + h) * in.Dv, (int64_t)in.Hv * in.Dv, c.rows, in.Dv);
        tile_copy<DV>(rs, VS, a.drs + p * 64 * DV, DV, 64, DV);
        tile_copy<DV>(ns, VS, a.news + p * 64 * DV, DV, 64, DV);
#pragma unroll
        for (int b = 0; b < DV / 64; ++b) tile_copy<DK>(ss + 64 * b * KS, KS, a.state + (p * DV + 64 * b) * DK, DK, 64, DK);
        for (int e = tid; e < DELTA_ROWS * 64; e += 256) rows[e] = a.rows[p * DELTA_ROWS * 64 + e];
        __syncthreads();
        // X and Z, their products with QK and KK summed over rows and columns
        float row = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 x = zero4(), z = zero4(), both = zero4();
            if (t <= wv) {
#pragma unroll
                for (int s = 0; s < DV / 32; ++s) {
                    const bf16x8 nj = frag_n(ns, VS, 16 * t, 32 * s);
                    x = mfma16(nj, frag_n(os, VS, 16 * wv, 32 * s), x);
                    z = mfma16(nj, frag_n(rs, VS, 16 * wv, 32 * s), z);
                }
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int j = 16 * t + 4 * g4 + v;
                    const float e = j <= i ? expf((gh[i] - gh[j]) + (gl[i] - gl[j])) * rk[j] : 0.f;
                    x[v] = j <= i ? x[v] * e * rq[i] : 0.f;
                    z[v] = j < i ? -z[v] * e * beta[i] * rk[i] : 0.f;
                    both[v] = x[v] * qk[t][v] + z[v] * kk[t][v];
                    row += both[v];
                }
            }
            put4(xs + i * TS + 16 * t + 4 * g4, hi4(x));
            put4(zs + i * TS + 16 * t + 4 * g4, hi4(z));
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                float s = both[v];
#pragma unroll
                for (int m = 1; m < 16; m <<= 1) s += __shfl_xor(s, m, 64);
                if (l16 == 0) dg_col[wv][16 * t + 4 * g4 + v] = s;
            }
        }
        row += __shfl_xor(row, 16, 64);
        row += __shfl_xor(row, 32, 64);
        if (g4 == 0) dg_row[i] = row;
        {   // dR.N: four threads per row
            const int r = tid >> 2, c0 = (tid & 3) * (DV / 4);
            float s = 0.f;
            for (int e = 0; e < DV / 4; ++e) s += (float)rs[r * VS + c0 + e] * (float)ns[r * VS + c0 + e];
            s += __shfl_xor(s, 1, 64);
            s += __shfl_xor(s, 2, 64);
            if ((tid & 3) == 0) dbeta[r] = s;
        }
        // through S0: scale e^G dO S0^T into dQ, -beta e^G dR S0^T into dK
        f32x4 fq, fk, dotq = zero4(), dotk = zero4();
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int r = 16 * wv + 4 * g4 + v;
            fq[v] = eg[r] * rq[r];
            fk[v] = -beta[r] * eg[r] * rk[r];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 x = zero4(), y = zero4();
#pragma unroll
            for (int s = 0; s < DV / 32; ++s) {
                const bf16x8 b = frag_t(ss, KS, 32 * s, 16 * t);
                x = mfma16(frag_n(os, VS, 16 * wv, 32 * s), b, x);
                y = mfma16(frag_n(rs, VS, 16 * wv, 32 * s), b, y);
            }
            x *= fq;
            y *= fk;
            dq[t] += x;
            dk[t] += y;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int r = 16 * wv + 4 * g4 + v;
                dotq[v] += x[v] * (float)qs[r * KS + 16 * t + l16];
                dotk[v] += y[v] * (float)ks[r * KS + 16 * t + l16];
            }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) {
                dotq[v] += __shfl_xor(dotq[v], m, 64);
                dotk[v] += __shfl_xor(dotk[v], m, 64);
            }
            if (l16 == 0) {
                dg_q[16 * wv + 4 * g4 + v] = dotq[v];
                dg_k[16 * wv + 4 * g4 + v] = dotk[v];
            }
        }
        __syncthreads();
        // dS1 in the place of S0, their product summed on the way
        float dot = 0.f;
#pragma unroll
        for (int b = 0; b < DV / 64; ++b) {
            Tile64<DK> t1;
            tile_load<DK>(t1, a.dstate + (p * DV + 64 * b) * DK, DK, 64, DK);
#pragma unroll
            for (int e = 0; e < DK / 32; ++e) {
                const int at = tid + 256 * e;
                bf16_t *const q = ss + (64 * b + at / (DK / 8)) * KS + at % (DK / 8) * 8;
                dot = dot8_chain(__builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_any *>(q)), __builtin_bit_cast(bf16x8, t1.x[e]), dot);
                *reinterpret_cast<u32x4_any *>(q) = t1.x[e];
            }
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) dot += __shfl_xor(dot, m, 64);
        if (lane == 0) dots[wv] = dot;
        // X K, X^T Q, (Z + Z^T) K
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool low = 32 * s <= 16 * wv + 15, up = 32 * s + 31 >= 16 * wv;      // columns up to the row; rows from it on
            const bf16x8 x = frag_n(xs, TS, 16 * wv, 32 * s), z = frag_n(zs, TS, 16 * wv, 32 * s);
            const bf16x8 xt = frag_t(xs, TS, 32 * s, 16 * wv), zt = frag_t(zs, TS, 32 * s, 16 * wv);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bf16x8 kb = frag_t(ks, KS, 32 * s, 16 * t);
                if (low) {
                    dq[t] = mfma16(x, kb, dq[t]);
                    dk[t] = mfma16(z, kb, dk[t]);
                }
                if (up) {
                    dk[t] = mfma16(zt, kb, dk[t]);
                    dk[t] = mfma16(xt, frag_t(qs, KS, 32 * s, 16 * t), dk[t]);
                }
            }
        }
        __syncthreads();
        // through dS1: e^(G_63 - G) N dS1^T into dK
        f32x4 fs, dots_ = zero4();
#pragma unroll
        for (int v = 0; v < 4; ++v) fs[v] = ec[16 * wv + 4 * g4 + v] * rk[16 * wv + 4 * g4 + v];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4 x = zero4();
#pragma unroll
            for (int s = 0; s < DV / 32; ++s) x = mfma16(frag_n(ns, VS, 16 * wv, 32 * s), frag_t(ss, KS, 32 * s, 16 * t), x);
            x *= fs;
            dk[t] += x;
#pragma unroll
            for (int v = 0; v < 4; ++v) dots_[v] += x[v] * (float)ks[(16 * wv + 4 * g4 + v) * KS + 16 * t + l16];
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) dots_[v] += __shfl_xor(dots_[v], m, 64);
            if (l16 == 0) dg_s[16 * wv + 4 * g4 + v] = dots_[v];
        }
        __syncthreads();
        if (wv == 0) {                                   // lane: its row
            float ends = dg_s[lane];
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) ends += __shfl_xor(ends, m, 64);
            ends += eg[63] * ((dots[0] + dots[1]) + (dots[2] + dots[3]));
            float dg = dg_row[lane] - ((dg_col[0][lane] + dg_col[1][lane]) + (dg_col[2][lane] + dg_col[3][lane])) + dg_q[lane] + dg_k[lane] - dg_s[lane];
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const float x = __shfl_down(dg, m, 64);
                if (lane + m < 64) dg += x;
            }
            dg += ends;
            float da = 0.f, dlog = 0.f;
            if (lane < c.rows) {
                const int64_t t = c.row0 + lane;
                const float g = delta_gate(in, t, h), x = load_any(in.a, t * in.a_tok + h, in.a_f32) + load_any(in.dt_bias, h, in.param_f32);
                da = -expf(load_any(in.a_log, h, in.param_f32)) / (1.f + expf(-x)) * dg;
                dlog = g * dg;
                if (g == -1e4f) da = dlog = 0.f;
                store_any(a.da, t * in.Hv + h, in.a_f32, da);
                store_any(a.db, t * in.Hv + h, in.b_f32, (1.f - beta[lane]) * dbeta[lane]);
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
    __syncthreads();
    f32x4 pq = zero4(), pk = zero4();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int r = 16 * wv + 4 * g4 + v;
            pq[v] += dq[t][v] * (float)qs[r * KS + 16 * t + l16];
            pk[v] += dk[t][v] * (float)ks[r * KS + 16 * t + l16];
        }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int r = 16 * wv + 4 * g4 + v;
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) {
            pq[v] += __shfl_xor(pq[v], m, 64);
            pk[v] += __shfl_xor(pk[v], m, 64);
        }
        const float x = rq[r] / in.scale;
        pq[v] *= in.l2_norm ? x * x : 0.f;
        pk[v] *= in.l2_norm ? rk[r] * rk[r] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {                    // (a lane's own places)
            const int at = (16 * wv + 4 * g4 + v) * KS + 16 * t + l16;
            qs[at] = (bf16_t)(dq[t][v] - pq[v] * (float)qs[at]);
            ks[at] = (bf16_t)(dk[t][v] - pk[v] * (float)ks[at]);
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < DK / 32; ++e) {
        const int at = tid + 256 * e, r = at / (DK / 8), d = at % (DK / 8) * 8;
        if (r < c.rows && d < in.Dk) {
            *reinterpret_cast<u32x4_any *>(a.dq + ((int64_t)(c.row0 + r) * in.Hk + hk) * in.Dk + d) = *reinterpret_cast<const u32x4_any *>(qs + r * KS + d);
            *reinterpret_cast<u32x4_any *>(a.dk + ((int64_t)(c.row0 + r) * in.Hk + hk) * in.Dk + d) = *reinterpret_cast<const u32x4_any *>(ks + r * KS + d);
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

extern "C" hipError_t dsa_launch_delta_bwd(const DeltaArgs *a, hipStream_t stream) {
    const dim3 walks((unsigned)((int64_t)a->in.N * a->in.Hv * (a->Dvp / 64))), grid(a->slots, a->in.Hk);
    if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_back_kernel<64>), walks, dim3(256), 0, stream, *a);
    else hipLaunchKernelGGL((dsa_delta_back_kernel<128>), walks, dim3(256), 0, stream, *a);
    if (a->Dkp == 64 && a->Dvp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<64, 64>), grid, dim3(256), 0, stream, *a);
    else if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<64, 128>), grid, dim3(256), 0, stream, *a);
    else if (a->Dvp == 64) hipLaunchKernelGGL((dsa_delta_grad_kernel<128, 64>), grid, dim3(256), 0, stream, *a);
    else hipLaunchKernelGGL((dsa_delta_grad_kernel<128, 128>), grid, dim3(256), 0, stream, *a);
    hipLaunchKernelGGL(dsa_delta_param_kernel, dim3(2 * a->in.Hv), dim3(256), 0, stream, *a);
    return hipGetLastError();
}
