// Gated delta rule, chunked forward: the chunks' own matrices, then the walk of the state (see dsa_delta.h for the formulas).
#include "dsa_delta.h"

// ---- T and P of every chunk; one workgroup per chunk and key head, its value heads in turn --------------------------------------------------
// The products of q and k rows are shared by the key head's value heads and stay in registers (wave w: columns 16 w .. of the transposed
// products, so that a lane holds four neighbours of a row of P and A).  T by blocks of 16 rows: the diagonal blocks by substitution, a wave
// each, then T_ij = -T_ii sum_k A_ik T_kj from the diagonal outwards, in fp32 (mfma of 16x16x4): a run of equal keys, whose A is a full triangle of
// ones, has a T of ones and minus ones that powers of A would lose in cancellation.
template <int DK>
__global__ __launch_bounds__(256) void dsa_delta_prep_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, FS = 68;
    __shared__ bf16_t ks[64 * KS], qs[64 * KS];
    __shared__ float am[64 * FS], tm[64 * FS], ms[4][16 * 17], rk[64], rq[64], gh[64], gl[64], bt[64];
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, l16 = lane & 15, g4 = lane >> 4;
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
    const int i = 16 * wv + l16;
    for (int u = 0; u < rep; ++u) {
        const int h = hk * rep + u;
        const int64_t p = (int64_t)slot * in.Hv + h;
        __syncthreads();                                 // (the previous head's LDS has been read)
        float *const rows = a.rows + p * DELTA_ROWS * 64;
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
        bf16_t *const pm = a.pmat + p * 4096;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 x = zero4(), y = zero4();
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int j = 16 * t + 4 * g4 + v;
                const float e = j <= i ? expf((gh[i] - gh[j]) + (gl[i] - gl[j])) : 0.f;
                x[v] = j <= i ? e * rq[i] * rk[j] * qk[t][v] : 0.f;
                y[v] = j < i ? e * bt[i] * rk[i] * rk[j] * kk[t][v] : 0.f;
            }
            put4(pm + i * 64 + 16 * t + 4 * g4, hi4(x));
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
                for (int k = 0; k < r; ++k) s -= am[(16 * wv + r) * FS + 16 * wv + k] * x[k];
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
        {
            bf16_t *const th = a.tmat + p * 8192 + (tid >> 2) * 64 + (tid & 3) * 16, *const tl = th + 4096;
#pragma unroll
            for (int e = 0; e < 4; ++e) put_split4(th + 4 * e, tl + 4 * e, *reinterpret_cast<const f32x4 *>(tm + (tid >> 2) * FS + (tid & 3) * 16 + 4 * e));
        }
    }
}

// ---- the walk: one workgroup per sequence, value head and 64 columns of the state, a wave per 16 of them ----------------------------------
// A wave's 16 columns (Dk x 16 fp32) stay in its registers from the first chunk to the last; what it multiplies with is shared by the four
// waves in LDS, the next chunk's on its way into registers meanwhile.  Bound by the chain of a chunk's three products, each of which has to be laid out
// anew for the next one (through the wave's own LDS, no barrier).
template <int DK, bool SAVE>
__global__ __launch_bounds__(256) void dsa_delta_walk_kernel(DeltaArgs a) {
    constexpr int KS = DK + 8, TS = DELTA_TS, NS = 20;
    __shared__ bf16_t ks[64 * KS], qs[64 * KS], th[64 * TS], tl[64 * TS], ps[64 * TS], vs[64 * TS];
    __shared__ bf16_t wsh[4][16 * KS], wsl[4][16 * KS], wrh[4][16 * TS], wrl[4][16 * TS], wn[4][3][64 * NS];
    __shared__ float rows[5 * 64];
    const dsa_delta_args &in = a.in;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, l16 = lane & 15, g4 = lane >> 4;
    const int blocks = a.Dvp / 64, h = blockIdx.x / blocks % in.Hv, seg = blockIdx.x / blocks / in.Hv, dv0 = blockIdx.x % blocks * 64;
    const int hk = h / (in.Hv / in.Hk), dv = dv0 + 16 * wv + l16;
    int slot0, chunks, s0, L;
    delta_segment(in.cu, in.N, seg, slot0, chunks, s0, L);
    chunks = min(chunks, a.slots - slot0);
    s0 = max(s0, 0);
    bf16_t *const sh = wsh[wv], *const sl = wsl[wv], *const rh = wrh[wv], *const rl = wrl[wv], *const nh = wn[wv][0], *const nl = wn[wv][1], *const np = wn[wv][2];
    f32x4 st[DK / 16];                                   // S[dk = 16 t + 4 g4 + v][dv]
    const int64_t cell = ((int64_t)seg * in.Hv + h) * in.Dk * in.Dv + dv;
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int k = 16 * t + 4 * g4 + v;
            st[t][v] = a.initial && k < in.Dk && dv < in.Dv ? a.initial[cell + (int64_t)k * in.Dv] : 0.f;
        }
    Tile64<DK> tk, tq;
    Tile64<64> tth, ttl, tp, tv;
    float tr[2];
    auto fetch = [&](int c) __attribute__((always_inline)) {
        const int row0 = s0 + 64 * c, n = min(min(64, L - 64 * c), in.T - row0);
        const int64_t p = (int64_t)(slot0 + c) * in.Hv + h;
        tile_load<DK>(tk, (const bf16_t *)in.k + row0 * in.k_tok + hk * in.k_head, in.k_tok, n, in.Dk);
        tile_load<DK>(tq, (const bf16_t *)in.q + row0 * in.q_tok + hk * in.q_head, in.q_tok, n, in.Dk);
        tile_load<64>(tth, a.tmat + p * 8192, 64, 64, 64);
        tile_load<64>(ttl, a.tmat + p * 8192 + 4096, 64, 64, 64);
        tile_load<64>(tp, a.pmat + p * 4096, 64, 64, 64);
        tile_load<64>(tv, (const bf16_t *)in.v + row0 * in.v_tok + h * in.v_head + dv0, in.v_tok, n, in.Dv - dv0);
        tr[0] = a.rows[p * DELTA_ROWS * 64 + tid];
        tr[1] = tid < 64 ? a.rows[p * DELTA_ROWS * 64 + 256 + tid] : 0.f;
    };
    if (chunks > 0) fetch(0);
    for (int c = 0; c < chunks; ++c) {
        const int row0 = s0 + 64 * c, n = min(min(64, L - 64 * c), in.T - row0);
        const int64_t p = (int64_t)(slot0 + c) * in.Hv + h;
        tile_put<DK>(tk, ks, KS);
        tile_put<DK>(tq, qs, KS);
        tile_put<64>(tth, th, TS);
        tile_put<64>(ttl, tl, TS);
        tile_put<64>(tp, ps, TS);
        tile_put<64>(tv, vs, TS);
        rows[tid] = tr[0];
        if (tid < 64) rows[256 + tid] = tr[1];
        __syncthreads();
        if (c + 1 < chunks) fetch(c + 1);
        const float *const eg = rows + DELTA_EG * 64, *const ec = rows + DELTA_EC * 64, *const beta = rows + DELTA_BETA * 64, *const rk = rows + DELTA_RK * 64,
                    *const rq = rows + DELTA_RQ * 64;
        // S0 as [dv][dk]
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            const u32x2 x = hi4(st[t]);
            put4(sh + l16 * KS + 16 * t + 4 * g4, x);
            put4(sl + l16 * KS + 16 * t + 4 * g4, lo4(st[t], x));
            if (SAVE) put4(a.state + (p * a.Dvp + dv) * DK + 16 * t + 4 * g4, x);
        }
        wave_sync();
        f32x4 o[4], r[4];                                // o: [dv = 4 g4 + v][row 16 m + l16];  r: [row 16 m + 4 g4 + v][dv = l16]
#pragma unroll
        for (int m = 0; m < 4; ++m) o[m] = r[m] = zero4();
#pragma unroll
        for (int s = 0; s < DK / 32; ++s) {
            const bf16x8 bh = frag_n(sh, KS, 0, 32 * s), bl = frag_n(sl, KS, 0, 32 * s);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const bf16x8 ka = frag_n(ks, KS, 16 * m, 32 * s);
                r[m] = mfma16(ka, bl, r[m]);
                r[m] = mfma16(ka, bh, r[m]);
                o[m] = mfma16(bh, frag_n(qs, KS, 16 * m, 32 * s), o[m]);
            }
        }
        // R = beta (V - e^G K S0), as [dv][row]
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 x;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int i = 16 * m + 4 * g4 + v;
                x[v] = beta[i] * ((float)vs[i * TS + 16 * wv + l16] - eg[i] * rk[i] * r[m][v]);
            }
            put_split4(rh + l16 * TS + 16 * m + 4 * g4, rl + l16 * TS + 16 * m + 4 * g4, x);
        }
        wave_sync();
        // N^T = R^T T^T: [dv = 4 g4 + v][row 16 m + l16]; rows of T end at the diagonal
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            f32x4 x = zero4();
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (32 * s > 16 * m + 15) continue;
                const bf16x8 ah = frag_n(rh, TS, 0, 32 * s), al = frag_n(rl, TS, 0, 32 * s), bh = frag_n(th, TS, 16 * m, 32 * s), bl = frag_n(tl, TS, 16 * m, 32 * s);
                x = mfma16(al, bh, x);
                x = mfma16(ah, bl, x);
                x = mfma16(ah, bh, x);
            }
            const int i = 16 * m + l16;
            const u32x2 y = hi4(x);
            put4(np + i * NS + 4 * g4, y);
            if (SAVE) put4(a.news + (p * 64 + i) * a.Dvp + dv0 + 16 * wv + 4 * g4, y);
            const float f = ec[i] * rk[i];
            put_split4(nh + i * NS + 4 * g4, nl + i * NS + 4 * g4, x * f);
        }
        wave_sync();
        // O^T = scale e^G S0^T Q^T + N^T P^T
        bf16x8 na[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) na[s] = frag_t(np, NS, 32 * s, 0);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int i = 16 * m + l16;
            o[m] *= eg[i] * rq[i];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (32 * s <= 16 * m + 15) o[m] = mfma16(na[s], frag_n(ps, TS, 16 * m, 32 * s), o[m]);
            const int d = dv0 + 16 * wv + 4 * g4;
            if (i < n && d < in.Dv) put4(a.out + ((int64_t)(row0 + i) * in.Hv + h) * in.Dv + d, hi4(o[m]));
        }
        // S1 = e^G_63 S0 + K^T e^(G_63 - G) N
        const float e = eg[63];
        bf16x8 bh[2], bl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bh[s] = frag_t(nh, NS, 32 * s, 0);
            bl[s] = frag_t(nl, NS, 32 * s, 0);
        }
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            st[t] *= e;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 ka = frag_t(ks, KS, 32 * s, 16 * t);
                st[t] = mfma16(ka, bl[s], st[t]);
                st[t] = mfma16(ka, bh[s], st[t]);
            }
        }
        __syncthreads();
    }
    if (a.final) {
#pragma unroll
        for (int t = 0; t < DK / 16; ++t)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int k = 16 * t + 4 * g4 + v;
                if (k < in.Dk && dv < in.Dv) a.final[cell + (int64_t)k * in.Dv] = st[t][v];
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

extern "C" hipError_t dsa_launch_delta_fwd(const DeltaArgs *a, int save, hipStream_t stream) {
    if (a->in.T > 0) {
        const dim3 grid(a->slots, a->in.Hk);
        if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_prep_kernel<64>), grid, dim3(256), 0, stream, *a);
        else hipLaunchKernelGGL((dsa_delta_prep_kernel<128>), grid, dim3(256), 0, stream, *a);
    }
    const dim3 walks((unsigned)((int64_t)a->in.N * a->in.Hv * (a->Dvp / 64)));
    if (a->in.T > 0 || a->final) {
        if (a->Dkp == 64) {
            if (save) hipLaunchKernelGGL((dsa_delta_walk_kernel<64, true>), walks, dim3(256), 0, stream, *a);
            else hipLaunchKernelGGL((dsa_delta_walk_kernel<64, false>), walks, dim3(256), 0, stream, *a);
        } else {
            if (save) hipLaunchKernelGGL((dsa_delta_walk_kernel<128, true>), walks, dim3(256), 0, stream, *a);
            else hipLaunchKernelGGL((dsa_delta_walk_kernel<128, false>), walks, dim3(256), 0, stream, *a);
        }
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
