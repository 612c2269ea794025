// Gated delta rule: the chunks' own matrices, in front of the walk of the state (see dsa_delta.h for the formulas), and single tokens.
#include "dsa_delta.h"

// ---- T and P of every chunk; one workgroup per chunk and key head, its value heads in turn --------------------------------------------------
// The products of q and k rows are shared by the key head's value heads and stay in registers (wave w: columns 16 w .. of the transposed
// products, so that a lane holds four neighbours of a row of P and A).  T by blocks of 16 rows: the diagonal blocks by substitution, a wave
// each, then T_ij = -T_ii sum_k A_ik T_kj from the diagonal outwards, in fp32 (mfma of 16x16x4): a run of equal keys, whose A is a full triangle of
// ones, has a T of ones and minus ones that powers of A would lose in cancellation.  Bound by what it writes where a backward follows (50 KB of a chunk and head, without
// the quarters that are zeros: 16 384 rows of 32 heads 130 us, 3.1 TB/s) and by the substitution's chain otherwise (100 us); four workgroups a compute unit
// pass the one's waits under the others' work (two, with K and Q in LDS of their own: 220 us).
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
        if (blockIdx.z) return;
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
    for (int u = blockIdx.z; u < rep; u += gridDim.z) {
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
            // (past the caches, as everything that a later kernel reads: the walk of 1 sequence of 32 768 rows 1067 -> 1030 us, of 33 sequences 322 -> 308)
            __builtin_nontemporal_store(u32x4{xh[0], xh[1], yh[0], yh[1]}, reinterpret_cast<u32x4 *>(to + at));
            __builtin_nontemporal_store(u32x4{xl[0], xl[1], yl[0], yl[1]}, reinterpret_cast<u32x4 *>(to + 4096 + at));
        };
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            // a lane's columns: four, and four 16 further (as a walk's registers hold the rows that they meet)
            const int at = tid + 256 * e, r = at / 128 * 16 + l16, half = at / 64 % 2, c0 = 32 * half + 4 * g4;
            if (r >= 32 || half == 0) {                  // (the quarter that is all zeros is neither written nor read)
                plane(tg, at * 8, *reinterpret_cast<const f32x4 *>(tm + r * FS + c0), *reinterpret_cast<const f32x4 *>(tm + r * FS + c0 + 16));
                plane(pm, at * 8, *reinterpret_cast<const f32x4 *>(am + r * FS + c0), *reinterpret_cast<const f32x4 *>(am + r * FS + c0 + 16));
            }
            if (a.planes > 2 && (r < 32 || half == 1)) { // transposed
                f32x4 x[2], y[2];
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    x[v / 4][v % 4] = tm[(c0 + 16 * (v / 4) + v % 4) * FS + r];
                    y[v / 4][v % 4] = am[(c0 + 16 * (v / 4) + v % 4) * FS + r];
                }
                plane(tg + 2 * 4096, at * 8, x[0], x[1]);
                plane(pm + 2 * 4096, at * 8, y[0], y[1]);
            }
        }
    }
}

// ---- one token for each of B requests: the state passes through registers once ----------------------------------------------------------------
// o = scale (e^g S^T q + (k.q) d), S += k d^T with d = beta (v - e^g S^T k): both sums over Dk come from the state as it was read, so it is read
// and written once.  A workgroup takes 32 columns of one head's state (a row of them is 128 bytes, 8 lanes of 16), 32 rows at a time.
// Bound by memory: 256 requests of 32 heads of 128 x 128, 1.07 GB, 218 us, 4.9 TB/s - as a copy; one request 6 us, a launch.
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

extern "C" void dsa_launch_delta_walk(const DeltaArgs *a, int save, hipStream_t stream);
extern "C" hipError_t dsa_launch_delta_fwd(const DeltaArgs *a, int save, hipStream_t stream) {
    if (a->in.T > 0) {
        // the value heads of a key head one after the other, or a workgroup each where all of these find room at once (16 / 32 heads of 128, us, the first and the
        // second: 300 rows 17, 12; 1500 rows 20, 17; 3000 rows 26, 28)
        const int rep = a->in.Hv / a->in.Hk;
        const dim3 grid(a->slots, a->in.Hk, (int64_t)a->slots * a->in.Hv <= 1024 ? rep : 1);
        if (a->Dkp == 64) hipLaunchKernelGGL((dsa_delta_prep_kernel<64>), grid, dim3(256), 0, stream, *a);
        else hipLaunchKernelGGL((dsa_delta_prep_kernel<128>), grid, dim3(256), 0, stream, *a);
    }
    if (a->in.T > 0 || a->final) dsa_launch_delta_walk(a, save, stream);
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_delta_step(const dsa_delta_args *in, float *state, int64_t state_req, void *out, hipStream_t stream) {
    const int64_t grid = (int64_t)in->T * in->Hv * ((in->Dv + 31) / 32);
    if (grid == 0) return hipSuccess;
    if (in->Dk <= 64) hipLaunchKernelGGL((dsa_delta_step_kernel<64>), dim3((unsigned)grid), dim3(256), 0, stream, *in, state, state_req, (bf16_t *)out);
    else hipLaunchKernelGGL((dsa_delta_step_kernel<128>), dim3((unsigned)grid), dim3(256), 0, stream, *in, state, state_req, (bf16_t *)out);
    return hipGetLastError();
}
