// The element-wise operators of a gated-delta-rule layer and of the residual stream around a block:
//   short convolution   z_t = bias + sum_j w[c][W-1-j] x_{t-j} within a sequence, y = z sigmoid(z)
//   gated norm          y = x rsqrt(mean x^2 + eps) w z sigmoid(z), a row per token and head
//   residual norm       x' = x + scale sigmoid(gate) [norm(y) post], h = norm(x') w, a row per token
// All are bound by memory: each row is read and written once per pass, sums stay in fp32 registers, parameter gradients are per-workgroup
// partial sums that a second kernel adds in a fixed order (no atomics).
#include "dsa_rows.h"
#include "../../include/dsa_attn.h"

#include <type_traits>

__device__ __forceinline__ f32x8 zero8() {
    f32x8 z;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = 0.f;
    return z;
}
__device__ __forceinline__ float sigmoid_f(float x) { return 1.f / (1.f + __expf(-x)); }
// eight elements of a bf16 or fp32 row
template <bool F32>
__device__ __forceinline__ f32x8 load8(const void *p, int64_t i) {
    if (F32) {
        const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>((const float *)p + i));
        const f32x4 b = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>((const float *)p + i) + 1);
        return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
    return bf8_to_f32(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>((const bf16_t *)p + i)));
}
template <bool F32>
__device__ __forceinline__ void store8(void *p, int64_t i, f32x8 x) {
    if (F32) {
        __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>((float *)p + i));
        __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4 *>((float *)p + i) + 1);
    } else {
        __builtin_nontemporal_store(f32_to_bf8(x), reinterpret_cast<u32x4 *>((bf16_t *)p + i));
    }
}
// Squares are summed at 2^-14 of their size: 8192 of them overflow only where their mean does.
#define SQUARE_SCALE 0x1p-14f
__device__ __forceinline__ float squares8(f32x8 x) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] * SQUARE_SCALE * x[i];
    return s;
}
__device__ __forceinline__ float load1(const void *p, int64_t i, int f32) { return f32 ? ((const float *)p)[i] : (float)((const bf16_t *)p)[i]; }
__device__ __forceinline__ f32x8 load8_any(const void *p, int64_t i, int f32) {          // a parameter: any alignment; i a multiple of 8
    if (((uintptr_t)p & 15) == 0) return f32 ? load8<true>(p, i) : load8<false>(p, i);
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = load1(p, i + e, f32);
    return r;
}
__device__ __forceinline__ void store1(void *p, int64_t i, int f32, float x) {
    if (f32) ((float *)p)[i] = x;
    else ((bf16_t *)p)[i] = (bf16_t)x;
}

// Column sums: out[i][e] = sum over b < blocks of part[b * stride + at[i] + e], up to three outputs in one launch.  A workgroup has sixteen columns, four to a
// thread, and 64 threads to a column: each adds every 64th block's, then the 64 are added in order (sixteen of four) - the same order on every run.  (With a column
// to a thread and sixteen threads to a column, 1024 blocks of 4096: 7.6 us; this form 4.)
struct SumArgs {
    const float *part;
    int blocks;
    int64_t stride;
    int at[3], n[3], f32[3];
    void *out[3];
};
__global__ __launch_bounds__(256) void dsa_column_sum_kernel(SumArgs a) {
    __shared__ f32x4 red[64][4], red2[16][4];
    const int x = threadIdx.x & 3, y = threadIdx.x >> 2, i = blockIdx.y, e = blockIdx.x * 16 + 4 * x;
    const bool live = e < a.n[i];                        // (every n is a multiple of 4)
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        const float *const p = a.part + a.at[i] + e;
#pragma unroll 8
        for (int b = y; b < a.blocks; b += 64) s += *reinterpret_cast<const f32x4 *>(p + b * a.stride);
    }
    red[y][x] = s;
    __syncthreads();
    if (y < 16) {
        s = red[4 * y][x];
#pragma unroll
        for (int k = 1; k < 4; ++k) s += red[4 * y + k][x];
        red2[y][x] = s;
    }
    __syncthreads();
    if (y == 0 && live) {
        s = red2[0][x];
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red2[k][x];
#pragma unroll
        for (int v = 0; v < 4; ++v) store1(a.out[i], e + v, a.f32[i], s[v]);
    }
}
static void column_sums(const float *part, int blocks, int64_t stride, int count, const int *at, const int *n, void *const *out, const int *f32, hipStream_t stream) {
    SumArgs a = {part, blocks, stride};
    int most = 0, m = 0;
    for (int i = 0; i < count; ++i)
        if (out[i]) {
            a.at[m] = at[i];
            a.n[m] = n[i];
            a.out[m] = out[i];
            a.f32[m++] = f32[i];
            most = n[i] > most ? n[i] : most;
        }
    hipLaunchKernelGGL(dsa_column_sum_kernel, dim3((most + 15) / 16, m), dim3(256), 0, stream, a);
}

// ---- short convolution -------------------------------------------------------------------------------------------------------------------
// A thread keeps four channels over a run of consecutive rows: the last W-1 inputs stay in registers, so a row is read once (and W-1 rows once
// more per run); the next CONV_BATCH rows' loads are in flight while these are worked on.  lanes_c threads of a workgroup, whole waves, lie
// side by side over the channels, the others take further runs: a wave's rows and their addresses are scalars.
// 16 384 rows of 8192, W 4: forwards 112 us, 4.8 TB/s, bound by memory; backwards 185 us, 4.4 TB/s, memory and the 35 instructions an element about even.
// (Eight channels took 256 registers in the backward, two waves per SIMD: 330 us; rows' addresses per lane: 230 us.)
#define CONV_BATCH 4
struct ConvArgs {
    const bf16_t *x, *dy, *state;                        // (T, C) rows x_tok, dy_tok apart;  (N, C, W-1)
    int64_t x_tok, dy_tok;
    const void *w, *bias;                                // (C, W), (C)
    int w_f32, b_f32, silu;
    const int32_t *cu;
    int T, N, C, lanes_c, run;
    bf16_t *y;                                           // y or dx, contiguous
    float *part;                                         // (runs of workgroups, C, W + 1)
};
__device__ __forceinline__ f32x4 bf4_to_f32(u32x2 w) {
    return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
}
__device__ __forceinline__ u32x2 f32_to_bf4(f32x4 x) { return u32x2{pack2bf(x[0], x[1]), pack2bf(x[2], x[3])}; }
__device__ __forceinline__ f32x4 zero4f() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
// the W weights of channels c0 .. c0 + N - 1, which lie one after the other
template <int W, int N>
__device__ __forceinline__ void conv_weights(const void *w, int f32, int c0, float (&out)[N][W]) {
    if (f32) {
#pragma unroll
        for (int i = 0; i < N * W; ++i) out[i / W][i % W] = ((const float *)w)[(int64_t)c0 * W + i];
    } else if (((uintptr_t)w & 7) == 0) {
        const u32x2 *const p = reinterpret_cast<const u32x2 *>((const bf16_t *)w + (int64_t)c0 * W);           // (N is a multiple of 4)
#pragma unroll
        for (int i = 0; i < N * W / 4; ++i) {
            const f32x4 x = bf4_to_f32(p[i]);
#pragma unroll
            for (int v = 0; v < 4; ++v) out[(4 * i + v) / W][(4 * i + v) % W] = x[v];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N * W; ++i) out[i / W][i % W] = (float)((const bf16_t *)w)[(int64_t)c0 * W + i];
    }
}
// where a run stands: the sequence of row t, its first row and the row behind its last
struct ConvPlace {
    int seg, start, end;
    __device__ __forceinline__ void find(const int32_t *cu, int N, int t) {
        seg = find_segment(cu, N, t);
        start = cu[seg];
        end = cu[seg + 1];
    }
    // on to the sequence of row t, which is the row behind the last one or further
    __device__ __forceinline__ void next(const int32_t *cu, int N, int t) {
        while (t >= end && seg + 1 < N) {
            ++seg;
            start = cu[seg];
            end = cu[seg + 1];
        }
    }
};
// the input `back` rows before a sequence's first row: the state's column, or zero
template <int W>
__device__ __forceinline__ f32x4 conv_before(const ConvArgs &a, const ConvPlace &p, int back, int c0) {
    if (!a.state || back > W - 1) return zero4f();
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (float)a.state[((int64_t)p.seg * a.C + c0 + i) * (W - 1) + W - 1 - back];
    return r;
}
template <int W, bool BWD>
__global__ __launch_bounds__(256, BWD ? 3 : 6) void dsa_conv_kernel(ConvArgs a) {
    const int lx = threadIdx.x % a.lanes_c, ly = __builtin_amdgcn_readfirstlane(threadIdx.x / a.lanes_c), runs_y = 256 / a.lanes_c;
    const int c0 = (blockIdx.x * a.lanes_c + lx) * 4;
    const bool live = c0 < a.C;
    const int64_t first = ((int64_t)blockIdx.y * runs_y + ly) * a.run;
    const int t0 = (int)(first < a.T ? first : a.T), t1 = min(a.T, t0 + a.run), last = min(max(a.cu[a.N], 0), a.T);
    f32x4 w[W], b = zero4f(), h[W - 1], acc[W], dw[W], db = zero4f();
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = acc[j] = dw[j] = zero4f();
    if (live) {
        float all[4][W];
        conv_weights<W, 4>(a.w, a.w_f32, c0, all);
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[j][i] = all[i][j];
        if (a.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = load1(a.bias, c0 + i, a.b_f32);
    }
    if (live && t0 < t1) {
        ConvPlace p;
        if (t0 < last) {
            p.find(a.cu, a.N, t0);
#pragma unroll
            for (int j = 1; j < W; ++j) {
                const int t = t0 - j;
                h[j - 1] = t >= p.start ? bf4_to_f32(*reinterpret_cast<const u32x2 *>(a.x + t * a.x_tok + c0)) : conv_before<W>(a, p, p.start - t, c0);
            }
        }
        // the backward goes on for W-1 rows: they have a share in the run's last gradients
        const int stop = min(BWD ? t1 + W - 1 : t1, last);
        // one row; INNER: t and the W-1 rows before it lie in the same sequence and in the run
        auto row = [&](int t, u32x2 xw, u32x2 gw, auto inner) {
            constexpr bool INNER = decltype(inner)::value;
            if (!INNER && t >= p.end) {
                p.next(a.cu, a.N, t);
#pragma unroll
                for (int j = 1; j < W; ++j) h[j - 1] = conv_before<W>(a, p, j, c0);
            }
            const f32x4 xt = bf4_to_f32(xw);
            f32x4 z = b + w[W - 1] * xt;
#pragma unroll
            for (int j = 1; j < W; ++j) z += w[W - 1 - j] * h[j - 1];
            if (!BWD) {
                if (a.silu) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[i] *= sigmoid_f(z[i]);
                }
                __builtin_nontemporal_store(f32_to_bf4(z), reinterpret_cast<u32x2 *>(a.y + (int64_t)t * a.C + c0));
            } else {
                f32x4 dz = bf4_to_f32(gw);
                if (a.silu) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float s = sigmoid_f(z[i]);
                        dz[i] *= s * (1.f + z[i] * (1.f - s));           // (s + z s - z s s would leave nothing of a large z's 1)
                    }
                }
                if (INNER || t < t1) {
                    db += dz;
                    dw[W - 1] += dz * xt;
#pragma unroll
                    for (int j = 1; j < W; ++j) dw[W - 1 - j] += dz * h[j - 1];
                }
                // acc[j]: the gradient of row t - j so far
                acc[0] = w[W - 1] * dz;
#pragma unroll
                for (int j = 1; j < W; ++j)
                    if (INNER || t - j >= p.start) acc[j] += w[W - 1 - j] * dz;
                const int done = t - (W - 1);
                if (INNER || (done >= t0 && done < t1)) __builtin_nontemporal_store(f32_to_bf4(acc[W - 1]), reinterpret_cast<u32x2 *>(a.y + (int64_t)done * a.C + c0));
#pragma unroll
                for (int j = W - 1; j > 0; --j) acc[j] = acc[j - 1];
            }
#pragma unroll
            for (int j = W - 2; j > 0; --j) h[j] = h[j - 1];
            h[0] = xt;
        };
        u32x2 xr[CONV_BATCH], gr[CONV_BATCH];
        auto fetch = [&](int tb) {
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u) {
                const int64_t t = min(tb + u, a.T - 1);
                xr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(a.x + t * a.x_tok + c0));
                if (BWD) gr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(a.dy + t * a.dy_tok + c0));
            }
        };
        fetch(t0);
        for (int tb = t0; tb < stop; tb += CONV_BATCH) {
            u32x2 xn[CONV_BATCH], gn[CONV_BATCH];
#pragma unroll
            for (int u = 0; u < CONV_BATCH; ++u) {
                xn[u] = xr[u];
                gn[u] = gr[u];
            }
            fetch(tb + CONV_BATCH);
            if (tb + CONV_BATCH <= min(p.end, BWD ? t1 : stop) && (!BWD || tb - (W - 1) >= max(t0, p.start))) {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u) row(tb + u, xn[u], gn[u], std::true_type{});
            } else {
#pragma unroll
                for (int u = 0; u < CONV_BATCH; ++u)
                    if (tb + u < stop) row(tb + u, xn[u], gn[u], std::false_type{});
            }
        }
        if (BWD) {
            // rows that no further row adds to: acc[j] is row stop - j now
#pragma unroll
            for (int j = W - 1; j > 0; --j) {
                const int t = stop - j;
                if (t >= t0 && t < t1 && t < last) __builtin_nontemporal_store(f32_to_bf4(acc[j]), reinterpret_cast<u32x2 *>(a.y + (int64_t)t * a.C + c0));
            }
        }
        // rows behind the last sequence: zeros
        for (int t = max(t0, last); t < t1; ++t) *reinterpret_cast<u32x2 *>(a.y + (int64_t)t * a.C + c0) = u32x2{0u, 0u};
    }
    if (BWD) {
        // the workgroup's sums, its runs in order
        __shared__ f32x4 red[256];
        const int64_t base = (int64_t)blockIdx.y * (W + 1) * a.C;
#pragma unroll
        for (int j = 0; j <= W; ++j) {
            f32x4 s = j < W ? dw[j < W ? j : 0] : db;
            if (runs_y > 1) {
                __syncthreads();
                red[threadIdx.x] = s;
                __syncthreads();
                for (int r = 1; r < runs_y && ly == 0; ++r) s += red[r * a.lanes_c + lx];
            }
            if (ly == 0 && live) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (j < W) a.part[base + (int64_t)(c0 + i) * W + j] = s[i];
                    else a.part[base + (int64_t)W * a.C + c0 + i] = s[i];
                }
            }
        }
    }
}
// the last W-1 inputs of every sequence, those before its first row from the initial state
__global__ __launch_bounds__(256) void dsa_conv_state_kernel(ConvArgs a, int W, bf16_t *__restrict__ out) {
    const int64_t n = (int64_t)a.N * a.C * (W - 1);
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        const int j = (int)(e % (W - 1)), c = (int)(e / (W - 1) % a.C), s = (int)(e / (W - 1) / a.C);
        const int start = a.cu[s], len = max(a.cu[s + 1] - start, 0), at = len - (W - 1) + j;      // row of the sequence
        bf16_t v = (bf16_t)0.f;
        if (at >= 0) {
            if (start >= 0 && start + at < a.T) v = a.x[(int64_t)(start + at) * a.x_tok + c];
        } else if (a.state) {
            v = a.state[((int64_t)s * a.C + c) * (W - 1) + W - 1 + at];
        }
        out[e] = v;
    }
}
// one token per request; the state (B, C, W-1) moves on by one
template <int W>
__global__ __launch_bounds__(256) void dsa_conv_step_kernel(ConvArgs a, bf16_t *__restrict__ state, int64_t state_req) {
    const int per = a.C / 8;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, req = e / per;
    if (req >= a.T) return;
    const int c0 = (int)(e - req * per) * 8;
    bf16_t *const s = state + req * state_req + (int64_t)c0 * (W - 1);
    alignas(16) bf16_t old[8 * (W - 1)], now[8 * (W - 1)];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) reinterpret_cast<bf16x8 *>(old)[i] = reinterpret_cast<const bf16x8 *>(s)[i];
    const bf16x8 x = *reinterpret_cast<const bf16x8 *>(a.x + req * a.x_tok + c0);
    float w[8][W];
    conv_weights<W, 8>(a.w, a.w_f32, c0, w);
    f32x8 z;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        z[i] = a.bias ? load1(a.bias, c0 + i, a.b_f32) : 0.f;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            z[i] += w[i][j] * (float)old[i * (W - 1) + j];
            now[i * (W - 1) + j] = j + 1 < W - 1 ? old[i * (W - 1) + j + 1] : x[i];
        }
        z[i] += w[i][W - 1] * (float)x[i];
        if (a.silu) z[i] *= sigmoid_f(z[i]);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) reinterpret_cast<bf16x8 *>(s)[i] = reinterpret_cast<const bf16x8 *>(now)[i];
    *reinterpret_cast<u32x4 *>(a.y + req * a.C + c0) = f32_to_bf8(z);
}

// Threads side by side over the channels, and the rows of a run, none shorter than 16 (W-1 of them come on top).  As many workgroups as run at once, six to a
// compute unit forwards and three backwards; 16 384 rows of 8192: forwards 112 us (three: 117), backwards 185 and 6 for the sums (six: 190 and 10).
static void conv_shape(ConvArgs &a, int &cols, int &rows, int groups) {
    a.lanes_c = 64;
    while (a.lanes_c < 256 && a.lanes_c * 4 < a.C) a.lanes_c *= 2;
    cols = (a.C / 4 + a.lanes_c - 1) / a.lanes_c;
    const int runs_y = 256 / a.lanes_c;
    const int64_t want = (groups + cols - 1) / cols * (int64_t)runs_y;      // runs
    const int64_t run = (a.T + want - 1) / want;
    a.run = (int)(run < 16 ? 16 : run);
    const int64_t per = (int64_t)a.run * runs_y;
    rows = (int)((a.T + per - 1) / per);
}
extern "C" int dsa_conv_blocks(int T, int C) {
    ConvArgs a = {};
    a.T = T;
    a.C = C;
    int cols, rows;
    conv_shape(a, cols, rows, 768);
    return rows;
}
#define CONV_SWITCH(W, CALL)                  \
    switch (W) {                              \
        case 2: { CALL(2); break; }           \
        case 3: { CALL(3); break; }           \
        default: { CALL(4); break; }          \
    }
extern "C" hipError_t dsa_launch_conv_fwd(const void *x, int64_t x_tok, const void *w, int w_f32, const void *bias, int b_f32, int silu, const int32_t *cu, int T, int N,
                                          int C, int W, const void *state, void *y, void *final, hipStream_t stream) {
    ConvArgs a = {(const bf16_t *)x, nullptr, (const bf16_t *)state, x_tok, 0, w, bias, w_f32, b_f32, silu, cu, T, N, C, 0, 0, (bf16_t *)y, nullptr};
    int cols, rows;
    conv_shape(a, cols, rows, 1536);
#define CONV_FWD(WW) hipLaunchKernelGGL((dsa_conv_kernel<WW, false>), dim3(cols, rows), dim3(256), 0, stream, a)
    if (T > 0) CONV_SWITCH(W, CONV_FWD)
    if (final) {
        const int64_t n = ((int64_t)N * C * (W - 1) + 255) / 256;
        hipLaunchKernelGGL(dsa_conv_state_kernel, dim3((unsigned)(n < 8192 ? n : 8192)), dim3(256), 0, stream, a, W, (bf16_t *)final);
    }
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_conv_bwd(const void *x, int64_t x_tok, const void *dy, int64_t dy_tok, const void *w, int w_f32, const void *bias, int b_f32, int silu,
                                          const int32_t *cu, int T, int N, int C, int W, const void *state, void *dx, void *dw, void *dbias, float *part,
                                          hipStream_t stream) {
    ConvArgs a = {(const bf16_t *)x, (const bf16_t *)dy, (const bf16_t *)state, x_tok, dy_tok, w, bias, w_f32, b_f32, silu, cu, T, N, C, 0, 0, (bf16_t *)dx, part};
    int cols, rows;
    conv_shape(a, cols, rows, 768);
#define CONV_BWD(WW) hipLaunchKernelGGL((dsa_conv_kernel<WW, true>), dim3(cols, rows), dim3(256), 0, stream, a)
    if (T > 0) CONV_SWITCH(W, CONV_BWD)
    const int64_t stride = (int64_t)(W + 1) * C;
    const int at[2] = {0, W * C}, n[2] = {W * C, C}, f32[2] = {w_f32, b_f32};
    void *const out[2] = {dw, dbias};
    column_sums(part, T > 0 ? rows : 0, stride, 2, at, n, out, f32, stream);
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_conv_step(const void *x, int64_t x_tok, const void *w, int w_f32, const void *bias, int b_f32, int silu, int B, int C, int W, void *state,
                                           int64_t state_req, void *y, hipStream_t stream) {
    ConvArgs a = {(const bf16_t *)x, nullptr, nullptr, x_tok, 0, w, bias, w_f32, b_f32, silu, nullptr, B, 0, C, 0, 0, (bf16_t *)y, nullptr};
    const unsigned blocks = (unsigned)(((int64_t)B * (C / 8) + 255) / 256);
#define CONV_STEP(WW) hipLaunchKernelGGL((dsa_conv_step_kernel<WW>), dim3(blocks), dim3(256), 0, stream, a, (bf16_t *)state, state_req)
    if (blocks) CONV_SWITCH(W, CONV_STEP)
    return hipGetLastError();
}

// ---- gated norm --------------------------------------------------------------------------------------------------------------------------
// A row of D elements is spread over LPR = D/8 lanes (rounded up to a power of two), 64/LPR rows per wave and step; the mean is a butterfly over them.
// 524 288 rows of 128: forwards 71 us, 5.6 TB/s, backwards 124 us, 5.4 TB/s - as a copy.
struct GatedNormArgs {
    const bf16_t *x, *z, *dy;
    int64_t x_tok, x_head, z_tok, z_head;
    const void *w;
    int w_f32, H, D;
    float eps, offset;
    int64_t rows;
    bf16_t *y, *dx, *dz;
    float *rstd, *part;                                  // (blocks, D)
};
template <int LPR, bool BWD>
__global__ __launch_bounds__(256) void dsa_gated_norm_kernel(GatedNormArgs a) {
    constexpr int RPW = 64 / LPR;
    __shared__ float red[4][LPR * 8];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = lane / LPR, d0 = lane % LPR * 8;
    const bool in_d = d0 < a.D;
    f32x8 w = zero8(), dw = zero8();
    if (in_d) w = load8_any(a.w, d0, a.w_f32) + a.offset;
    const float inv = 1.f / (float)a.D;
    const int64_t step = (int64_t)gridDim.x * 4 * RPW;
    for (int64_t r0 = ((int64_t)blockIdx.x * 4 + wv) * RPW; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + sub, t = r / a.H;
        const int hh = (int)(r - t * a.H);
        const bool live = in_d && r < a.rows;
        f32x8 x = zero8(), z = zero8(), g = zero8();
        if (live) {
            x = load8<false>(a.x, t * a.x_tok + hh * a.x_head + d0);
            z = load8<false>(a.z, t * a.z_tok + hh * a.z_head + d0);
            if (BWD) g = load8<false>(a.dy, r * a.D + d0);
        }
        f32x8 s;                                         // (z s first: 0 for the lowest z, which times anything else may pass fp32's range)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = sigmoid_f(z[i]);
        if (!BWD) {
            float ss = squares8(x);
#pragma unroll
            for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m, 64);
            const float rs = rsqrtf(ss * (inv / SQUARE_SCALE) + a.eps);
            if (live) {
                store8<false>(a.y, r * a.D + d0, x * rs * w * (z * s));
                if (d0 == 0 && a.rstd) a.rstd[r] = rs;
            }
        } else {
            const float rs = live ? a.rstd[r] : 0.f;
            const f32x8 xh = x * rs, gs = g * (z * s), dn = gs * w;
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += dn[i] * xh[i];
#pragma unroll
            for (int m = 1; m < LPR; m <<= 1) dot += __shfl_xor(dot, m, 64);
            dw += gs * xh;
            if (live) {
                store8<false>(a.dx, r * a.D + d0, (dn - xh * (dot * inv)) * rs);
                store8<false>(a.dz, r * a.D + d0, g * xh * w * s * (1.f + z * (1.f - s)));
            }
        }
    }
    if (BWD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int m = LPR; m < 64; m <<= 1) dw[i] += __shfl_xor(dw[i], m, 64);
            if (sub == 0) red[wv][d0 + i] = dw[i];
        }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += 256) a.part[(int64_t)blockIdx.x * a.D + d] = (red[0][d] + red[1][d]) + (red[2][d] + red[3][d]);
    }
}
static int gated_norm_lanes(int D) {
    int l = 8;
    while (l * 8 < D) l *= 2;
    return l;
}
static int gated_norm_grid(int64_t rows, int D, int most) {
    const int64_t per = 4 * (64 / gated_norm_lanes(D)), want = (rows + per - 1) / per;
    return (int)(want < most ? want : most);
}
extern "C" int dsa_gated_norm_blocks(int64_t rows, int D) { return gated_norm_grid(rows, D, 1024); }
#define GNORM_SWITCH(B, GRID)                                                                                           \
    switch (gated_norm_lanes(a.D)) {                                                                                     \
        case 8: hipLaunchKernelGGL((dsa_gated_norm_kernel<8, B>), dim3(GRID), dim3(256), 0, stream, a); break;           \
        case 16: hipLaunchKernelGGL((dsa_gated_norm_kernel<16, B>), dim3(GRID), dim3(256), 0, stream, a); break;         \
        case 32: hipLaunchKernelGGL((dsa_gated_norm_kernel<32, B>), dim3(GRID), dim3(256), 0, stream, a); break;         \
        default: hipLaunchKernelGGL((dsa_gated_norm_kernel<64, B>), dim3(GRID), dim3(256), 0, stream, a); break;         \
    }
extern "C" hipError_t dsa_launch_gated_norm_fwd(const void *x, int64_t x_tok, int64_t x_head, const void *z, int64_t z_tok, int64_t z_head, const void *w, int w_f32,
                                                float eps, float offset, int T, int H, int D, void *y, float *rstd, hipStream_t stream) {
    GatedNormArgs a = {(const bf16_t *)x, (const bf16_t *)z, nullptr, x_tok, x_head, z_tok, z_head, w, w_f32, H, D, eps, offset, (int64_t)T * H, (bf16_t *)y, nullptr,
                       nullptr, rstd, nullptr};
    const int grid = gated_norm_grid(a.rows, D, 8192);
    if (grid) GNORM_SWITCH(false, grid)
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_gated_norm_bwd(const void *dy, const void *x, int64_t x_tok, int64_t x_head, const void *z, int64_t z_tok, int64_t z_head, const void *w,
                                                int w_f32, float offset, int T, int H, int D, const float *rstd, void *dx, void *dz, void *dw, float *part,
                                                hipStream_t stream) {
    GatedNormArgs a = {(const bf16_t *)x, (const bf16_t *)z, (const bf16_t *)dy, x_tok, x_head, z_tok, z_head, w, w_f32, H, D, 0.f, offset, (int64_t)T * H, nullptr,
                       (bf16_t *)dx, (bf16_t *)dz, const_cast<float *>(rstd), part};
    const int grid = gated_norm_grid(a.rows, D, 1024);
    if (grid) GNORM_SWITCH(true, grid)
    const int at[1] = {0};
    column_sums(part, grid, D, 1, at, &D, &dw, &w_f32, stream);
    return hipGetLastError();
}

// ---- residual norm ------------------------------------------------------------------------------------------------------------------------
// A row of C elements is spread over TPR threads, eight elements each: a wave up to 512, then as many waves as it takes, so that a thread holds one
// piece of everything (with two pieces per thread the row's values and the three parameters took 256 registers, one wave per SIMD).  The next row's loads go
// out before this row's sums.  The backward forms both norms' gradients in one pass: d = dx' + norm'(dh) goes to x as it is and on through scale, gate and the
// first norm to y.  The forward's norm reads x' before it is rounded: a bf16 stream's is formed again from x and y (STREAM_BEFORE), which a gate, a scale or a first norm
// read anyway and a plain addition 67 MB more of for 8192 rows of 4096 (x' as it was rounded leaves dx off by 2.5e-3 instead of its own rounding's 1.7e-3, and dw, in
// fp32 too, by 1.7e-3).  Those rows: forwards 51 us, 5.2 TB/s, backwards 73 us, 5.5 TB/s (of x' as it was rounded 63 us).
struct ResidualArgs {
    const void *x;                                       // bf16 or fp32 (X32), all (T, C) contiguous
    const bf16_t *y, *gate;
    const void *w, *post, *scale;
    int w_f32, post_f32, scale_f32, C;
    float eps, offset;
    int64_t rows;
    void *xn;                                            // x';  backward, DSA_STREAM_BF16_BEFORE: x
    bf16_t *h;
    float *rstd, *rstd_y;
    const void *dxn;                                     // gradients of x' and h (null: none)
    const bf16_t *dh;
    void *dx;
    bf16_t *dy, *dgate;
    float *part;                                         // (blocks, 3, C): of w, post, scale
};
// the sum over a row's threads, on each of them
template <int TPR>
__device__ __forceinline__ float row_total(float s, float *red) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
    if (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wv = threadIdx.x >> 6, row = wv / W * W;
        __syncthreads();                                 // (the sum before has been read)
        if ((threadIdx.x & 63) == 0) red[wv] = s;
        __syncthreads();
        s = red[row];
#pragma unroll
        for (int i = 1; i < W; ++i) s += red[row + i];
    }
    return s;
}
constexpr int residual_threads(int tpr) { return tpr < 256 ? 256 : tpr; }
// eight elements of a row as they lie in memory
template <bool F32>
struct Raw8 {
    u32x4 v[F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        const u32x4 *const q = reinterpret_cast<const u32x4 *>((const char *)p + i * (F32 ? 4 : 2));
#pragma unroll
        for (int k = 0; k < (F32 ? 2 : 1); ++k) v[k] = __builtin_nontemporal_load(q + k);
    }
    __device__ __forceinline__ f32x8 get() const {
        if (!F32) return bf8_to_f32(v[0]);
        f32x8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = __uint_as_float(v[F32 ? i / 4 : 0][i % 4]);
        return r;
    }
};
// the elements of a row that a thread has, or zeros
__device__ __forceinline__ f32x8 or_zero(f32x8 x, bool keep) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = keep ? x[i] : 0.f;
    return x;
}
// THROUGH: the block's output passes a norm, a gate or a scale
template <int TPR, bool X32, bool THROUGH>
__global__ __launch_bounds__(residual_threads(TPR)) void dsa_residual_norm_fwd_kernel(ResidualArgs a) {
    __shared__ float red[16];
    constexpr int RPB = residual_threads(TPR) / TPR;
    const int c = threadIdx.x % TPR * 8, ly = threadIdx.x / TPR;
    const bool in_c = c < a.C;
    const int cc = in_c ? c : 0;                         // (a thread past C reads the row's first elements, and drops them)
    const float inv = 1.f / (float)a.C;
    f32x8 w = zero8(), post = zero8(), scale = zero8() + 1.f;
    if (in_c) {
        w = load8_any(a.w, c, a.w_f32) + a.offset;
        if (THROUGH && a.post) post = load8_any(a.post, c, a.post_f32) + a.offset;
        if (THROUGH && a.scale) scale = load8_any(a.scale, c, a.scale_f32);
    }
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + ly;
    Raw8<X32> xr;
    Raw8<false> yr, gr;
    auto fetch = [&](int64_t row) {
        const int64_t at = (row < a.rows ? row : a.rows - 1) * a.C + cc;
        yr.load(a.y, at);
        xr.load(a.x, at);
        if (THROUGH && a.gate) gr.load(a.gate, at);
    };
    fetch(r);
    for (int64_t rb = (int64_t)blockIdx.x * RPB; rb < a.rows; rb += step, r += step) {
        const int64_t at = r * a.C + c;
        const bool live = in_c && r < a.rows;
        f32x8 v = or_zero(yr.get(), in_c), x = or_zero(xr.get(), in_c);
        if (THROUGH && a.gate) {
            const f32x8 g = gr.get();
            f32x8 s;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = sigmoid_f(g[i]);
            fetch(r + step);
            if (a.post) {
                const float rs = rsqrtf(row_total<TPR>(squares8(v), red) * (inv / SQUARE_SCALE) + a.eps);
                if (live && c == 0 && a.rstd_y) a.rstd_y[r] = rs;
                v = v * rs * post;
            }
            v *= s;
        } else {
            fetch(r + step);
            if (THROUGH && a.post) {
                const float rs = rsqrtf(row_total<TPR>(squares8(v), red) * (inv / SQUARE_SCALE) + a.eps);
                if (live && c == 0 && a.rstd_y) a.rstd_y[r] = rs;
                v = v * rs * post;
            }
        }
        x += v * scale;
        const float rs = rsqrtf(row_total<TPR>(squares8(x), red) * (inv / SQUARE_SCALE) + a.eps);
        if (live) {
            store8<X32>(a.xn, at, x);
            store8<false>(a.h, at, x * rs * w);
            if (c == 0 && a.rstd) a.rstd[r] = rs;
        }
    }
}
template <int TPR, int STREAM, bool THROUGH>
__global__ __launch_bounds__(residual_threads(TPR)) void dsa_residual_norm_bwd_kernel(ResidualArgs a) {
    constexpr int RPB = residual_threads(TPR) / TPR;
    constexpr bool X32 = STREAM == DSA_STREAM_F32, BEFORE = STREAM == DSA_STREAM_BF16_BEFORE;
    // AHEAD: the next row's loads before this row's sums, the parameters in registers.  1024 threads have 128 registers each, which the sums of three parameters
    // leave no room for: there every row reads the parameters again, for each of its two sums, and forms the block's output for each (8192 rows of 8192 with norm, gate and
    // scale, forwards and backwards: 504 us, of an fp32 stream 622; kept through the sum 945 and 728, in registers that spill).
    constexpr bool AHEAD = !(THROUGH && TPR == 1024);
    __shared__ float red[16], sums[RPB > 1 ? 256 : 1][8];
    const int c = threadIdx.x % TPR * 8, ly = threadIdx.x / TPR;
    const bool in_c = c < a.C;
    const int cc = in_c ? c : 0;
    const float inv = 1.f / (float)a.C;
    f32x8 w = zero8(), post = zero8() + 1.f, scale = zero8() + 1.f, dw = zero8(), dpost = zero8(), dscale = zero8();
    auto parameters = [&](int e) {
        w = load8_any(a.w, e, a.w_f32) + a.offset;
        if (THROUGH && a.post) post = load8_any(a.post, e, a.post_f32) + a.offset;
        if (THROUGH && a.scale) scale = load8_any(a.scale, e, a.scale_f32);
    };
    if (AHEAD) parameters(cc);
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t r = (int64_t)blockIdx.x * RPB + ly;
    Raw8<X32> dr, xr;
    Raw8<false> hr, yr, gr;
    float rs_next = 0.f, ry_next = 1.f;
    auto fetch = [&](int64_t row) {
        const int64_t clamped = row < a.rows ? row : a.rows - 1, at = clamped * a.C + cc;
        if (a.dxn) dr.load(a.dxn, at);
        if (a.dh) {
            hr.load(a.dh, at);
            xr.load(a.xn, at);
            rs_next = a.rstd[clamped];
        }
        if (THROUGH || (BEFORE && a.dh)) yr.load(a.y, at);
        if (THROUGH) {
            if (a.gate) gr.load(a.gate, at);
            if (a.post) ry_next = a.rstd_y[clamped];
        }
    };
    if (AHEAD) fetch(r);
    for (int64_t rb = (int64_t)blockIdx.x * RPB; rb < a.rows; rb += step, r += step) {
        const int64_t at = r * a.C + c;
        const bool live = in_c && r < a.rows;
        if (!AHEAD) {
            int e = cc;
            asm volatile("" : "+v"(e));                  // (so that they are not kept after all)
            parameters(e);
            fetch(r);
        }
        const float rs = rs_next, ry = ry_next;
        f32x8 d = zero8(), xh = zero8(), y = zero8(), sg = zero8() + 1.f, dh = zero8();
        if (a.dxn) d = or_zero(dr.get(), live);
        if (a.dh) {
            dh = or_zero(hr.get(), live);
            xh = or_zero(xr.get(), live);
        }
        auto block = [&]() {                             // the block's output, normed, and its gate
            y = or_zero(yr.get(), live);
            if (THROUGH) {
                y *= ry;
                if (a.gate) {
                    const f32x8 g = gr.get();
#pragma unroll
                    for (int i = 0; i < 8; ++i) sg[i] = sigmoid_f(g[i]);
                }
            }
        };
        if (AHEAD ? THROUGH || (BEFORE && a.dh) : BEFORE && a.dh) block();
        if (AHEAD) fetch(r + step);
        if (a.dh) {
            if (BEFORE) xh += THROUGH ? y * post * sg * scale : y;       // (the forward's order)
            xh *= rs;
            dw += dh * xh;
            dh *= w;
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += dh[i] * xh[i];
            d += (dh - xh * (row_total<TPR>(dot, red) * inv)) * rs;
        }
        if (live) store8<X32>(a.dx, at, d);
        if (THROUGH) {
            if (!AHEAD) {
                int e = cc;
                asm volatile("" : "+v"(e), "+v"(yr.v[0]), "+v"(gr.v[0]));        // (formed again: not kept through the sum)
                parameters(e);
                block();
            }
            const f32x8 p = y * post;                    // what gate and scale multiply
            if (a.gate && live) store8<false>(a.dgate, at, d * p * scale * sg * (1.f - sg));
            dscale += or_zero(d * p * sg, live);         // (a row past the last one has its gate's copy)
            d *= scale * sg;
            if (a.post) {
                dpost += or_zero(d * y, live);
                d *= post;
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) dot += d[i] * y[i];
                d = (d - y * (row_total<TPR>(dot, red) * inv)) * ry;
            }
        }
        if (live) store8<false>(a.dy, at, d);
    }
    float *const part = a.part + (int64_t)blockIdx.x * 3 * a.C;
#pragma unroll
    for (int which = 0; which < (THROUGH ? 3 : 1); ++which) {
        if ((which == 1 && !a.post) || (which == 2 && !a.scale)) continue;
        f32x8 s = which == 0 ? dw : which == 1 ? dpost : dscale;
        if (RPB > 1) {                                   // the workgroup's rows, in order
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[RPB > 1 ? threadIdx.x : 0][i] = s[i];
            __syncthreads();
            for (int k = 1; k < RPB; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += sums[RPB > 1 ? k * TPR + threadIdx.x % TPR : 0][i];
        }
        if (in_c && ly == 0) {
            *reinterpret_cast<f32x4 *>(part + (int64_t)which * a.C + c) = f32x4{s[0], s[1], s[2], s[3]};
            *reinterpret_cast<f32x4 *>(part + (int64_t)which * a.C + c + 4) = f32x4{s[4], s[5], s[6], s[7]};
        }
    }
}
static int residual_tpr(int C) {
    int t = 64;
    while (t * 8 < C) t *= 2;
    return t;
}
static int residual_grid(int64_t rows, int C, int most) {
    const int tpr = residual_tpr(C), rpb = residual_threads(tpr) / tpr;
    const int64_t want = (rows + rpb - 1) / rpb;
    return (int)(want < most ? want : most);
}
// The backward's workgroups: one or two to every compute unit, so that they all run at once (260 for 1037 rows of 2560: 41 us, 256: 27), and so that
// their sums, 12 C bytes each, stay a small part of what is written.
extern "C" int dsa_residual_norm_blocks(int64_t rows, int C) { return residual_grid(rows, C, rows < 2048 ? 256 : 512); }
#define RNORM_SWITCH(K, X, P, GRID)                                                                               \
    switch (residual_tpr(a.C)) {                                                                                   \
        case 64: hipLaunchKernelGGL((K<64, X, P>), dim3(GRID), dim3(256), 0, stream, a); break;                    \
        case 128: hipLaunchKernelGGL((K<128, X, P>), dim3(GRID), dim3(256), 0, stream, a); break;                  \
        case 256: hipLaunchKernelGGL((K<256, X, P>), dim3(GRID), dim3(256), 0, stream, a); break;                  \
        case 512: hipLaunchKernelGGL((K<512, X, P>), dim3(GRID), dim3(512), 0, stream, a); break;                  \
        default: hipLaunchKernelGGL((K<1024, X, P>), dim3(GRID), dim3(1024), 0, stream, a); break;                 \
    }
#define RNORM_LAUNCH(K, X, GRID)                                               \
    {                                                                          \
        if (a.post || a.gate || a.scale) RNORM_SWITCH(K, X, true, GRID)        \
        else RNORM_SWITCH(K, X, false, GRID)                                   \
    }
extern "C" hipError_t dsa_launch_residual_norm_fwd(const void *x, int x_f32, const void *y, const void *gate, const void *w, int w_f32, const void *post, int post_f32,
                                                   const void *scale, int scale_f32, float eps, float offset, int T, int C, void *xn, void *h, float *rstd, float *rstd_y,
                                                   hipStream_t stream) {
    ResidualArgs a = {x, (const bf16_t *)y, (const bf16_t *)gate, w, post, scale, w_f32, post_f32, scale_f32, C, eps, offset, T, xn, (bf16_t *)h, rstd, rstd_y};
    const int grid = residual_grid(T, C, 1024);
    if (grid && x_f32) RNORM_LAUNCH(dsa_residual_norm_fwd_kernel, true, grid)
    else if (grid) RNORM_LAUNCH(dsa_residual_norm_fwd_kernel, false, grid)
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_residual_norm_bwd(const void *dxn, const void *dh, const void *xn, int stream_kind, const void *y, const void *gate, const void *w, int w_f32,
                                                   const void *post, int post_f32, const void *scale, int scale_f32, float offset, int T, int C, const float *rstd,
                                                   const float *rstd_y, void *dx, void *dy, void *dgate, void *dw, void *dpost, void *dscale, float *part,
                                                   hipStream_t stream) {
    ResidualArgs a = {nullptr, (const bf16_t *)y, (const bf16_t *)gate, w, post, scale, w_f32, post_f32, scale_f32, C, 0.f, offset, T, const_cast<void *>(xn), nullptr,
                      const_cast<float *>(rstd), const_cast<float *>(rstd_y), dxn, (const bf16_t *)dh, dx, (bf16_t *)dy, (bf16_t *)dgate, part};
    const int grid = dsa_residual_norm_blocks(T, C);
    if (grid && stream_kind == DSA_STREAM_F32) RNORM_LAUNCH(dsa_residual_norm_bwd_kernel, DSA_STREAM_F32, grid)
    else if (grid && stream_kind == DSA_STREAM_BF16_BEFORE) RNORM_LAUNCH(dsa_residual_norm_bwd_kernel, DSA_STREAM_BF16_BEFORE, grid)
    else if (grid) RNORM_LAUNCH(dsa_residual_norm_bwd_kernel, DSA_STREAM_BF16, grid)
    const int at[3] = {0, C, 2 * C}, n[3] = {C, C, C}, f32[3] = {w_f32, post_f32, scale_f32};
    void *const out[3] = {dw, post ? dpost : nullptr, scale ? dscale : nullptr};
    column_sums(part, grid, 3 * (int64_t)C, 3, at, n, out, f32, stream);
    return hipGetLastError();
}
