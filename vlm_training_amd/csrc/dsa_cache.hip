// Rows into a paged cache and back.
//
// A wave takes one token: all its heads' keys and values, 8 elements a lane, a row of D in a group of lanes (a power of two of them).  The rows' loads are issued in front of
// the search for the token's request and its page, which take three round trips to memory one after the other.
// e4m3: the largest magnitude of a row comes from its bf16 bits as integers (NaN and infinity above all others), its power of two from that alone, and
// x * 2^-e is exact, so that each value is rounded once, to nearest even.
//
// What bounds them: memory.  12 388 rows of 8 + 8 heads of 128 into a bf16 cache 20.6 us (4.9 TB/s), into an 8-bit one 19 us and back 12; 32 768 rows out of an 8-bit cache 39 us
// (5.2 TB/s; 45 with the rows going through the caches), out of a bf16 one 47 (5.7).  One token for each of 256 requests: 4.5 us each, those round trips.
#include "dsa_paged.h"

namespace {

struct CacheRows { const void *k, *v; int64_t k_tok, k_head, v_tok, v_head; };

// Four tokens to a workgroup.  A launch has fewer than 2^32 threads along x - more are cut to 32 bits without an error -, so that workgroups go on along y.
inline dim3 token_grid(int T) {
    const unsigned blocks = (unsigned)(((int64_t)T + 3) / 4), x = blocks < 1u << 22 ? blocks : 1u << 22;
    return dim3(x, (blocks + x - 1) / x);
}
__device__ __forceinline__ int token_of_wave() { return (int)((blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6)); }

// lanes of a row: the power of two that holds D / 8
inline int row_lanes_shift(int D) {
    int s = 0;
    while ((8 << s) < D) ++s;
    return s;
}

template <bool E4M3>
__global__ __launch_bounds__(256) void dsa_cache_write_kernel(dsa_cache_args c, CacheRows in, const int32_t *__restrict__ cu, const int32_t *__restrict__ lengths, int T, int N,
                                                              int pshift, int lshift) {
    const int lane = threadIdx.x & 63, t = token_of_wave();
    if ((uint32_t)t >= (uint32_t)T) return;
    const int sub = lane & ((1 << lshift) - 1), per = 64 >> lshift, mine = lane >> lshift, d = 8 * sub;
    const int items = 2 * c.Hkv;                         // keys of every head, then values
    constexpr int AHEAD = 4;
    u32x4 x[AHEAD];
    auto load = [&](int item) {
        const bool val = item >= c.Hkv;
        const int head = val ? item - c.Hkv : item;
        const bf16_t *src = val ? (const bf16_t *)in.v + t * in.v_tok + head * in.v_head : (const bf16_t *)in.k + t * in.k_tok + head * in.k_head;
        return item < items && d < c.D ? __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + d)) : u32x4{0u, 0u, 0u, 0u};
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = load(i * per + mine);
    const int n = find_request(cu, N, t);
    if (n < 0 || n >= N) return;
    const int p = max(lengths[n], 0) - (cu[n + 1] - t);
    if (p < 0) return;
    const int id = page_of(c, n, pshift, p), place = p & (c.page - 1);
    if (id < 0) return;
    for (int base = 0; base < items; base += AHEAD * per) {
        if (base > 0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) x[i] = load(base + i * per + mine);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int item = base + i * per + mine;
            const bool val = item >= c.Hkv, live = item < items && d < c.D;
            const int head = val ? item - c.Hkv : item;
            const int64_t row = (int64_t)head * c.page + place;
            if constexpr (!E4M3) {
                bf16_t *dst = val ? (bf16_t *)c.v + id * c.v_page + row * c.D : (bf16_t *)c.k + id * c.k_page + row * c.D;
                if (live) *reinterpret_cast<u32x4 *>(dst + d) = x[i];
            } else {
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) most = max(most, max(x[i][j] & 0x7fffu, (x[i][j] >> 16) & 0x7fffu));
                for (int off = 1; off < (1 << lshift); off <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, 64));
                const int e = scale_exponent(most);
                const bool finite = most < 0x7f80u;
                const float mul = __uint_as_float((uint32_t)(127 - e) << 23);
                // Next to bf16's largest value (a power of 2^120) the nearest code may stand for 2^128: 240 of the power is the last that is finite, and off by 2^-4 at most (0x7f70 is it)
                if (most > 0x7f70u) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[i][j] = (x[i][j] & 0x80008000u) | min(x[i][j] & 0x7fffu, 0x7f70u) | min(x[i][j] & 0x7fff0000u, 0x7f700000u);
                }
                u32x2 codes;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t a = x[i][2 * j], b = x[i][2 * j + 1];
                    int w = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(a << 16) * mul, __uint_as_float(a & 0xffff0000u) * mul, 0, false);
                    w = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(b << 16) * mul, __uint_as_float(b & 0xffff0000u) * mul, w, true);
                    codes[j] = finite ? (uint32_t)w : 0x7f7f7f7fu;
                }
                uint8_t *dst = val ? (uint8_t *)c.v + id * c.v_page + row * c.D : (uint8_t *)c.k + id * c.k_page + row * c.D;
                uint8_t *ex = val ? (uint8_t *)c.v_exp + id * c.vx_page + row : (uint8_t *)c.k_exp + id * c.kx_page + row;
                if (live) *reinterpret_cast<u32x2 *>(dst + d) = codes;
                if (live && sub == 0) *ex = finite ? (uint8_t)(e + 127) : (uint8_t)255;
            }
        }
    }
}

template <bool E4M3>
__global__ __launch_bounds__(256) void dsa_cache_read_kernel(dsa_cache_args c, const int32_t *__restrict__ cu, const int32_t *__restrict__ first, int T, int N, int pshift,
                                                             int lshift, bf16_t *__restrict__ k_out, bf16_t *__restrict__ v_out) {
    const int lane = threadIdx.x & 63, t = token_of_wave();
    if ((uint32_t)t >= (uint32_t)T) return;
    const int sub = lane & ((1 << lshift) - 1), per = 64 >> lshift, mine = lane >> lshift, d = 8 * sub;
    const int items = 2 * c.Hkv;
    const int n = find_request(cu, N, t);
    int id = -1, place = 0;
    if (n >= 0 && n < N) {
        const int64_t p = (int64_t)(first ? first[n] : 0) + t - cu[n];
        if (p >= 0 && p <= INT32_MAX) {
            id = page_of(c, n, pshift, (int)p);
            place = (int)p & (c.page - 1);
        }
    }
    for (int base = 0; base < items; base += 4 * per) {
        u32x4 x[4];
        uint32_t ex[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int item = base + i * per + mine;
            const bool val = item >= c.Hkv;
            const int64_t row = (int64_t)(val ? item - c.Hkv : item) * c.page + place;
            x[i] = u32x4{0u, 0u, 0u, 0u};
            ex[i] = 127;
            if (item < items && d < c.D && id >= 0) {
                if constexpr (!E4M3) {
                    const bf16_t *src = val ? (const bf16_t *)c.v + id * c.v_page + row * c.D : (const bf16_t *)c.k + id * c.k_page + row * c.D;
                    x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(src + d));
                } else {
                    const uint8_t *src = val ? (const uint8_t *)c.v + id * c.v_page + row * c.D : (const uint8_t *)c.k + id * c.k_page + row * c.D;
                    const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(src + d));
                    x[i] = u32x4{w[0], w[1], 0u, 0u};
                    ex[i] = val ? ((const uint8_t *)c.v_exp)[id * c.vx_page + row] : ((const uint8_t *)c.k_exp)[id * c.kx_page + row];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int item = base + i * per + mine;
            const bool val = item >= c.Hkv;
            if (item >= items || d >= c.D) continue;
            if constexpr (E4M3) {
                const float s = exponent_scale(ex[i]);
                const u32x2 a = e4m3_to_bf16(x[i][0], s), b = e4m3_to_bf16(x[i][1], s);
                x[i] = u32x4{a[0], a[1], b[0], b[1]};
            }
            bf16_t *dst = (val ? v_out : k_out) + ((int64_t)t * c.Hkv + (val ? item - c.Hkv : item)) * c.D;
            __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4 *>(dst + d));
        }
    }
}

inline int log2_of(int x) { return __builtin_ctz((unsigned)x); }

}  // namespace

extern "C" hipError_t dsa_launch_cache_write(const dsa_cache_args *c, const void *k, int64_t k_tok, int64_t k_head, const void *v, int64_t v_tok, int64_t v_head, const int32_t *cu,
                                             const int32_t *lengths, int T, int N, hipStream_t stream) {
    const dim3 grid = token_grid(T);
    const CacheRows in{k, v, k_tok, k_head, v_tok, v_head};
    const auto kernel = c->kind == DSA_CACHE_E4M3 ? &dsa_cache_write_kernel<true> : &dsa_cache_write_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, *c, in, cu, lengths, T, N, log2_of(c->page), row_lanes_shift(c->D));
    return hipGetLastError();
}
extern "C" hipError_t dsa_launch_cache_read(const dsa_cache_args *c, const int32_t *cu, const int32_t *first, int T, int N, void *k_out, void *v_out, hipStream_t stream) {
    const dim3 grid = token_grid(T);
    const auto kernel = c->kind == DSA_CACHE_E4M3 ? &dsa_cache_read_kernel<true> : &dsa_cache_read_kernel<false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, *c, cu, first, T, N, log2_of(c->page), row_lanes_shift(c->D), (bf16_t *)k_out, (bf16_t *)v_out);
    return hipGetLastError();
}
