// The gated delta rule's kernels share this: arguments, workspace, tiles of 64 rows in LDS and their MFMA fragments.
//
// One value head of one sequence carries a state S (Dk x Dv, fp32):
//     S_t = e^g_t S_{t-1} + beta_t k_t (v_t - e^g_t S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t
// with q, k of unit length, g = -e^a_log softplus(a + dt_bias), beta = sigmoid(b).  In chunks of 64 rows, G the running sum of g inside the
// chunk, E_ij = e^(G_i - G_j) for j <= i:
//     A_ij = beta_i E_ij k_i.k_j (j < i)      P_ij = scale E_ij q_i.k_j (j <= i)      T = (I + A)^-1
//     R = beta (V - e^G K S0)     N = T R     O = scale e^G Q S0 + P N     S1 = e^G_63 S0 + K^T e^(G_63 - G) N
// T and P depend on no state: all chunks at once; S goes from chunk to chunk, its columns independent of each other.  The factors
// 1/|q|, 1/|k|, e^G, beta multiply rows of fp32 results, so that q, k and v enter the products as the bf16 they are; T, P, S, R and N go in as two
// bf16 (hi + lo, off by 2^-18 of the value at the most, a product of two, without lo x lo, by three times that): where keys repeat, rows of P N are sums of 64 terms
// that cancel to the size of one.  One exception: the chunk gradients read S0 and dS1, which the walks keep for them, as one bf16 each (dsa_delta_bwd.hip).
#pragma once
#include "dsa_tile.h"
#include "../../include/dsa_attn.h"

#define DELTA_CHUNK 64
#define DELTA_TS 72                    // row stride of a 64-wide tile: 16-byte rows, four banks on per row
#define DELTA_RS 36                    // of a 32-wide one
// factors of a chunk's rows, 64 floats each: e^G, e^(G_63 - G), beta, 1/|k|, scale/|q|, G in two floats (hi + lo)
enum { DELTA_EG, DELTA_EC, DELTA_BETA, DELTA_RK, DELTA_RQ, DELTA_GH, DELTA_GL, DELTA_ROWS };

struct DeltaArgs {
    dsa_delta_args in;
    int slots, Dkp, Dvp;               // chunks at the most; head dims padded to 64 or 128
    // A chunk of a value head ("cell", slots x Hv of them) has a block of each of three arrays.
    // mats: the rows' factors (DELTA_ROWS x 64 floats), then planes of 64 x 64 bf16: T as hi, lo and, where a backward follows, transposed hi, lo; P the same.
    //       A plane lies in blocks of 16 rows and 32 columns, lane l's eight elements together: row l%16, columns 4 (l/16) + 0..3 and 16 further.  Blocks that are
    //       all zeros (the upper right quarter, of a transposed one the lower left) are neither written nor read.
    // saved, for the backward: S0 (Dvp x Dkp), N as hi, lo (Dvp x 64 x 2);  back, the backward's own: dS1, dR as hi, lo.  They lie as the walks' lanes
    //       have them, 16 columns of the values together: a state 32 rows at a time, lane l's rows 4 (l/16) + 0..3 and 16 further of column l%16; N and dR 16 rows at
    //       a time, lane l's row l%16, columns 4 (l/16) + 0..3 as hi, then as lo.
    // (A quad of lanes that reads or writes four rows takes four times as long as one that stays in one: with rows of T, P, S and N in row order, K and
    // Q as fragments straight from their rows and 8-byte stores, the walk of 16 384 tokens took 0.62 ms.)
    char *mats, *saved, *back;
    int planes, mats_bytes, saved_bytes, back_bytes;
    int choose, maybe_one;             // a launch of walks is one of several forms, of which delta_form tells the one; DELTA_ONE is among them
    const float *initial;              // (N, Hv, Dk, Dv) or null
    float *final;
    bf16_t *out;
    // backward
    const bf16_t *dout;
    const float *dfinal;
    float *part;                       // (2, Hv, slots) sums of a chunk for da_log and ddt_bias
    float *dinitial;
    bf16_t *dq, *dk, *dv;
    void *da, *db, *da_log, *ddt;
};
#define DELTA_T 2048                   // byte of a cell's block in mats where the planes begin
#define DELTA_PLANE 8192

// a chunk of the batch: its segment's first row and the chunk's first row and number of rows.  cu is read as it is, but rows stay within [0, T).
struct DeltaChunk { int row0, rows, seg, index, of; };
// slot -> chunk, by a whole wave (slot wave-uniform); false: a spare slot, `index` then counts the spare ones
__device__ __forceinline__ bool delta_locate(const int32_t *cu, int N, int T, int slot, DeltaChunk &c) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < N; base += 64) {
        const int seg = min(base + lane, N - 1);
        const int lo = cu[seg], len = cu[seg + 1] - lo;
        const int nb = base + lane < N && len > 0 ? (len + DELTA_CHUNK - 1) / DELTA_CHUNK : 0, upto = wave_prefix_i(nb);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > slot);
        if (past) {
            const int w = (int)__builtin_ctzll(past);
            const int s0 = __builtin_amdgcn_readlane(lo, w), L = __builtin_amdgcn_readlane(len, w);
            c.of = __builtin_amdgcn_readlane(nb, w);
            c.index = slot - (__builtin_amdgcn_readlane(upto, w) - c.of);
            c.seg = base + w;
            c.row0 = max(s0 + c.index * DELTA_CHUNK, 0);
            c.rows = max(0, min(min(DELTA_CHUNK, L - c.index * DELTA_CHUNK), T - c.row0));
            return true;
        }
        slot -= __builtin_amdgcn_readlane(upto, 63);
    }
    c.index = slot;
    return false;
}
// segment -> its first slot, its chunks and first row, by a whole wave
__device__ __forceinline__ void delta_segment(const int32_t *cu, int N, int seg, int &slot0, int &chunks, int &s0, int &L) {
    const int lane = threadIdx.x & 63;
    slot0 = 0;
    for (int base = 0; base < seg; base += 64) {
        const int i = min(base + lane, N - 1), len = cu[i + 1] - cu[i];
        slot0 += wave_sum_i(base + lane < seg && len > 0 ? (len + DELTA_CHUNK - 1) / DELTA_CHUNK : 0);
    }
    s0 = cu[seg];
    L = max(cu[seg + 1] - s0, 0);
    chunks = (L + DELTA_CHUNK - 1) / DELTA_CHUNK;
}

// What a wave's lanes wrote to LDS is there for its other lanes: the hardware keeps a wave's LDS operations in order, the compiler has to.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- fragments of mfma16 (16x16x32): lane l of a row-major tile ------------------------------------------------------------------------
// rows r0 + l%16, columns c0 + 8 (l/16) ..: an operand whose contraction runs along the row
__device__ __forceinline__ bf16x8 frag_n(const bf16_t *t, int stride, int r0, int c0, int l) {
    return *reinterpret_cast<const bf16x8 *>(t + (r0 + (l & 15)) * stride + c0 + 8 * (l >> 4));
}
// rows k0 + 8 (l/16) .., column m0 + l%16: an operand whose contraction runs down the rows
__device__ __forceinline__ bf16x8 frag_t(bf16_t *t, int stride, int k0, int m0, int l) {
    const int s = l & 15;
    bf16_t *const p = t + (k0 + 8 * (l >> 4) + (s >> 2)) * stride + m0 + 4 * (s & 3);
    return tr_pair((lds_u8 *)p, (lds_u8 *)(p + 4 * stride));
}
__device__ __forceinline__ bf16x8 frag_n(const bf16_t *t, int stride, int r0, int c0) { return frag_n(t, stride, r0, c0, threadIdx.x & 63); }
__device__ __forceinline__ bf16x8 frag_t(bf16_t *t, int stride, int k0, int m0) { return frag_t(t, stride, k0, m0, threadIdx.x & 63); }
// column c0 + l%16, rows r0 + 4 (l/16) + 0..3 and 16 further
__device__ __forceinline__ bf16x8 frag_column(bf16_t *t, int stride, int r0, int c0) {
    const int l = threadIdx.x & 63, s = l & 15;
    bf16_t *const p = t + (r0 + 4 * (l >> 4) + (s >> 2)) * stride + c0 + 4 * (s & 3);
    return tr_pair((lds_u8 *)p, (lds_u8 *)(p + 16 * stride));
}
// the lane as a value that the compiler knows nothing about: addresses made from it inside a loop are not carried into it in registers
__device__ __forceinline__ int fresh_lane() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

typedef uint32_t __attribute__((may_alias, ext_vector_type(2))) u32x2_any;
typedef uint32_t __attribute__((may_alias, ext_vector_type(4))) u32x4_any;
__device__ __forceinline__ u32x2 hi4(f32x4 x) { return u32x2{pack2bf(x[0], x[1]), pack2bf(x[2], x[3])}; }
// what hi4 left over
__device__ __forceinline__ u32x2 lo4(f32x4 x, u32x2 h) {
    return u32x2{pack2bf(x[0] - __uint_as_float(h[0] << 16), x[1] - __uint_as_float(h[0] & 0xffff0000u)),
                 pack2bf(x[2] - __uint_as_float(h[1] << 16), x[3] - __uint_as_float(h[1] & 0xffff0000u))};
}
__device__ __forceinline__ void put4(bf16_t *p, u32x2 x) { *reinterpret_cast<u32x2_any *>(p) = x; }
__device__ __forceinline__ void put_split4(bf16_t *h, bf16_t *l, f32x4 x) {
    const u32x2 a = hi4(x);
    put4(h, a);
    put4(l, lo4(x, a));
}

// ---- tiles of 64 rows by 256 threads: global -> registers -> LDS -------------------------------------------------------------------------
template <int W> struct Tile64 { u32x4 x[W / 32]; };
// rows of `width` (a multiple of 8, at most W) elements, `tok` elements apart; beyond `rows` and `width` zero
template <int W>
__device__ __forceinline__ void tile_load(Tile64<W> &t, const bf16_t *src, int64_t tok, int rows, int width) {
#pragma unroll
    for (int u = 0; u < W / 32; ++u) {
        const int i = threadIdx.x + 256 * u, r = i / (W / 8), c = i % (W / 8) * 8;
        t.x[u] = r < rows && c < width ? *reinterpret_cast<const u32x4 *>(src + r * tok + c) : u32x4{0u, 0u, 0u, 0u};
    }
}
template <int W>
__device__ __forceinline__ void tile_put(const Tile64<W> &t, bf16_t *lds, int stride) {
#pragma unroll
    for (int u = 0; u < W / 32; ++u) {
        const int i = threadIdx.x + 256 * u;
        *reinterpret_cast<u32x4_any *>(lds + i / (W / 8) * stride + i % (W / 8) * 8) = t.x[u];
    }
}
template <int W>
__device__ __forceinline__ void tile_copy(bf16_t *lds, int stride, const bf16_t *src, int64_t tok, int rows, int width) {
    Tile64<W> t;
    tile_load<W>(t, src, tok, rows, width);
    tile_put<W>(t, lds, stride);
}

// ---- memory through buffers: a wave-uniform start, an offset per lane that stays the same from chunk to chunk, zeros past the end (and nothing
// written there).  A lane that has nothing to read or write gets the offset NOWHERE once, in front of the loop; no address is formed inside it.
// (With 64-bit addresses and masks formed per chunk a walk of 512 chunks took 1.74 ms, most of it their arithmetic.)
#define NOWHERE 0x7fffff00
__device__ __forceinline__ int further(int off, int by) { return (int)((uint32_t)off + (uint32_t)by); }       // (from NOWHERE on still past any end)
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const void *p, int bytes) {
    const int64_t a = reinterpret_cast<int64_t>(p);
    const int64_t u = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)a) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) << 32);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
// rows of a strided tensor: from the first row's first element, `rows` rows `tok` elements apart of `width` elements
__device__ __forceinline__ buffer_t rows_buffer(const char *p, int tok, int rows, int width) { return buffer_of(p, rows > 0 ? ((rows - 1) * tok + width) * 2 : 0); }
// `at`: a constant that the end is not checked for
__device__ __forceinline__ bf16x8 buf16(buffer_t b, int off, int at = 0) { return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(b, off, at, 0)); }
__device__ __forceinline__ float buf4(buffer_t b, int off) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, off, 0, 0)); }
__device__ __forceinline__ void buf_put8(buffer_t b, int off, u32x2 x) { __builtin_amdgcn_raw_buffer_store_b64(x, b, off, 0, 0); }
// every load so far has arrived: in front of a loop whose loads are waited for by count (what is in flight there from before would be counted in with them)
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }
// (Never with a scalar offset: the compiler then leaves out the wait state between a 16-byte store and an instruction that overwrites what it stores, and
// stored values came out wrong here and there.)
__device__ __forceinline__ void buf_put16(buffer_t b, int off, u32x4 x) { __builtin_amdgcn_raw_buffer_store_b128(x, b, off, 0, 0); }
// the same, past the caches: what only the chunks' gradients will read (walks of 33 sequences of 16 384 rows together, of 1 of 32 768 and of 4 of 4096, forward / backward:
// 328 / 369 us -> 326 / 356, 1084 / 1179 -> 1073 / 1139, 372 / 385 -> 366 / 374; outputs so, whose lines come in parts, cost 50 us of the first).
__device__ __forceinline__ void buf_put16_past(buffer_t b, int off, u32x4 x) { __builtin_amdgcn_raw_buffer_store_b128(x, b, off, 0, 2); }
// four or eight elements at a time
template <int N> struct Piece { uint32_t x[N / 2]; };
template <int N> __device__ __forceinline__ Piece<N> buf_piece(buffer_t b, int off) {
    if constexpr (N == 8) return __builtin_bit_cast(Piece<8>, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
    else return __builtin_bit_cast(Piece<4>, __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, 0));
}
template <int N> __device__ __forceinline__ void buf_put_piece_past(buffer_t b, int off, Piece<N> p) {
    if constexpr (N == 8) buf_put16_past(b, off, __builtin_bit_cast(u32x4, p));
    else buf_put8(b, off, __builtin_bit_cast(u32x2, p));
}
template <int N> __device__ __forceinline__ void buf_put_piece(buffer_t b, int off, Piece<N> p) {
    if constexpr (N == 8) buf_put16(b, off, __builtin_bit_cast(u32x4, p));
    else buf_put8(b, off, __builtin_bit_cast(u32x2, p));
}
// LDS, on 8-byte boundaries
template <int N> __device__ __forceinline__ void put_piece(bf16_t *t, Piece<N> p) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) *reinterpret_cast<u32x2_any *>(t + 4 * i) = u32x2{p.x[2 * i], p.x[2 * i + 1]};
}
template <int N> __device__ __forceinline__ Piece<N> get_piece(const bf16_t *t) {
    Piece<N> p;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const u32x2 x = *reinterpret_cast<const u32x2_any *>(t + 4 * i);
        p.x[2 * i] = x[0];
        p.x[2 * i + 1] = x[1];
    }
    return p;
}
// 16 bytes of a row from column c on, zero where there is none
__device__ __forceinline__ bf16x8 row_frag(const bf16_t *row, int c, bool in) {
    return in ? *reinterpret_cast<const bf16x8 *>(row + c) : zero_bf16x8();
}
__device__ __forceinline__ f32x4 up4(u32x2 x) {
    return f32x4{__uint_as_float(x[0] << 16), __uint_as_float(x[0] & 0xffff0000u), __uint_as_float(x[1] << 16), __uint_as_float(x[1] & 0xffff0000u)};
}

// The r-th longest segment, so that no long walk begins when the others end (64 segments at most: more even out by themselves)
__device__ __forceinline__ int delta_longest(const int32_t *cu, int N, int r) {
    if (N > 64) return r;
    const int lane = threadIdx.x & 63, i = min(lane, N - 1), n = lane < N ? max(cu[i + 1] - cu[i], 0) : -1;
    int rank = 0;
    for (int j = 0; j < N; ++j) {
        const int o = __builtin_amdgcn_readlane(n, j);
        rank += o > n || (o == n && j < lane);
    }
    return (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < N && rank == r));
}

// How the state's walks are split over workgroups.  A head's chunk takes
//     DELTA_ONE   eight of 16 columns (dsa_delta_chain.hip)       1.7 to 2.2 us alone, a third more work
//     DELTA_TWO   four of 32 columns (there too)                  2.5 to 3.1 us alone, 4 to 5.9 for two that share a compute unit
//     DELTA_HEAD  one, heads of 128 (dsa_delta_walk.hip)          6 us alone, 8.5 with its like on all compute units, when memory bounds it
// so it depends on how many walks as long as the longest all chunks would make, r: little more than one workgroup of the first for each compute unit, up to 150 heads
// of the second, then the third.  Forward / backward with 32 heads, us, the three:
//     r    32   1 of 32 768          1030 / 1138   1307 / 1325
//          39   4000, 1, 63, 700      139 / 143     166 / 171
//          64   2 of 8192             532 / 510     361 / 425
//          95   8 of 200 .. 4000                    245 / 263     450 / 431
//         128   4 of 4096             525 / 505     334 / 370     486 / 489
//         160   5 of 3200                           396 / 414     392 / 415
//         256   8 of 2048                           361 / 379     276 / 309
//         334   33 of 65 .. 1669                    382 / 409     319 / 349
// The lengths are on the device: where more than one form can be right the launches of the others look, and end (4.5 us each).
enum { DELTA_ONE = 1, DELTA_TWO = 2, DELTA_HEAD = 3 };
__host__ __device__ __forceinline__ int delta_form_of(const DeltaArgs &a, int64_t chunks_heads, int64_t longest) {
    if (chunks_heads * (a.Dvp / 16) * 3 <= longest * 1024) return DELTA_ONE;
    return a.Dkp == 128 && a.Dvp == 128 && chunks_heads >= longest * 150 ? DELTA_HEAD : DELTA_TWO;
}
// by a whole wave
__device__ __forceinline__ int delta_form(const DeltaArgs &a) {
    const dsa_delta_args &in = a.in;
    const int lane = threadIdx.x & 63;
    int all = 0, longest = 0;
    for (int base = 0; base < in.N; base += 64) {
        const int i = min(base + lane, in.N - 1), len = in.cu[i + 1] - in.cu[i];
        const int n = base + lane < in.N && len > 0 ? (len + DELTA_CHUNK - 1) / DELTA_CHUNK : 0;
        all += wave_sum_i(n);
        longest = max(longest, n);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) longest = max(longest, __shfl_xor(longest, m, 64));
    const int form = delta_form_of(a, (int64_t)all * in.Hv, __builtin_amdgcn_readfirstlane(longest));
    return form == DELTA_ONE && !a.maybe_one ? DELTA_TWO : form;
}

// Which walk a workgroup takes: the column blocks of one head on one of the chip's eight dies (consecutive workgroups go round them), where they find the
// rows that they share in its L2.  False: a spare workgroup.
__device__ __forceinline__ bool delta_walk_unit(int id, int blocks, int64_t units, int64_t &unit, int &block) {
    const int die = id & 7, j = id >> 3;
    unit = (int64_t)(j / blocks) * 8 + die;
    block = j % blocks;
    return unit < units;
}

__device__ __forceinline__ float load_any(const void *p, int64_t i, int f32) {
    return f32 ? reinterpret_cast<const float *>(p)[i] : (float)reinterpret_cast<const bf16_t *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, int64_t i, int f32, float x) {
    if (f32) reinterpret_cast<float *>(p)[i] = x;
    else reinterpret_cast<bf16_t *>(p)[i] = (bf16_t)x;
}
__device__ __forceinline__ float softplus_f(float x) { return x > 20.f ? x : log1pf(expf(x)); }
// e^x for x <= 0 between rows of a chunk: off by |x| 2^-24 of its value, next to the 2^-18 that it loses in the products
__device__ __forceinline__ float delta_decay(float x) { return __builtin_amdgcn_exp2f(fminf(x, 0.f) * 1.442695041f); }
// the log decay of a row.  Held above -1e4, where e^g has long been zero: a decay of -inf would make G_i - G_j of later rows NaN.  (A NaN stays one.)
__device__ __forceinline__ float delta_gate(const dsa_delta_args &in, int64_t t, int h) {
    const float x = load_any(in.a, t * in.a_tok + h, in.a_f32) + load_any(in.dt_bias, h, in.param_f32);
    const float g = -expf(load_any(in.a_log, h, in.param_f32)) * softplus_f(x);
    return g < -1e4f ? -1e4f : g;
}
__device__ __forceinline__ float delta_beta(const dsa_delta_args &in, int64_t t, int h) {
    return 1.f / (1.f + expf(-load_any(in.b, t * in.b_tok + h, in.b_f32)));
}
