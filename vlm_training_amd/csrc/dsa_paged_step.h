// Attention of a few rows over a paged cache, and the joining of pieces.
//
// A workgroup takes up to 16 RG rows - a row is one (query, head of the kv group) - of one request and kv head, and a piece of its keys; its waves take the
// piece's tiles of 32 keys in turn, each by itself:
//   S^T[key,row] = K[key,:].Q[row,:]            (A = K tile row-wise from LDS, B = Q^T in registers)
//   online softmax on the C layout (lane = row, 8 keys a lane)
//   O^T[d,row]  += V^T[d,key] P^T[key,row]      (A = V tile transposed from LDS, B = P^T as it lies; keys 4 g .. 4 g + 3 and 16 more of lane group g on both sides)
// Every wave has its own tiles in LDS, two of them, filled straight from memory (bf16), or one, into which it writes the values that it has loaded as e4m3 in front
// of the last tile's products: no barrier until the waves' sums are joined.  Pieces of a block are joined by dsa_paged_join_kernel, in order.
//
// P is rounded to bf16 for the second product (each probability by at most 2^-8 of itself, at random); its sum, the statistics and the output's sums are fp32.
//
// What bounds it: memory.  256 requests over an 8-bit cache of 2.3 GB 434 us (5.4 TB/s with the join), 64 requests of 64 to 8192 bf16 keys 90 us (5.0), one of 131 072 with two heads of
// 256 64 us (4.2); short batches by the chain of a piece's first loads: offsets and lengths, page numbers, rows, 2 to 3 us, and 1 for the waves' join (one token over 1000 keys:
// 6.5 us, the join 3.8).  16-row MFMAs: a decoded token's heads are 1 to 16 rows, and two tiles' products of 32-row MFMAs would take as long again.  Sums in vector registers (the
// compiler's flag for it): with 64 to 128 accumulation registers and their copies one long request took 54 us instead of 48.
// Two or four workgroups of fewer waves to a unit, waves' tiles two ahead instead of one in an 8-bit cache: within 2 %.  Equal shares instead of equal pieces of each
// request: 64 requests 99 -> 90, drafts of 24 36 -> 28, two requests of 131 072 and 77 level.
#pragma once
#include "dsa_paged.h"

__device__ __forceinline__ float group_max(float v) {                   // over the four lanes 16 apart
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <int D, bool E4M3, int RG, int RING = 2>
constexpr int step_wave_bytes() {
    const int ring = (E4M3 ? 2 : 2 * RING) * DirectTile<D>::BYTES, sums = RG * 16 * (D + 4) * 4 + RG * 16 * 8;
    return ring > sums ? ring : sums;
}

// RING: tiles that a wave of a bf16 cache has in LDS
template <int D, bool E4M3, int RG, int NW, int RING = 2>
__device__ __forceinline__ void paged_step(const dsa_cache_args &c, const PagePlan &plan, const bf16_t *__restrict__ q, int64_t q_tok, int64_t q_head, int Hq, int gshift, int pshift,
                                           float scale_log2, int tail, bf16_t *__restrict__ out, float *__restrict__ lse, float *__restrict__ part_o, float *__restrict__ part_ml,
                                           int share, int kvh) {
    typedef DirectTile<D> TL;
    constexpr int KS = D / 32, DT = D / 16, ROWS = 16 * RG, PITCH = D + 4;
    constexpr int WAVE_B = step_wave_bytes<D, E4M3, RG, RING>();
    extern __shared__ __attribute__((aligned(1024))) unsigned char dyn_lds[];
    const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hkv = c.Hkv, G = Hq / Hkv, T = plan.T, d_real = c.D;
    ShareWalk walk;
    walk.start(plan, share);
    PagePiece pc;
    while (walk.next(plan, pc)) {
    const int keys = min(pc.length, plan.capacity);      // positions that exist
    const int chunks = d_real / 8;

    // rows: their q, and the last position each attends (rows that are none, and those of no keys: whatever the block does)
    bf16x8 qB[RG][KS];
    int klim[RG];
    const int past = pc.length - pc.m, block_last = past + min(pc.first + plan.qb, pc.m) - 1;
    auto query_of = [&](int row) { return pc.first + (row >> gshift); };
    auto live = [&](int row) { return (row >> gshift) < plan.qb && query_of(row) < pc.m && (row & ((1 << gshift) - 1)) < G; };
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const int row = rg * 16 + j;
        const bool ok = live(row);
        klim[rg] = min(ok ? past + query_of(row) : block_last, keys - 1);
        const bf16_t *const src = q + (int64_t)(pc.row0 + min(query_of(row), pc.m - 1)) * q_tok + (int64_t)(kvh * G + min(row & ((1 << gshift) - 1), G - 1)) * q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qB[rg][ks] = ok && 4 * ks + g < chunks ? load_bf16x8(src + 32 * ks + 8 * g) : zero_bf16x8();
    }
    const bool one_limit = pc.m == 1;                    // every row attends all keys that there are

    // ---- tiles ----
    unsigned char *const ring = dyn_lds + wv * WAVE_B;   // K | V, or K | V | K | V
    const uint32_t lds0 = lds_address(dyn_lds) + wv * WAVE_B;
    const __attribute__((address_space(4))) int32_t *const ids = (const __attribute__((address_space(4))) int32_t *)(c.table + (int64_t)pc.n * c.table_row);
    auto page_id = [&](int p) __attribute__((always_inline)) {           // of position p (wave-uniform), -1 where nothing lies
        const int at = __builtin_amdgcn_readfirstlane(p >> pshift);
        const int id = at < c.table_pages ? ids[at] : -1;
        return (uint32_t)id < (uint32_t)c.pages ? id : -1;
    };
    int voff[TL::SOURCES];
    if constexpr (!E4M3) {
#pragma unroll
        for (int i = 0; i < TL::SOURCES; ++i) voff[i] = TL::source(i, lane, d_real * 2, chunks);
    }
    auto request = [&](int tile, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int p = tile * 32 + 16 * hf, id = page_id(p);
            const int64_t at = ((int64_t)kvh * c.page + (p & (c.page - 1))) * d_real;
            const int bytes = id < 0 ? 0 : min(max(keys - p, 0), 16) * d_real * 2;
#pragma unroll
            for (int op = 0; op < 2; ++op) {
                const bf16_t *const pool = op ? (const bf16_t *)c.v + max(id, 0) * c.v_page : (const bf16_t *)c.k + max(id, 0) * c.k_page;
                const buffer_rsrc rs = make_buffer_rsrc(pool + at, bytes);
#pragma unroll
                for (int i = 0; i < TL::LOADS / 2; ++i)
                    buffer_load_lds16(rs, voff[i % TL::SOURCES] + i / TL::SOURCES * TL::SOURCES * TL::LOAD_ROWS * d_real * 2,
                                      lds0 + (2 * slot + op) * TL::BYTES + TL::load_lds(hf * (TL::LOADS / 2) + i));
            }
        }
    };
    // e4m3: a lane has 16 values of rows NL (lane / LPR) .. + NL - 1 (lanes 0 .. 31 the first 16 rows of a tile), one load each
    constexpr int LPR = D / 16, NL = D / 32;
    typedef uint32_t codes_t __attribute__((ext_vector_type(4)));
    codes_t raw[E4M3 ? 2 : 1][E4M3 ? NL : 1];
    uint32_t ex[2][NL > 4 ? 2 : 1];
    const int e_row = NL * (lane / LPR), e_chunk = lane % LPR;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        const int p0 = tile * 32, id0 = page_id(p0), id1 = page_id(p0 + 16);
        const int id = lane < 32 ? id0 : id1, p = p0 + e_row;
        const int64_t row = (int64_t)kvh * c.page + (p & (c.page - 1));
#pragma unroll
        for (int op = 0; op < 2; ++op) {
            const uint8_t *const src = (op ? (const uint8_t *)c.v + max(id, 0) * c.v_page : (const uint8_t *)c.k + max(id, 0) * c.k_page) + row * d_real + 16 * e_chunk;
            const uint8_t *const se = (op ? (const uint8_t *)c.v_exp + max(id, 0) * c.vx_page : (const uint8_t *)c.k_exp + max(id, 0) * c.kx_page) + row;
#pragma unroll
            for (int i = 0; i < NL; ++i) raw[op][i] = id >= 0 && 16 * e_chunk < d_real ? *reinterpret_cast<const codes_t *>(src + i * d_real) : codes_t{0u, 0u, 0u, 0u};
            if constexpr (NL == 2) ex[op][0] = id >= 0 ? *reinterpret_cast<const uint16_t *>(se) : 0u;
            if constexpr (NL == 4) ex[op][0] = id >= 0 ? *reinterpret_cast<const uint32_t *>(se) : 0u;
            if constexpr (NL == 8) {
                const u32x2 w = id >= 0 ? *reinterpret_cast<const u32x2 *>(se) : u32x2{0u, 0u};
                ex[op][0] = w[0];
                ex[op][NL > 4 ? 1 : 0] = w[1];
            }
        }
    };
    auto unpack = [&](int tile) __attribute__((always_inline)) {
        const bool all = tile * 32 + 32 <= keys;
#pragma unroll
        for (int op = 0; op < 2; ++op)
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int r = e_row + i;
                const bool gone = !all && tile * 32 + r >= keys;        // (what lies behind the last key, values and powers, may be anything)
                const float s = exponent_scale(gone ? 127u : (ex[op][i >> 2] >> (8 * (i & 3))) & 0xff);
                const codes_t w = gone ? codes_t{0u, 0u, 0u, 0u} : raw[op][i];
                const u32x2 a = e4m3_to_bf16(w[0], s), b = e4m3_to_bf16(w[1], s), x = e4m3_to_bf16(w[2], s), y = e4m3_to_bf16(w[3], s);
                unsigned char *const to = ring + op * TL::BYTES + r / TL::GROUP * TL::GROUP_B + r % TL::GROUP * TL::ROW_B;
                *reinterpret_cast<u32x4 *>(to + (((2 * e_chunk) ^ TL::xor_of(r)) << 4)) = u32x4{a[0], a[1], b[0], b[1]};
                *reinterpret_cast<u32x4 *>(to + (((2 * e_chunk + 1) ^ TL::xor_of(r)) << 4)) = u32x4{x[0], x[1], y[0], y[1]};
            }
    };
    // operand addresses
    int ka[4], va[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int i = j >> 2, hi = (j & 3) >> 1, sub = (j & 1) << 3, vr = 4 * g + i;
        const int kb = j / TL::GROUP * TL::GROUP_B + j % TL::GROUP * TL::ROW_B, vb = vr / TL::GROUP * TL::GROUP_B + vr % TL::GROUP * TL::ROW_B;
        ka[b] = D == 64 ? kb + (((4 * (b & 1) + g) ^ TL::xor_of(j)) << 4) : kb + ((4 * (b ^ (j & 3)) + g) << 4);
        va[b] = D == 64 ? vb + (((2 * b + hi) ^ TL::xor_of(vr)) << 4) + sub : vb + ((4 * (b ^ i) + hi) << 4) + sub;
    }
    constexpr int HALF = 16 / TL::GROUP * TL::GROUP_B;   // bytes to the tile's second sixteen rows
    auto read_k = [&](int kt, int ks, int slot) __attribute__((always_inline)) {
        return *reinterpret_cast<const bf16x8 *>(ring + 2 * slot * TL::BYTES + ka[ks & 3] + kt * HALF + (D == 64 ? 0 : (ks >> 2) * 256));
    };
    auto read_v = [&](int dt, int slot) __attribute__((always_inline)) {
        lds_u8 *const at = (lds_u8 *)ring + (2 * slot + 1) * TL::BYTES + (D == 64 ? va[dt & 3] : va[(dt >> 1) & 3] + (dt >> 3) * 256 + (dt & 1) * 32);
        return tr_pair(at, at + HALF);
    };

    f32x4 oacc[RG][DT];
    float mrun[RG], lsum[RG];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        mrun[rg] = -INFINITY;
        lsum[rg] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[rg][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int tile0 = pc.tile0 + wv, tile1 = pc.tile1;
    const int low_last = min(past + pc.first, keys - 1);  // the least position that a row of the block attends up to
    auto compute = [&](int tile, int slot) __attribute__((always_inline)) {
        const bool masked = tile * 32 + 31 > low_last;
        bf16x8 pB[RG];
        float p[RG][8];
        f32x4 s[RG][2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) s[rg][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 a = read_k(kt, ks, slot);
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) s[rg][kt] = mfma16(a, qB[rg][ks], s[rg][kt]);
            }
        }
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
            float y[8], most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = s[rg][e >> 2][e & 3] * scale_log2;
                if (masked && tile * 32 + (e >> 2) * 16 + 4 * g + (e & 3) > klim[rg]) y[e] = -INFINITY;
                most = fmaxf(most, y[e]);
            }
            most = group_max(most);
            const float m = fmaxf(mrun[rg], most);
            if (__builtin_amdgcn_ballot_w64(m > mrun[rg])) {
                const float alpha = mrun[rg] == -INFINITY ? 0.f : fast_exp2(mrun[rg] - m);
                lsum[rg] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) oacc[rg][dt] *= alpha;
                mrun[rg] = m;
            }
            const float neg = m == -INFINITY ? 0.f : -m;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[rg][e] = fast_exp2(y[e] + neg);
                lsum[rg] += p[rg][e];
            }
            pB[rg] = pack8(p[rg]);
        }
        // keys that some rows of the block do not attend: their zero probabilities must not meet an infinite or NaN value
        bool odd = false;
        if (masked && !one_limit) {
            uint32_t bad = 0;
            for (int i = lane; i < 32 * TL::CPR; i += 64) {
                const int r = i / TL::CPR;
                const u32x4 w = *reinterpret_cast<const u32x4 *>(ring + (2 * slot + 1) * TL::BYTES + r / TL::GROUP * TL::GROUP_B + r % TL::GROUP * TL::ROW_B + i % TL::CPR * 16);
#pragma unroll
                for (int x = 0; x < 4; ++x) bad |= ((w[x] & 0x7f80u) == 0x7f80u) | ((w[x] & 0x7f800000u) == 0x7f800000u);
            }
            odd = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        }
        if (!odd) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8 a = read_v(dt, slot);
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) oacc[rg][dt] = mfma16(a, pB[rg], oacc[rg][dt]);
            }
        } else {
            // one key after the other, those that a row attends alone
            for (int key = 0; key < 32; ++key) {
                const unsigned char *const vrow = ring + (2 * slot + 1) * TL::BYTES + key / TL::GROUP * TL::GROUP_B + key % TL::GROUP * TL::ROW_B;
                const int x = TL::xor_of(key), e = (key >> 4) * 4 + (key & 3);
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) {
                    float mine = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) mine = i == e ? p[rg][i] : mine;
                    const float pr = __uint_as_float(pack2bf(__shfl(mine, ((key & 15) >> 2) * 16 + j, 64), 0.f) << 16);          // (as the product takes it)
                    const bool attends = tile * 32 + key <= klim[rg];
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const int d = 16 * dt + 4 * g + v;
                            const float val = (float)*reinterpret_cast<const bf16_t *>(vrow + (((d >> 3) ^ x) << 4) + (d & 7) * 2);
                            if (attends) oacc[rg][dt][v] = fmaf(pr, val, oacc[rg][dt][v]);
                        }
                }
            }
        }
    };
    if constexpr (E4M3) {
        if (tile0 < tile1) fetch(tile0);
        for (int tile = tile0; tile < tile1; tile += NW) {
            unpack(tile);
            if (tile + NW < tile1) fetch(tile + NW);
            compute(tile, 0);
        }
    } else {
        if (tile0 < tile1) request(tile0, 0);
        if (RING == 2 && tile0 + NW < tile1) request(tile0 + NW, 1);
        int slot = 0;
        for (int tile = tile0; tile < tile1; tile += NW) {
            if (RING == 2 && tile + NW < tile1) wait_vmcnt<2 * TL::LOADS>();
            else wait_vmcnt<0>();
            compute(tile, slot);
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");        // (the tile is read out before it is filled again)
            if (tile + RING * NW < tile1) request(tile + RING * NW, slot);
            if (RING == 2) slot ^= 1;
        }
    }

    // ---- the waves' sums, joined ----
    float *const sums = reinterpret_cast<float *>(dyn_lds + wv * WAVE_B), *const stats = sums + ROWS * PITCH;
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const float l = group_sum(lsum[rg]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(sums + (rg * 16 + j) * PITCH + 16 * dt + 4 * g) = oacc[rg][dt];
        if (g == 0) {
            stats[2 * (rg * 16 + j)] = row_maximum(mrun[rg], l);
            stats[2 * (rg * 16 + j) + 1] = l;
        }
    }
    __syncthreads();
    const int rows = plan.qb << gshift;
    const bool whole = pc.pieces == 1;
    const int64_t record = (int64_t)pc.slot * Hkv + kvh;
    for (int i = tid; i < rows * chunks; i += NW * 64) {
        const int row = i / chunks, d = i % chunks * 8;
        if (!live(row)) continue;
        float m = -INFINITY, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        const unsigned char *at = dyn_lds;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, reinterpret_cast<const float *>(at + w * WAVE_B)[ROWS * PITCH + 2 * row]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float *const ws = reinterpret_cast<const float *>(at + w * WAVE_B);
            const float mw = ws[ROWS * PITCH + 2 * row], f = mw == -INFINITY ? 0.f : fast_exp2(mw - m);
            l = fmaf(f, ws[ROWS * PITCH + 2 * row + 1], l);
            if (mw != -INFINITY) {
                const f32x4 a = *reinterpret_cast<const f32x4 *>(ws + row * PITCH + d), b = *reinterpret_cast<const f32x4 *>(ws + row * PITCH + d + 4);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    o[x] = fmaf(f, a[x], o[x]);
                    o[4 + x] = fmaf(f, b[x], o[4 + x]);
                }
            }
        }
        if (whole) {
            const int64_t t = pc.row0 + query_of(row), hq = kvh * G + (row & ((1 << gshift) - 1));
            const float inv = m == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] *= inv;
            *reinterpret_cast<bf16x8 *>(out + (t * Hq + hq) * d_real + d) = pack8(o);
            if (lse && d == 0) lse[hq * T + t] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * LN2_F;
        } else {
            float *const to = part_o + (record * rows + row) * d_real + d;
            *reinterpret_cast<f32x4 *>(to) = f32x4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<f32x4 *>(to + 4) = f32x4{o[4], o[5], o[6], o[7]};
            if (d == 0) *reinterpret_cast<f32x2 *>(part_ml + (record * rows + row) * 2) = f32x2{m, l};
        }
    }
    __syncthreads();                                     // the sums are read: the next piece's tiles may come
    }
    if (tail) zero_tail(plan, Hq, Hkv, kvh, share, plan.target, d_real, NW * 64, out, lse);
}
