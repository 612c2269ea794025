// Attention of a chunk of new tokens over a paged cache: the pipelined walk of dsa_tile_fwd.hip, its tiles taken from pages.
//
// A workgroup holds 128 rows - a row is one (query, head of the kv group) - of one request and kv head and walks a piece of its keys in tiles of 32, shared by its four
// waves:
//   S^T[key,row] = K[key,:].Q[row,:]            (A = K tile row-wise from LDS, B = Q^T in registers)
//   online softmax on the C layout (lane = row; one cross-lane step per statistic)
//   O^T[d,row]  += V^T[d,key] P^T[key,row]      (A = V tile transposed from LDS, B = P^T from the C layout)
// Step t issues the MFMAs of O += P(t) V(t) and of S(t+2) in pairs, with the softmax of tile t+1 between them.
//
// Every wave brings eight rows of each tile, which lie on one page whatever its size; their page's number comes from a ring in LDS (two batches of 64 numbers a
// wave, the next one requested as soon as the one before the last is done with: dsa_paged_ring.h).  A bf16 cache: rows go from memory straight into LDS, K five tiles ahead, V three.  An 8-bit
// one: values are loaded into registers a step ahead of the one that writes them to LDS as bf16, K(t+4) and V(t+2) in step t: one conversion for 128 rows, and no rounding, as
// the scales are powers of two.
//
// What bounds it: as the packed forward, power and the instructions beside the MFMAs.  2048 new tokens behind 14 336 (32 heads over 8 of 128) 472 to 485 us = 1.06 to 1.09 PFLOP/s (16 over 2 of 256: 488, 8-bit 573), MFMA busy 0.6 of the
// units' time; page addresses formed in 64 bits for each operand cost 8 % of it, two long walks on one unit (the second half of a launch of one round goes in reverse) 3 %.
// An 8-bit cache: 1024 behind 60 000 1370 to 1390 us (bf16 1110); the loads two steps ahead instead of one left no registers for operands four MFMAs ahead (1498), and converting in
// the loads' own step spilled.  A chunk of 512 behind 7680 and a prompt of 333: 93 us, of them 8 for the first loads and 8 for the pieces' sums (33 MB).
#pragma once
#include "dsa_paged.h"
#include "dsa_paged_ring.h"

constexpr int WALK_WAVES = 4;
template <int D>
constexpr int walk_lds_bytes() { return 8 * DirectTile<D>::BYTES + WALK_WAVES * 512 + 16; }

// AGPR: the sums in accumulation registers, by name (mfma32_agpr_late); VA: operands of V read ahead (divides NP)
template <int D, bool E4M3, bool AGPR, int VA = 4>
__device__ __forceinline__ void paged_walk(const dsa_cache_args &c, const PagePlan &plan, const bf16_t *__restrict__ q, int64_t q_tok, int64_t q_head, int Hq, int gshift, int pshift,
                                           float scale_log2, uint32_t flip, int slots, int tail, bf16_t *__restrict__ out, float *__restrict__ lse, float *__restrict__ part_o,
                                           float *__restrict__ part_ml, int slot, int kvh) {
    typedef DirectTile<D> TL;
    constexpr int NW = WALK_WAVES, KS = D / 16, DT = D / 32, NP = 2 * DT, NS = KS > NP ? KS : NP;
    constexpr int LPW = TL::LOADS / NW;                     // wave loads per wave, step and operand (bf16)
    constexpr int LPS = E4M3 ? (D == 256 ? 8 : 4) : 2 * LPW;   // everything a wave requests in a step, ids apart
    extern __shared__ __attribute__((aligned(1024))) unsigned char dyn_lds[];    // 4 K slots | 4 V slots | page numbers

    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, j = lane & 31;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hkv = c.Hkv, G = Hq / Hkv, T = plan.T, d_real = c.D, chunks = d_real / 8;
    PagePiece pc;
    int spare;
    if (!locate_piece<false>(plan, slot, pc, spare)) {
        if (tail) zero_tail(plan, Hq, Hkv, kvh, slot - spare, slots - spare, d_real, NW * 64, out, lse);
        return;
    }
    if (pc.piece >= pc.pieces) return;
    const int keys = min(pc.length, plan.capacity), past = pc.length - pc.m;
    const int r = wv * 32 + j, query = pc.first + (r >> gshift), head = r & ((1 << gshift) - 1);
    const bool row_ok = query < pc.m && head < G;
    const int t = pc.row0 + min(query, pc.m - 1), hq = kvh * G + min(head, G - 1);
    const int klim = min(past + query, keys - 1);           // last key this row attends
    const int base = pc.tile0, ntiles = pc.tile1 - pc.tile0;    // tiles are counted from the piece's first
    const bool whole_out = pc.pieces == 1;
    const int64_t record = ((int64_t)(pc.slot + pc.piece) * Hkv + kvh) * (plan.qb << gshift) + r;

    float mrun = -INFINITY, lsum = 0.f;
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        oacc[dt] = zero16();
        if (AGPR) settle(oacc[dt]);
    }
    auto finish = [&]() __attribute__((always_inline)) {
        const float l = half_sum_f(lsum);
        mrun = row_maximum(mrun, l);
        if (AGPR) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) settle(oacc[dt]);
        }
        if (!row_ok) return;
        if (whole_out) {
            const float inv = mrun == -INFINITY ? 0.f : 1.f / l;
            if (lse && h == 0) lse[(int64_t)hq * T + t] = mrun == -INFINITY ? -INFINITY : (mrun + log2f(l)) * LN2_F;
            bf16_t *const row = out + ((int64_t)t * Hq + hq) * d_real;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) store_c_tile(row + dt * 32, oacc[dt], inv, h, chunks - 4 * dt);
        } else {
            if (h == 0) *reinterpret_cast<f32x2 *>(part_ml + 2 * record) = f32x2{mrun, l};
            float *const row = part_o + record * d_real;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    if (4 * dt + g4 < chunks)
                        *reinterpret_cast<f32x4 *>(row + 32 * dt + 8 * g4 + 4 * h) = f32x4{oacc[dt][4 * g4], oacc[dt][4 * g4 + 1], oacc[dt][4 * g4 + 2], oacc[dt][4 * g4 + 3]};
        }
    };
    if (ntiles == 0) {                                       // rows without any key
        finish();
        return;
    }

    // ---- pages ----
    const uint32_t lds0 = lds_address(dyn_lds);
    const int32_t *const mine = reinterpret_cast<const int32_t *>(dyn_lds + 8 * TL::BYTES + wv * 512);
    const uint32_t ids0 = lds0 + 8 * TL::BYTES + wv * 512;
    const int32_t *const table = c.table + (int64_t)pc.n * c.table_row;
    auto load_ids = [&](int batch) __attribute__((always_inline)) {      // numbers of pages 64 batch .. + 63
        const int from = batch * 64, there = max(min(c.table_pages - from, 64), 0);
        buffer_load_lds4(make_buffer_rsrc(table + min(from, c.table_pages), there * 4), lane * 4, ids0 + (batch & 1) * 256);
    };
    // Where the wave's rows of a tile lie.  All of it is scalar and short: scalar instructions too are issued in between the MFMAs (64-bit products of element strides, formed
    // for each operand and tile, were 130 a step)
    const int row0 = __builtin_amdgcn_readfirstlane(base * 32 + 8 * wv), end = __builtin_amdgcn_readfirstlane(min(keys, (base + ntiles) * 32)), pmask = c.page - 1;
    const uint32_t row_b = d_real * (E4M3 ? 1 : 2), k_stride = (uint32_t)c.k_page * (E4M3 ? 1u : 2u), v_stride = (uint32_t)c.v_page * (E4M3 ? 1u : 2u);
    const unsigned char *const k_pool = (const unsigned char *)c.k + (int64_t)kvh * c.page * row_b, *const v_pool = (const unsigned char *)c.v + (int64_t)kvh * c.page * row_b;
    auto page_at = [&](int tile) __attribute__((always_inline)) {        // number of their page: looked up one step ahead of its use
        return mine[PageRing::place((row0 + tile * 32) >> pshift)];
    };
    struct Where { uint32_t id, rows, place; };             // page, rows that exist, the first one's place among the page's
    auto where = [&](int tile, int id_) __attribute__((always_inline)) {
        const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane(id_), p = row0 + tile * 32;
        const int left = max(end - (int)p, 0);
        int rows = left;
        asm("s_min_i32 %0, %0, 8" : "+s"(rows) : : "scc");  // (a clamp would go through the vector pipe and come back)
        const bool there = id < (uint32_t)c.pages;
        return Where{there ? id : 0u, there ? (uint32_t)rows : 0u, p & pmask};
    };
    auto address = [&](const unsigned char *pool, uint32_t stride, const Where &w, uint32_t bytes) __attribute__((always_inline)) {
        return pool + (uint64_t)w.id * stride + w.place * bytes;
    };

    // ---- requests: bf16 ----
    constexpr int NV = LPW < TL::SOURCES ? LPW : TL::SOURCES;
    int voff[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) voff[i] = TL::source(i, lane, d_real * 2, chunks);
    auto load_tile = [&](const unsigned char *pool, uint32_t stride, int tile, int id, int slot) __attribute__((always_inline)) {
        const Where w = where(tile, id);
        int off[LPW];
#pragma unroll
        for (int i = 0; i < LPW; ++i) off[i] = voff[i % NV] + i / NV * NV * TL::LOAD_ROWS * d_real * 2;
        constexpr int P1 = LPW > 1 ? 1 : 0, P2 = LPW > 2 ? 2 : P1, P3 = LPW > 2 ? 3 : P2;
        buffer_load_lds16_n<LPW, TL::load_lds(P1), TL::load_lds(P2) - TL::load_lds(P1), TL::load_lds(P3) - TL::load_lds(P2)>(
            scalar_buffer_rsrc(address(pool, stride, w, row_b), w.rows * row_b), off, lds0 + slot * TL::BYTES + TL::load_lds(wv * LPW));
    };
    // ---- requests: 8-bit.  A lane has D / 8 values of the wave's eight rows: 8 of row lane / 8 (head_dim 64), 16 of it, or 16 of rows lane / 16 and 4 more (256) ----
    constexpr int NC = D == 256 ? 2 : 1, CW = D == 64 ? 2 : 4, PER = D == 256 ? 16 : 8;
    typedef uint32_t codes_t __attribute__((ext_vector_type(CW)));
    codes_t kraw[NC], vraw[NC];
    uint32_t kex[NC], vex[NC];
    const int e_row = lane / PER, e_col = lane % PER * 4 * CW, e_off = e_col < d_real ? e_row * d_real + e_col : (int)0x80000000;
    // (buffers that end with the rows that exist: others read as zero)
    const uint32_t kx_stride = (uint32_t)c.kx_page, vx_stride = (uint32_t)c.vx_page;
    const unsigned char *const kx_pool = (const unsigned char *)c.k_exp + (int64_t)kvh * c.page, *const vx_pool = (const unsigned char *)c.v_exp + (int64_t)kvh * c.page;
    auto fetch = [&](const unsigned char *pool, uint32_t stride, const unsigned char *exps, uint32_t xstride, int tile, int id, codes_t (&raw)[NC], uint32_t (&ex)[NC]) __attribute__((always_inline)) {
        const Where w = where(tile, id);
        const auto values = __builtin_amdgcn_make_buffer_rsrc((void *)address(pool, stride, w, row_b), 0, w.rows * row_b, 0x00020000);
        const auto powers = __builtin_amdgcn_make_buffer_rsrc((void *)address(exps, xstride, w, 1u), 0, w.rows, 0x00020000);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if constexpr (CW == 4) raw[i] = __builtin_amdgcn_raw_buffer_load_b128(values, e_off + 4 * i * d_real, 0, 0);
            else raw[i] = __builtin_amdgcn_raw_buffer_load_b64(values, e_off + 4 * i * d_real, 0, 0);
            ex[i] = __builtin_amdgcn_raw_buffer_load_b8(powers, e_row + 4 * i, 0, 0);
        }
    };
    auto unpack = [&](const codes_t (&raw)[NC], const uint32_t (&ex)[NC], int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int row = 8 * wv + e_row + 4 * i;
            const float s = exponent_scale(ex[i]);
            unsigned char *const to = dyn_lds + slot * TL::BYTES + row / TL::GROUP * TL::GROUP_B + row % TL::GROUP * TL::ROW_B;
#pragma unroll
            for (int w = 0; w < CW / 2; ++w) {
                const u32x2 a = e4m3_to_bf16(raw[i][2 * w], s), b = e4m3_to_bf16(raw[i][2 * w + 1], s);
                *reinterpret_cast<u32x4 *>(to + (((e_col / 8 + w) ^ TL::xor_of(row)) << 4)) = u32x4{a[0], a[1], b[0], b[1]};
            }
        }
    };
    auto fetch_k = [&](int tile, int id, codes_t (&raw)[NC], uint32_t (&ex)[NC]) __attribute__((always_inline)) {
        fetch(k_pool, k_stride, kx_pool, kx_stride, tile, id, raw, ex);
    };
    auto fetch_v = [&](int tile, int id, codes_t (&raw)[NC], uint32_t (&ex)[NC]) __attribute__((always_inline)) {
        fetch(v_pool, v_stride, vx_pool, vx_stride, tile, id, raw, ex);
    };
    auto load_k = [&](int tile, int id) __attribute__((always_inline)) { load_tile(k_pool, k_stride, tile, id, tile & 3); };
    auto load_v = [&](int tile, int id) __attribute__((always_inline)) { load_tile(v_pool, v_stride, tile, id, 4 + (tile & 3)); };

    // page numbers of the first tiles, q in the meantime
    const PageRing ring{base, pshift};
    load_ids(ring.batch(0));
    load_ids(ring.batch(0) + 1);
    bf16x8 qB[KS];
    {
        const bf16_t *const qrow = q + (int64_t)t * q_tok + (int64_t)hq * q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qB[ks] = row_ok && 2 * ks + h < chunks ? load_bf16x8(qrow + 16 * ks + 8 * h) : zero_bf16x8();
            qB[ks] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, qB[ks]) ^ flip);          // (a negative scale's sign)
        }
    }
    wait_vmcnt<0>();
    TL tl;
    tl.init(lane);
    auto meet_read = [&]() __attribute__((always_inline)) {               // (what this wave reads and writes of LDS is done)
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
        barrier_only();
    };
    f32x16 sE, sO;                                      // S of even and of odd tiles
    uint32_t pE[8], pO[8];                              // P of even and of odd tiles, packed (keys 0-15 | 16-31)
    if constexpr (!E4M3) {
        load_k(0, page_at(0)); load_k(1, page_at(1));
        load_v(0, page_at(0)); load_k(2, page_at(2)); load_v(1, page_at(1)); load_k(3, page_at(3)); load_v(2, page_at(2));
        wait_vmcnt<5 * LPW>();                          // K(0) and K(1) are there
    } else {
        codes_t r[6][NC];
        uint32_t x[6][NC];
#pragma unroll
        for (int i = 0; i < 4; ++i) fetch_k(i, page_at(i), r[i], x[i]);
        fetch_v(0, page_at(0), r[4], x[4]);
        fetch_v(1, page_at(1), r[5], x[5]);
        fetch_k(4, page_at(4), kraw, kex);
        fetch_v(2, page_at(2), vraw, vex);
#pragma unroll
        for (int i = 0; i < 6; ++i) unpack(r[i], x[i], i);              // (slots 0 .. 3 are K's, 4 and 5 V's first)
    }
    meet_read();

    lds_u8 *ka_[4], *va_[4];                            // operand addresses: of the K tile of S(t+2) and of V(t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ka_[i] = (lds_u8 *)dyn_lds + tl.rowq[i];
        va_[i] = (lds_u8 *)dyn_lds + tl.trq[i] + 4 * TL::BYTES;
    }
    auto advance = [&](lds_u8 *(&a)[4], int tile) __attribute__((always_inline)) {         // from tile - 1 to tile
        const int by = tile & 3 ? TL::BYTES : -3 * TL::BYTES;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] += by;
            asm volatile("" : "+v"(a[i]));
        }
    };
    auto read_k = [&](int ks) __attribute__((always_inline)) {
        return *reinterpret_cast<__attribute__((address_space(3))) const bf16x8 *>(ka_[TL::row_q(ks)] + TL::row_imm(ks));
    };
    auto read_v = [&](int i) __attribute__((always_inline)) {             // MFMA i of P V: keys of half i / DT, d-tile i % DT
        const int pair = i / DT, dt = i % DT;
        return tr_pair(va_[TL::tr_q(dt)] + TL::tr_imm(dt, 2 * pair), va_[TL::tr_q(dt)] + TL::tr_imm(dt, 2 * pair + 1));
    };
    // The keys of a tile this lane keeps, as they lie in memory; live(word): element vi then sits at bit 8*(vi/4) + vi%4
    const uint32_t row_mask = row_ok ? 0xffffffffu : 0u;
    auto live = [&](uint32_t w) __attribute__((always_inline)) { return (w >> (4 * h)) & row_mask; };
    auto word_of = [&](int tile) __attribute__((always_inline)) { return causal_bits(klim - (base + tile) * 32); };
    // (the row maximum is searched for where a sum says that some probability may have passed 2^8, or where a row has met no key yet: see dsa_tile_fwd.hip)
    auto masked = [&](float s, uint32_t word, int vi) __attribute__((always_inline)) {
        return keep_or_neginf(s, bit_mask(word, 8 * (vi >> 2) + (vi & 3)));
    };
    auto soft = [&](const f32x16 &s, uint32_t word, uint32_t (&p)[8], float &psum) __attribute__((always_inline)) {
        if (__builtin_amdgcn_ballot_w64(row_ok && (mrun == -INFINITY || !(psum <= 256.f)))) {
            asm volatile("" : "+v"(word));              // (nothing of the fast path is kept alive for this one)
            float mloc = -INFINITY;
#pragma unroll
            for (int vi = 0; vi < 16; ++vi) mloc = fmaxf(mloc, masked(s[vi], word, vi));
            mloc = half_max_f(mloc) * scale_log2;
            if (mloc > mrun) {
                const float alpha = fast_exp2(mrun - mloc);   // mrun = -inf: 0, and the sums are 0
                lsum *= alpha;
                if (AGPR) asm volatile("s_nop 11" : : : "memory");
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    if (AGPR) settle(oacc[dt]);
                    oacc[dt] *= alpha;
                    if (AGPR) settle(oacc[dt]);
                }
                mrun = mloc;
            }
            const float mneg = (mrun == -INFINITY) ? 0.f : -mrun;
            psum = 0.f;
#pragma unroll
            for (int vi = 0; vi < 16; vi += 2) {
                const float a = fast_exp2(fmaf(masked(s[vi], word, vi), scale_log2, mneg));
                psum += a;
                const float b = fast_exp2(fmaf(masked(s[vi + 1], word, vi + 1), scale_log2, mneg));
                psum += b;
                p[vi >> 1] = pack2bf(a, b);
            }
        }
        lsum += psum;
    };
    // S of tiles 0 and 1, P of tile 0
    auto gemm_s = [&](f32x16 &s) __attribute__((always_inline)) {
        s = zero16();
        bf16x8 ka[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) ka[ks] = read_k(ks);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = mfma32(ka[ks], qB[ks], s);
    };
    gemm_s(sE);
    advance(ka_, 1);
    if (ntiles > 1) gemm_s(sO);
    {
        float psum = INFINITY;                          // (no reference yet: the maximum is searched for)
        if (!row_ok) psum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) pE[i] = 0u;
        soft(sE, live(word_of(0)), pE, psum);
    }
    int id_k = page_at(5), id_v = page_at(3);           // of what the next step requests
    if constexpr (!E4M3) {
        wait_vmcnt<LPW>();                              // all but V(2): step 0 reads its first operands of V(1) itself
        meet_read();                                    // every wave is done with K(0) and K(1): their slots may be filled again
        load_k(4, page_at(4));
    } else {
        meet_read();
    }
    if (ring.due_early()) load_ids(ring.batch(2) + 1);  // (one load more on its way: the waits that count loads wait for more)
    constexpr int KA = 4;                               // (divides KS: an operand keeps its register from step to step)
    static_assert(KS % KA == 0 && NP % VA == 0);
    bf16x8 kr[KA], vr[VA];                              // operands of the next MFMA pairs
    advance(ka_, 2);
#pragma unroll
    for (int i = 0; i < KA; ++i) kr[i] = read_k(i);
#pragma unroll
    for (int i = 0; i < VA; ++i) vr[i] = read_v(i);
    uint32_t word_next = word_of(1);                    // (one-tile pieces never use it)

    // Step t: O += P(t) V(t) with `p`; softmax of tile t+1 from `s` into `pn` (SM); S(t+2) into `sn` (NEXT); requests (REQ)
    auto step = [&](auto masked_, auto sm_, auto next_, auto req_, int t_, const uint32_t (&p)[8], const f32x16 &s, uint32_t (&pn)[8],
                    f32x16 &sn) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked_)::value, SM = decltype(sm_)::value, NEXT = decltype(next_)::value, REQ = decltype(req_)::value;
        const u32x4 w0 = {p[0], p[1], p[2], p[3]}, w1 = {p[4], p[5], p[6], p[7]};
        const bf16x8 pB0 = __builtin_bit_cast(bf16x8, w0), pB1 = __builtin_bit_cast(bf16x8, w1);
        const uint32_t word = MASKED ? live(word_next) : 0xffffffffu;
        float psum = 0.f;
        const float mneg = (mrun == -INFINITY) ? 0.f : -mrun;
        f32x16 snew;
        constexpr int H = 2 * NS - 2;                   // half-steps an element can start in
        float y[16], e[16];
        auto behind = [&](int hs) __attribute__((always_inline)) {
#pragma unroll
            for (int vi = 16 * (hs - 2) / H; vi < 16 * (hs - 1) / H; ++vi)
                if (hs >= 2) {
                    psum += e[vi];
                    if (vi & 1) {
                        pn[vi >> 1] = pack2bf(e[vi - 1], e[vi]);
                        asm volatile("" : "+v"(pn[vi >> 1]));
                    }
                }
#pragma unroll
            for (int vi = 16 * (hs - 1) / H; vi < 16 * hs / H; ++vi)
                if (hs >= 1 && hs <= H) {
                    e[vi] = fast_exp2(y[vi]);
                    asm volatile("" : "+v"(e[vi]));
                }
#pragma unroll
            for (int vi = 16 * hs / H; vi < 16 * (hs + 1) / H; ++vi)
                if (hs < H) {
                    y[vi] = fmaf(MASKED ? masked(s[vi], word, vi) : s[vi], scale_log2, mneg);
                    asm volatile("" : "+v"(y[vi]));
                }
            asm volatile("" : "+v"(psum) : : "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        // this step's requests: K(t+5) and V(t+3) into LDS; or K(t+4) and V(t+2) from registers into LDS, and the loads of K(t+5) and V(t+3)
        auto request = [&](int what) __attribute__((always_inline)) {
            if constexpr (!E4M3) {
                if (what == 0) load_k(t_ + 5, id_k);
                else load_v(t_ + 3, id_v);
            } else {
                if (what == 0) {
                    unpack(kraw, kex, t_ & 3);
                    fetch_k(t_ + 5, id_k, kraw, kex);
                } else {
                    unpack(vraw, vex, 4 + ((t_ + 2) & 3));
                    fetch_v(t_ + 3, id_v, vraw, vex);
                }
            }
            if (what == 1) {
                // numbers for the next step, and the next batch of them once V has come to a batch's first page
                if (ring.due(t_ + 3)) load_ids(ring.batch(t_ + 3) + 1);
                id_k = page_at(t_ + 6);
                id_v = page_at(t_ + 4);
            }
        };
#pragma unroll
        for (int i = 0; i < (NEXT ? NS : NP); ++i) {
            if (i < NP) {
                if (AGPR) mfma32_agpr_late(oacc[i % DT], vr[i % VA], i < DT ? pB0 : pB1, !SM);
                else oacc[i % DT] = mfma32(vr[i % VA], i < DT ? pB0 : pB1, oacc[i % DT]);
            }
#pragma unroll
            for (int r_ = 0; r_ < 2; ++r_)
                if (REQ && r_ * (NP / 2) / 3 == i) request(r_);
            // refill: the operand a few pairs on, of this step's tiles or, past their end, of the next step's
            if (i == NP - VA && SM) advance(va_, t_ + 1);
            if (i < NP && (i + VA < NP || SM)) vr[i % VA] = read_v((i + VA) % NP);
            if (SM) behind(2 * i);
            else __builtin_amdgcn_sched_barrier(0);
            if (NEXT && i < KS) {
                snew = mfma32(kr[i % KA], qB[i], i == 0 ? zero16() : snew);
                if (i == KS - KA) advance(ka_, t_ + 3);
                kr[i % KA] = read_k((i + KA) % KS);
                if (i == 0 && MASKED) word_next = word_of(t_ + 2);
            }
            if (SM) behind(2 * i + 1);
        }
        if (SM) soft(s, word, pn, psum);
        if (NEXT) sn = snew;
    };
    const std::true_type yes;
    const std::false_type no;
    auto meet = [&]() __attribute__((always_inline)) {
        if constexpr (E4M3) {
            // (this step's writes: at least six reads have been issued behind them, and LDS answers in order)
            asm volatile("s_waitcnt lgkmcnt(6)" : : : "memory");
            barrier_only();
        } else {
            wait_vmcnt<LPS>();                          // all but what this step requested
            barrier_only();
        }
    };
    auto full_step = [&](auto masked_, int t_, const uint32_t (&p)[8], const f32x16 &s, uint32_t (&pn)[8], f32x16 &sn) __attribute__((always_inline)) {
        step(masked_, yes, yes, yes, t_, p, s, pn, sn);
        meet();
    };
    int tt = 0;
    {
        // tiles every row of the block attends whole: the softmax without mask arithmetic
        const int whole = (min(past + pc.first, keys - 1) + 1) / 32 - base;
        for (; tt + 3 < ntiles && tt + 2 < whole; tt += 2) {
            full_step(no, tt, pE, sO, pO, sE);
            full_step(no, tt + 1, pO, sE, pE, sO);
        }
        word_next = word_of(tt + 1);
    }
    for (; tt + 2 < ntiles; tt += 2) {
        // (S of up to two tiles past the end is formed for nothing)
        full_step(yes, tt, pE, sO, pO, sE);
        full_step(yes, tt + 1, pO, sE, pE, sO);
    }
    if (tt + 1 < ntiles) {
        full_step(yes, tt, pE, sO, pO, sE);
        step(yes, no, no, no, tt + 1, pO, sE, pE, sO);
    } else {
        step(yes, no, no, no, tt, pE, sO, pO, sE);
    }
    wait_vmcnt<0>();                                    // no load is left on its way into LDS when the workgroup ends

    // A zero probability times an infinite or NaN value is NaN, and a value that some rows attend others do not.  Sums that are not finite: the block again, tile by tile, in
    // which the products of such values are formed by themselves, for the rows that attend them.  (Looked for here, once, and not in each tile: with it in the loop sums spill.)
    int *const flag = reinterpret_cast<int *>(dyn_lds + 8 * TL::BYTES + NW * 512);
    {
        float zero = 0.f;
        if (AGPR) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) settle(oacc[dt]);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int x = 0; x < 16; ++x) zero = fmaf(oacc[dt][x], 0.f, zero);
        if (lane == 0) flag[wv] = 0;
        if (row_ok && !(zero == 0.f)) flag[wv] = 1;
        __syncthreads();
        if (!(flag[0] | flag[1] | flag[2] | flag[3])) {
            finish();
            return;
        }
    }
    mrun = -INFINITY;
    lsum = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        oacc[dt] = zero16();
        if (AGPR) settle(oacc[dt]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ka_[i] = (lds_u8 *)dyn_lds + tl.rowq[i];
        va_[i] = (lds_u8 *)dyn_lds + tl.trq[i] + 4 * TL::BYTES;
    }
    auto value_at = [&](int row, int ch) {
        return dyn_lds + 4 * TL::BYTES + row / TL::GROUP * TL::GROUP_B + row % TL::GROUP * TL::ROW_B + ((ch ^ TL::xor_of(row)) << 4);
    };
    for (int tile = 0; tile < ntiles; ++tile) {
        const int id = page_of(c, pc.n, pshift, (base + tile) * 32 + 8 * wv);
        if constexpr (!E4M3) {
            load_tile(k_pool, k_stride, tile, id, 0);
            load_tile(v_pool, v_stride, tile, id, 4);
            wait_vmcnt<0>();
        } else {
            fetch_k(tile, id, kraw, kex);
            fetch_v(tile, id, vraw, vex);
            unpack(kraw, kex, 0);
            unpack(vraw, vex, 4);
        }
        meet_read();
        gemm_s(sE);
        float psum = row_ok ? INFINITY : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) pE[i] = 0u;
        soft(sE, live(word_of(tile)), pE, psum);
        for (int key = 0; key < 32; ++key) {
            const int vi = (key >> 3) * 4 + (key & 3), from = ((key >> 2) & 1) * 32 + j;     // where its probability lies
            uint32_t pair = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) pair = i == vi >> 1 ? pE[i] : pair;
            const float prob = __uint_as_float((uint32_t)__shfl((int)(vi & 1 ? pair & 0xffff0000u : pair << 16), from, 64));
            const bool attends = row_ok && (base + tile) * 32 + key <= klim;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const bf16x4 val = *reinterpret_cast<const bf16x4 *>(value_at(key, 4 * dt + g4) + 8 * h);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if (attends && !(fabsf((float)val[x]) < INFINITY)) oacc[dt][4 * g4 + x] = fmaf(prob, (float)val[x], oacc[dt][4 * g4 + x]);
                }
        }
        meet_read();
        for (int i = tid; i < 32 * TL::CPR; i += NW * 64) {
            u32x4 *const to = reinterpret_cast<u32x4 *>(value_at(i / TL::CPR, i % TL::CPR));
            u32x4 w = *to;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if ((w[x] & 0x7f80u) == 0x7f80u) w[x] &= 0xffff0000u;
                if ((w[x] & 0x7f800000u) == 0x7f800000u) w[x] &= 0xffffu;
            }
            *to = w;
        }
        meet_read();
        const u32x4 w0 = {pE[0], pE[1], pE[2], pE[3]}, w1 = {pE[4], pE[5], pE[6], pE[7]};
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (AGPR) mfma32_agpr_late(oacc[i % DT], read_v(i), __builtin_bit_cast(bf16x8, i < DT ? w0 : w1), true);
            else oacc[i % DT] = mfma32(read_v(i), __builtin_bit_cast(bf16x8, i < DT ? w0 : w1), oacc[i % DT]);
        }
        meet_read();
    }
    finish();
}
