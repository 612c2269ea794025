// The paged cache as kernels see it: where a row lies, e4m3 values as bf16, and how the work of an attention over it is cut.
#pragma once
#include "dsa_tile.h"
#include "../../include/dsa_attn.h"

// the request whose rows row t lies among: the last n with cu[n] <= t (empty ones are stepped over), by a whole wave.  64 offsets are looked at in one round
// trip and narrow the search to a 64th, so that it takes two of them up to 4096 requests.  -1 in front of the first, N behind the last.
__device__ __forceinline__ int find_request(const int32_t *__restrict__ cu, int N, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = N + 1;                               // entries lo .. lo + n - 1; those in front are <= t
    while (true) {
        const int step = (n + 63) >> 6, at = lane * step;
        const uint64_t hits = __builtin_amdgcn_ballot_w64(at < n && cu[lo + min(at, n - 1)] <= t);
        const int k = (int)__popcll(hits);
        if (k == 0) return lo - 1;
        lo += (k - 1) * step;
        n = min(step, n - (k - 1) * step);
        if (step == 1) return lo;
    }
}

// page of position p (p >= 0 and wave-uniform or a lane's own), or -1 where there is none
__device__ __forceinline__ int page_of(const dsa_cache_args &c, int n, int pshift, int p) {
    const int at = p >> pshift;
    if (at >= c.table_pages) return -1;
    const int id = c.table[(int64_t)n * c.table_row + at];
    return (uint32_t)id < (uint32_t)c.pages ? id : -1;
}

// ---- e4m3 ----
// The smallest e >= -100 with which `largest`, a bf16's bits without its sign, is at most 448 * 2^e = 1.75 * 2^(e + 8)
__device__ __forceinline__ int scale_exponent(uint32_t largest) {
    const int e = (int)(largest >> 7) - 127 - 8 + ((largest & 0x7f) > 0x60);
    return max(e, -100);
}
// four e4m3 values of a word -> bf16, times 2^(exp - 127); exact for the powers that are written.  (The instruction takes the exponent of its scale alone; at 255 it is
// NaN's, and the value itself is NaN in rows that were written so.)
__device__ __forceinline__ u32x2 e4m3_to_bf16(uint32_t w, float scale) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ float exponent_scale(uint32_t b) { return __uint_as_float(b == 255 ? 0x7fc00000u : b << 23); }

// ---- how the work is cut ----
// A request's new rows go in blocks of `qb` queries, and the keys of each of its blocks in `pieces` of about equal length, as many as make launches of about `target`
// workgroups for each kv head out of all requests together: a few long requests and a batch of short ones fill the card alike.  Lengths are on the device, so every
// workgroup forms the plan itself: sums over the requests, one in each lane.
struct PagePlan {
    int N, T, qb, few, side;       // requests of up to `few` new rows are side 0's, others side 1's; side -1: all of them
    int target, least;             // workgroups aimed at (per kv head); tiles of 32 keys that a piece has at the least
    const int32_t *cu, *lengths;
    int capacity;                  // positions that the table holds
};
struct PagePiece {
    int n, row0, m, length;        // request, its first row, its new rows, its length
    int first;                     // first query of the block
    int tile0, tile1;              // the piece's key tiles
    int piece, pieces;             // pieces of this block that have tiles (1 at the least)
    int slot;                      // of the block's first piece
};
struct PageRequest { int row0, m, length, blocks, tiles; };
__device__ __forceinline__ PageRequest page_request(const PagePlan &p, int n) {
    PageRequest r;
    const int at = min(n, p.N - 1), lo = min(max(p.cu[at], 0), p.T), hi = min(max(p.cu[at + 1], lo), p.T);
    r.row0 = lo;
    r.m = hi - lo;
    r.length = max(p.lengths[at], 0);
    const bool mine = n < p.N && r.m > 0 && (p.side < 0 || (r.m > p.few) == (p.side == 1));
    r.blocks = mine ? (r.m + p.qb - 1) / p.qb : 0;
    r.tiles = (min(r.length, p.capacity) + 31) >> 5;
    return r;
}
// Sums over the wave by DPP steps (no LDS round trips: a workgroup forms them in front of its first load)
__device__ __forceinline__ float plan_sum(float x) {
#define PLAN_STEP(ctrl, rows) x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), ctrl, rows, 0xf, false))
    PLAN_STEP(0x111, 0xf); PLAN_STEP(0x112, 0xf); PLAN_STEP(0x114, 0xf); PLAN_STEP(0x118, 0xf); PLAN_STEP(0x142, 0xa); PLAN_STEP(0x143, 0xc);
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
#undef PLAN_STEP
}
// tiles to a piece, from the sum of all blocks' tiles (a little over the sum's own rounding: the slots of a launch are counted for this many pieces)
__device__ __forceinline__ int piece_tiles(const PagePlan &p, float mine) {
    return max(p.least, (int)fminf(ceilf(plan_sum(mine) * 1.0001f / (float)p.target), 1e9f));
}
// Piece `slot` (BLOCKS: block `slot`) of the launch; false past the last one, with `spare` the number of slots in front that are taken
template <bool BLOCKS>
__device__ __forceinline__ bool locate_piece(const PagePlan &p, int slot, PagePiece &out, int &spare) {
    const int lane = threadIdx.x & 63;
    PageRequest r = page_request(p, lane);               // (up to 64 requests: looked at once)
    float sum = (float)r.blocks * (float)r.tiles;
    for (int n = 64 + lane; n < p.N; n += 64) {
        const PageRequest x = page_request(p, n);
        sum += (float)x.blocks * (float)x.tiles;
    }
    const int per = piece_tiles(p, sum);
    int slots = 0, taken = 0;                            // of pieces, and of what is counted
    for (int base = 0; base < p.N; base += 64) {
        if (base > 0) r = page_request(p, base + lane);
        const int np = max(1, (r.tiles + per - 1) / per), mine = r.blocks * np, count = BLOCKS ? r.blocks : mine;
        const int upto = wave_prefix_i(count), slots_upto = BLOCKS ? wave_prefix_i(mine) : upto;
        const uint64_t past = __builtin_amdgcn_ballot_w64(taken + upto > slot);
        if (past) {
            const int w = (int)__builtin_ctzll(past);
            const int np_w = __builtin_amdgcn_readlane(np, w), blocks = __builtin_amdgcn_readlane(r.blocks, w);
            const int at = slot - taken - (__builtin_amdgcn_readlane(upto, w) - __builtin_amdgcn_readlane(count, w));
            // (the last block, which has the most keys, first)
            const int order = BLOCKS ? at : at / np_w, i = BLOCKS ? 0 : at % np_w;
            out.n = base + w;
            out.row0 = __builtin_amdgcn_readlane(r.row0, w);
            out.m = __builtin_amdgcn_readlane(r.m, w);
            out.length = __builtin_amdgcn_readlane(r.length, w);
            out.first = (blocks - 1 - order) * p.qb;
            out.slot = slots + __builtin_amdgcn_readlane(slots_upto, w) - __builtin_amdgcn_readlane(mine, w) + order * np_w;
            const int last = out.length - out.m + min(out.first + p.qb, out.m) - 1;      // position of the block's last row
            const int tiles = last < 0 ? 0 : (min(last, p.capacity - 1) >> 5) + 1, len = (tiles + np_w - 1) / np_w;
            out.pieces = len > 0 ? (tiles + len - 1) / len : 1;
            out.piece = i;
            out.tile0 = min(i * len, tiles);
            out.tile1 = min(out.tile0 + len, tiles);
            return true;
        }
        taken += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slots_upto, 63);
    }
    spare = taken;
    return false;
}
// Rows behind the last request: zeros, by the workgroups that found no piece (the first of them is 0 of `step`; each its kv head's rows)
__device__ __forceinline__ void zero_tail(const PagePlan &p, int Hq, int Hkv, int kvh, int at, int step, int d_real, int threads, bf16_t *out, float *lse) {
    const int from = min(max(p.cu[p.N], 0), p.T), G = Hq / Hkv, tid = threadIdx.x;
    for (int t = from + at; t < p.T; t += step) {
        bf16_t *const row = out + ((int64_t)t * Hq + kvh * G) * d_real;
        for (int i = tid; i < G * d_real / 8; i += threads) *reinterpret_cast<u32x4 *>(row + 8 * i) = u32x4{0u, 0u, 0u, 0u};
        if (lse && tid < G) lse[(int64_t)(kvh * G + tid) * p.T + t] = -INFINITY;
    }
}
