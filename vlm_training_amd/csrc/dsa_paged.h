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

// ---- a row's statistics, once its sums are formed ----
// The largest logit of a row, for its joining with other pieces' sums: a maximum passes NaN over, so that a piece in which every logit is NaN would pass for one without a key,
// and one with some of them might weigh 0 beside a far larger logit.  A sum that is NaN counts as infinitely large: the row is NaN as a whole.
__device__ __forceinline__ float row_maximum(float m, float l) { return l == l ? m : INFINITY; }

// ---- how the work is cut ----
// A request's new rows go in blocks of `qb` queries.  Lengths are on the device, so every workgroup forms the plan itself: sums over the requests, one in each lane.
struct PagePlan {
    int N, T, qb, few, side;       // requests of up to `few` new rows are side 0's, others side 1's; side -1: all of them
    int target;                    // workgroups aimed at, or launched, for each kv head
    float per_target;              // 1 / target
    int least;                     // tiles of 32 keys that a piece of a block has at the least
    int whole;                     // no block is cut
    int pair;                      // workgroups of a kv head that run at once, one to a compute unit (0: no second one to a unit)
    int ushift;                    // shares are counted in units of 2^ushift tiles
    const int32_t *cu, *lengths;
    int capacity;                  // positions that the table holds
};
struct PagePiece {
    int n, row0, m, length;        // request, its first row, its new rows, its length
    int first;                     // first query of the block
    int tile0, tile1;              // the piece's key tiles
    int piece, pieces;             // which of how many pieces of this block (shares: whether it is the first, and whether there are others)
    int slot;                      // of the block's first piece's sums (shares: of this one's)
};
// A kernel's part of a call: its plan, its blocks for each kv head (0: none to join), the pieces of a block at the most, and the pieces' sums
struct PagedPart {
    PagePlan plan;
    int blocks, pieces;
    float *part_o, *part_ml;
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
    return p.whole ? 1 << 30 : max(p.least, (int)fminf(ceilf(plan_sum(mine) * 1.0001f / (float)p.target), 1e9f));
}
// Blocks of many rows: each in pieces of about equal length, as many as make launches of about `target` workgroups for each kv head out of all requests together, but no more
// than the root of its tiles (a piece more costs the block's sums once more to write and read).  Piece `slot` (BLOCKS: block `slot`) of the launch; false past the last one, with `spare`
// the number of slots in front that are taken.
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
    int slots = 0, taken = 0;                            // of sums, and of what is counted
    for (int base = 0; base < p.N; base += 64) {
        if (base > 0) r = page_request(p, base + lane);
        const int each = max(per, (int)sqrtf((float)r.tiles)), np = max(1, (r.tiles + each - 1) / each), mine = r.blocks * np, count = BLOCKS ? r.blocks : mine;
        const int upto = wave_prefix_i(count), sums = np > 1 ? mine : 0, sums_upto = wave_prefix_i(sums);      // (blocks that are not cut have no sums to keep)
        if (!BLOCKS && p.N <= 64) {
            // a launch of one round, the units' second workgroups: from the end, so that a unit with a long walk has a short one beside it
            const int total = __builtin_amdgcn_readlane(upto, 63);
            if (slot >= p.pair && slot < total && total <= 2 * p.pair) slot = total - 1 - (slot - p.pair);
        }
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
            out.slot = slots + __builtin_amdgcn_readlane(sums_upto, w) - __builtin_amdgcn_readlane(sums, w) + order * np_w;
            const int last = out.length - out.m + min(out.first + p.qb, out.m) - 1;      // position of the block's last row
            const int tiles = last < 0 ? 0 : (min(last, p.capacity - 1) >> 5) + 1, len = (tiles + np_w - 1) / np_w;
            out.pieces = len > 0 ? (tiles + len - 1) / len : 1;
            out.piece = i;
            out.tile0 = min(i * len, tiles);
            out.tile1 = min(out.tile0 + len, tiles);
            return true;
        }
        taken += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(sums_upto, 63);
    }
    spare = taken;
    return false;
}
// Blocks of a few rows: all blocks' tiles one behind the other, each block's behind a few that stand for what going to it costs (BLOCK_COST), cut into equal shares, one for each of `target`
// workgroups of a kv head: however the lengths are mixed, all of them end together.  A cut that falls within a 16th of a share from a block's end is moved there.  A workgroup goes from block to block through its share; a block that is
// cut has a piece for each share that it lies in.  Sums of piece 0 lie in slot 2 k - 1, of piece i > 0 in 2 (k + i - 1), k the first cut inside the block, counted from the launch's
// start: no two pieces share one, and there are 2 `target` of them.
// (a block's rows, the look-up of its first pages and the joining of its waves take 4 to 5 us one after the other, a tile of a workgroup 1 to 1.5)
#define BLOCK_COST 4
struct PageShares {
    int share, near, cost;         // units of a share, how far a cut is moved at the most, and units in front of a block's tiles
    __device__ __forceinline__ int first_cut(int u0) const { return (u0 + cost + near + share - 1) / share; }
    __device__ __forceinline__ int cuts(int u0, int u1) const { return max(0, max(u1 - near, 0) / share - first_cut(u0) + 1); }
    __device__ __forceinline__ int moved(int x, int u0, int u1) const { return x - u0 < cost + near ? u0 : u1 - x < near ? u1 : x; }
};
__device__ __forceinline__ int units_of(const PagePlan &p, int tiles) { return max(1, (BLOCK_COST + tiles + (1 << p.ushift) - 1) >> p.ushift); }
__device__ __forceinline__ PageShares page_shares(const PagePlan &p, const PageRequest &r) {
    const int lane = threadIdx.x & 63;
    int sum = r.blocks * units_of(p, r.tiles);           // (the host chose the unit for the sum to have less than 30 bits)
    for (int n = 64 + lane; n < p.N; n += 64) {
        const PageRequest x = page_request(p, n);
        sum += x.blocks * units_of(p, x.tiles);
    }
    sum = wave_sum_i(sum);
    PageShares s;
    // (a float's product, rounded up and one more, is enough: divisions of whole numbers take a wave 300 clocks each, in front of its first load)
    s.share = __builtin_amdgcn_readfirstlane(max(max(p.least >> p.ushift, 1), (int)((float)sum * p.per_target * 1.000001f) + 1));
    s.cost = BLOCK_COST >> p.ushift;
    s.near = p.whole ? 1 << 29 : max(1, s.share >> 4);
    return s;
}
// the block of request `n` (lane w of r) that is the order-th of its blocks (the last one, which has the most keys, first): whose it is, and its first query
__device__ __forceinline__ void share_block(const PagePlan &p, const PageRequest &r, int w, int n, int order, PagePiece &out) {
    out.n = n;
    out.row0 = __builtin_amdgcn_readlane(r.row0, w);
    out.m = __builtin_amdgcn_readlane(r.m, w);
    out.length = __builtin_amdgcn_readlane(r.length, w);
    out.first = (__builtin_amdgcn_readlane(r.blocks, w) - 1 - order) * p.qb;
}
struct ShareWalk {
    PageShares s;
    PageRequest r;
    int base, w, order, u0, mine, x0, x1;                // batch of 64 requests, the block's lane in it and its number, its first unit; the share and its ends
    bool more;
    __device__ __forceinline__ void start(const PagePlan &p, int share) {
        r = page_request(p, threadIdx.x & 63);           // (up to 64 requests: looked at once)
        s = page_shares(p, r);
        mine = share;
        x0 = share * s.share;
        x1 = x0 + s.share;
        more = false;
        int before = 0;
        for (base = 0; base < p.N; base += 64) {
            if (base > 0) r = page_request(p, base + (threadIdx.x & 63));
            const int units = units_of(p, r.tiles), count = r.blocks * units, upto = wave_prefix_i(count);
            const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > x0);
            if (past) {
                w = (int)__builtin_ctzll(past);
                const int at = before + __builtin_amdgcn_readlane(upto, w) - __builtin_amdgcn_readlane(count, w), per = __builtin_amdgcn_readlane(units, w);
                order = __builtin_amdgcn_readlane(r.blocks, w) > 1 ? (x0 - at) / per : 0;
                u0 = at + order * per;
                more = true;
                return;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
    }
    // the share's next piece
    __device__ __forceinline__ bool next(const PagePlan &p, PagePiece &out) {
        while (more && x1 > u0) {
            const int u1 = u0 + units_of(p, __builtin_amdgcn_readlane(r.tiles, w));
            const int lo = x0 <= u0 ? u0 : s.moved(x0, u0, u1), hi = x1 >= u1 ? u1 : s.moved(x1, u0, u1);
            if (lo < hi) {
                share_block(p, r, w, base + w, order, out);
                const int last = out.length - out.m + min(out.first + p.qb, out.m) - 1;      // position of the block's last row
                const int tiles = last < 0 ? 0 : (min(last, p.capacity - 1) >> 5) + 1;
                // (a first piece ends with the first cut inside the block, the next share's start; another begins with its share)
                out.piece = lo != u0;
                out.pieces = 1 + (lo != u0 || hi != u1);
                out.slot = 2 * mine + (lo == u0);
                out.tile0 = lo == u0 ? 0 : min((lo - u0 - s.cost) << p.ushift, tiles);
                out.tile1 = hi == u1 ? tiles : min((hi - u0 - s.cost) << p.ushift, tiles);
            }
            // on to the next block
            u0 = u1;
            if (++order >= __builtin_amdgcn_readlane(r.blocks, w)) {
                order = 0;
                uint64_t rest = __builtin_amdgcn_ballot_w64(r.blocks > 0) & (w < 63 ? ~0ull << (w + 1) : 0ull);
                while (!rest && base + 64 < p.N) {
                    base += 64;
                    r = page_request(p, base + (threadIdx.x & 63));
                    rest = __builtin_amdgcn_ballot_w64(r.blocks > 0);
                }
                more = rest != 0;
                w = more ? (int)__builtin_ctzll(rest) : 0;
            }
            if (lo < hi) return true;
        }
        return false;
    }
};
// Block `slot` of such a launch
__device__ __forceinline__ bool locate_share_block(const PagePlan &p, int slot, PagePiece &out) {
    PageRequest r = page_request(p, threadIdx.x & 63);
    const PageShares s = page_shares(p, r);
    int taken = 0, before = 0;
    for (int base = 0; base < p.N; base += 64) {
        if (base > 0) r = page_request(p, base + (threadIdx.x & 63));
        const int units = units_of(p, r.tiles), upto = wave_prefix_i(r.blocks), uupto = wave_prefix_i(r.blocks * units);
        const uint64_t past = __builtin_amdgcn_ballot_w64(taken + upto > slot);
        if (past) {
            const int w = (int)__builtin_ctzll(past), blocks = __builtin_amdgcn_readlane(r.blocks, w), per = __builtin_amdgcn_readlane(units, w);
            const int order = slot - taken - (__builtin_amdgcn_readlane(upto, w) - blocks);
            const int u0 = before + __builtin_amdgcn_readlane(uupto, w) - (blocks - order) * per;
            share_block(p, r, w, base + w, order, out);
            out.pieces = s.cuts(u0, u0 + per) + 1;
            out.slot = 2 * s.first_cut(u0) - 1;
            return true;
        }
        taken += __builtin_amdgcn_readlane(upto, 63);
        before += __builtin_amdgcn_readlane(uupto, 63);
    }
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
