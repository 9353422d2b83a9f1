// How the work on shared beginnings is cut, worked out alike by every CTA of a launch from the groups of rows on the device.
//
// A group is a set of one-token rows that hold the same first `tokens` tokens in the same pages. Its rows are cut into tiles
// of up to `rows_per_tile` rows (whose query heads of one kv head are the rows of a matrix product), and the shared keys of a
// (tile, kv head) into units of `chunk` blocks of 64 keys. chunk is the least for which all units are at most as many as the
// launch's slots (sum over tiles of ceil(blocks / chunk) <= sum(blocks) / chunk + tiles: a few tries tell), or all of them where there
// are more tiles than that. Units are numbered tile by tile, kv head by kv head; a partial result goes to the slot of its unit's number.
#pragma once
#include "common.cuh"

#define PU_MIN_CHUNK 2                // blocks of 64 keys a unit has at least

struct PrefixUnits {
    int units, chunk;                 // of all tiles and kv heads; blocks of 64 keys a unit
};
struct PrefixUnit {
    int group, tile, first;           // the group, the tile's number in it, the first unit of (tile, kv head 0)
    int splits, hk, split;            // units of each (tile, kv head); this one's kv head and place
    int start, count, blocks;         // the tile's rows in `members`, and the blocks of 64 keys they share (the last may be cut short)
};

__device__ __forceinline__ int pu_sum(int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int pu_max(int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// What a lane holds of up to 32 groups, g0 + lane: the first ones are read once (few steps have more).
struct PrefixGroups {
    const int32_t* groups;            // [n_groups][3]: start, count (0: none), tokens
    int n_groups, rows_per_tile;
    int start, tiles, count, blocks;  // of group `lane`
    __device__ __forceinline__ void read(int g, int& start_, int& tiles_, int& count_, int& blocks_) const {
        const bool there = g < n_groups;
        start_ = there ? groups[3 * g] : 0;
        count_ = there ? groups[3 * g + 1] : 0;
        blocks_ = there ? (groups[3 * g + 2] + 63) >> 6 : 0;
        tiles_ = (int)((unsigned)(count_ + rows_per_tile - 1) / (unsigned)rows_per_tile);
    }
    __device__ __forceinline__ PrefixGroups(const int32_t* groups_, int n, int rows) : groups(groups_), n_groups(n), rows_per_tile(rows) {
        read(threadIdx.x & 31, start, tiles, count, blocks);
    }
    __device__ __forceinline__ void at(int g0, int& start_, int& tiles_, int& count_, int& blocks_) const {
        if (g0 == 0) { start_ = start; tiles_ = tiles; count_ = count; blocks_ = blocks; }
        else read(g0 + (threadIdx.x & 31), start_, tiles_, count_, blocks_);
    }
};

// By a whole warp.
__device__ __forceinline__ PrefixUnits prefix_units(const PrefixGroups& all, int kv_heads, int slots) {
    int tiles = 0, blocks = 0, longest = 0;
    for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
        int s, t, c, k;
        all.at(g0, s, t, c, k);
        tiles += t; blocks += t * k; longest = max(longest, t > 0 ? k : 0);
    }
    tiles = pu_sum(tiles); blocks = pu_sum(blocks); longest = pu_max(longest);
    const int each = slots / kv_heads, budget = each - tiles;        // units a kv head; those beyond one a tile
    const int most = max(PU_MIN_CHUNK, budget > 0 ? min(longest, (blocks + budget - 1) / budget) : longest);   // surely enough
    PrefixUnits u;
    u.chunk = budget > 0 ? min(most, max(PU_MIN_CHUNK, (blocks + each - 1) / each)) : most;                     // at least this
    while (true) {
        int units = 0;
        for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
            int s, t, c, k;
            all.at(g0, s, t, c, k);
            units += t * (int)((unsigned)(k + u.chunk - 1) / (unsigned)u.chunk);
        }
        u.units = pu_sum(units) * kv_heads;
        if (u.chunk >= most || u.units <= slots) return u;
        ++u.chunk;
    }
}

// Unit `want` (< units), by a whole warp.
__device__ __forceinline__ PrefixUnit prefix_unit(const PrefixGroups& all, int kv_heads, int chunk, int want) {
    const int lane = threadIdx.x & 31;
    PrefixUnit u = {};
    int before = 0;
    for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
        int start, tiles, count, blocks;
        all.at(g0, start, tiles, count, blocks);
        const int splits = (int)((unsigned)(blocks + chunk - 1) / (unsigned)chunk), mine = tiles * splits * kv_heads;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > want);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int at = __shfl_sync(0xffffffffu, before + upto - mine, src);
            u.group = g0 + src;
            u.splits = __shfl_sync(0xffffffffu, splits, src);
            u.blocks = __shfl_sync(0xffffffffu, blocks, src);
            const int in_group = __shfl_sync(0xffffffffu, count, src), first_row = __shfl_sync(0xffffffffu, start, src);
            const unsigned rest = want - at, pair = rest / (unsigned)u.splits;    // the unit's (tile, kv head)
            u.split = (int)(rest - pair * u.splits);
            u.tile = (int)(pair / (unsigned)kv_heads);
            u.hk = (int)pair - u.tile * kv_heads;
            u.first = at + u.tile * kv_heads * u.splits;
            u.start = first_row + u.tile * all.rows_per_tile;
            u.count = min(all.rows_per_tile, in_group - u.tile * all.rows_per_tile);
            return u;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return u;
}
