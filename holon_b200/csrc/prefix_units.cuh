// How the work on shared beginnings is cut, worked out alike by every CTA of a launch from the groups of rows on the device.
//
// A group is a set of one-token rows that hold the same first `tokens` tokens in the same pages. Its rows are cut into tiles
// of up to `rows_per_tile` rows (whose query heads of one kv head are the rows of a matrix product), and the shared keys of a
// (tile, kv head) into units of `chunk` blocks of 64 keys. chunk is the least for which all units are at most as many as the
// launch's slots, as far as a closed form tells: sum over tiles of ceil(blocks / chunk) <= sum(blocks) / chunk + tiles. Units
// are numbered tile by tile, kv head by kv head; a partial result goes to the slot of its unit's number.
#pragma once
#include "common.cuh"

#define PU_MIN_CHUNK 2                // blocks of 64 keys a unit has at least

struct PrefixUnits {
    int units, chunk;                 // of all tiles and kv heads; blocks of 64 keys a unit
};
struct PrefixUnit {
    int group, tile, first;           // the group, the tile's number in it, the first unit of (tile, kv head 0)
    int splits, hk, split;            // units of each (tile, kv head); this one's kv head and place
    int start, count, tokens;         // the tile's rows in `members`, and the tokens they share
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

// By a whole warp. groups [n_groups][3]: start, count (0: none), tokens.
__device__ __forceinline__ PrefixUnits prefix_units(const int32_t* __restrict__ groups, int n_groups, int rows_per_tile, int kv_heads, int slots) {
    const int lane = threadIdx.x & 31;
    int tiles = 0, blocks = 0, longest = 0;
    for (int g0 = 0; g0 < n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int count = g < n_groups ? groups[3 * g + 1] : 0, tokens = g < n_groups ? groups[3 * g + 2] : 0;
        const int t = (count + rows_per_tile - 1) / rows_per_tile, k = (tokens + 63) / 64;
        tiles += t; blocks += t * k; longest = max(longest, t > 0 ? k : 0);
    }
    tiles = pu_sum(tiles); blocks = pu_sum(blocks); longest = pu_max(longest);
    const int budget = slots / kv_heads - tiles;                     // units a kv head beyond one a tile
    PrefixUnits u;
    u.chunk = max(PU_MIN_CHUNK, budget > 0 ? min(longest, (blocks + budget - 1) / budget) : longest);
    int units = 0;
    for (int g0 = 0; g0 < n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int count = g < n_groups ? groups[3 * g + 1] : 0, tokens = g < n_groups ? groups[3 * g + 2] : 0;
        units += (count + rows_per_tile - 1) / rows_per_tile * (((tokens + 63) / 64 + u.chunk - 1) / u.chunk);
    }
    u.units = pu_sum(units) * kv_heads;
    return u;
}

// Unit `want` (< units), by a whole warp.
__device__ __forceinline__ PrefixUnit prefix_unit(const int32_t* __restrict__ groups, int n_groups, int rows_per_tile, int kv_heads, int chunk, int want) {
    const int lane = threadIdx.x & 31;
    PrefixUnit u = {};
    int before = 0;
    for (int g0 = 0; g0 < n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int count = g < n_groups ? groups[3 * g + 1] : 0, tokens = g < n_groups ? groups[3 * g + 2] : 0;
        const int splits = ((tokens + 63) / 64 + chunk - 1) / chunk, mine = (count + rows_per_tile - 1) / rows_per_tile * splits * kv_heads;
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
            u.tokens = __shfl_sync(0xffffffffu, tokens, src);
            const int all = __shfl_sync(0xffffffffu, count, src), per_tile = u.splits * kv_heads, rest = want - at;
            u.tile = rest / per_tile;
            u.first = at + u.tile * per_tile;
            u.hk = (rest - u.tile * per_tile) / u.splits;
            u.split = rest - u.tile * per_tile - u.hk * u.splits;
            u.start = groups[3 * u.group] + u.tile * rows_per_tile;
            u.count = min(rows_per_tile, all - u.tile * rows_per_tile);
            return u;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return u;
}
