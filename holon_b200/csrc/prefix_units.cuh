// How the work on shared beginnings is cut, worked out alike by every CTA of a launch from the groups of rows on the device.
//
// A group is a set of one-token rows that hold the same first `tokens` tokens in the same pages. Its rows are cut into tiles
// of up to `rows_per_tile` rows (whose query heads of one kv head are the rows of a matrix product), and the shared keys of a
// (tile, kv head) into units of `chunk` blocks of 64 keys. chunk is the least for which all units are at most as many as the
// launch's slots (sum over tiles of ceil(blocks / chunk) <= sum(blocks) / chunk + tiles: a few tries tell), or all of them where there
// are more tiles than that. Units are numbered tile by tile, kv head by kv head; a partial result goes to the slot of its unit's number.
// No (tile, kv head) is cut into more than PU_MOST_PARTS units: attention_rows.cu weighs them in shared memory that holds so many.
#pragma once
#include "common.cuh"

#define PU_MIN_CHUNK 2                // blocks of 64 keys a unit has at least
#define PU_MOST_PARTS 240             // units of a (tile, kv head) at most; reached with one kv head off tcgen05 alone (296 slots)

struct PrefixUnits {
    int units, chunk;                 // of all tiles and kv heads; blocks of 64 keys a unit
};
struct PrefixUnit {
    int group, tile, first;           // the group, the tile's number in it, the first unit of (tile, kv head 0)
    int splits, hk, split;            // units of each (tile, kv head); this one's kv head and place
    int start, count, tokens, slot;   // the tile's rows in `members`, the tokens they share, the block table's row where those lie
};

// a / b for 0 <= a < 2^24, b > 0: an approximate quotient, off by one at most where it is below 2^22, and put right. (Seven
// divisions stand before a CTA's first load; what they cost is the code that has to come.)
__device__ __forceinline__ int pu_div(int a, int b) {
    const int q = (int)__fdividef((float)a, (float)b), rest = a - q * b;
    return q + (rest >= b ? 1 : rest < 0 ? -1 : 0);
}
__device__ __forceinline__ int pu_ceil(int a, int b) { return pu_div(a + b - 1, b); }

// What a lane holds of up to 32 groups, g0 + lane: the first ones are read once (few steps have more).
struct PrefixGroups {
    const int4* groups;               // [n_groups]: start, count (0: none), tokens, the block table's row of one of them
    int n_groups, rows_per_tile;
    int start, tiles, count, blocks, tokens, slot;  // of group `lane`
    __device__ __forceinline__ void read(int g) {
        const int4 x = g < n_groups ? groups[g] : make_int4(0, 0, 0, 0);
        start = x.x; count = x.y; tokens = x.z; slot = x.w;
        blocks = (tokens + 63) >> 6;
        tiles = pu_ceil(count, rows_per_tile);
    }
    __device__ __forceinline__ PrefixGroups(const int32_t* groups_, int n, int rows) : groups((const int4*)groups_), n_groups(n), rows_per_tile(rows) {
        read(threadIdx.x & 31);
    }
    __device__ __forceinline__ PrefixGroups from(int g0) const {     // groups g0 ..
        PrefixGroups x = *this;
        if (g0 > 0) x.read(g0 + (threadIdx.x & 31));
        return x;
    }
};

// The numbers of blocks a unit that are tried, from `least` to `most`, for `tiles` tiles of `blocks` blocks together, the longest of `longest`
// blocks, and `each` slots a kv head.
struct PrefixChunks {
    int least, most;
    __host__ __device__ __forceinline__ PrefixChunks(int tiles, int blocks, int longest, int each) {
        const int budget = each - tiles;                             // units a kv head; those beyond one a tile
        const int in_parts = (longest + PU_MOST_PARTS - 1) / PU_MOST_PARTS, floor = in_parts > PU_MIN_CHUNK ? in_parts : PU_MIN_CHUNK;
        most = longest;
        if (budget > 0 && (blocks + budget - 1) / budget < longest) most = (blocks + budget - 1) / budget;      // surely enough
        if (most < floor) most = floor;
        least = most;
        if (budget > 0) {
            least = (blocks + each - 1) / each;                      // at least this
            if (least < floor) least = floor;
            if (least > most) least = most;
        }
    }
};

// By a whole warp.
__device__ __forceinline__ PrefixUnits prefix_units(const PrefixGroups& all, int kv_heads, int slots) {
    int tiles = 0, blocks = 0, longest = 0;
    for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
        const PrefixGroups x = all.from(g0);
        tiles += x.tiles; blocks += x.tiles * x.blocks; longest = max(longest, x.tiles > 0 ? x.blocks : 0);
    }
    tiles = __reduce_add_sync(0xffffffffu, tiles); blocks = __reduce_add_sync(0xffffffffu, blocks); longest = __reduce_max_sync(0xffffffffu, longest);
    const PrefixChunks tried(tiles, blocks, longest, slots / kv_heads);
    PrefixUnits u;
    u.chunk = tried.least;
    while (true) {
        int units = 0;
        for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
            const PrefixGroups x = all.from(g0);
            units += x.tiles * pu_ceil(x.blocks, u.chunk);
        }
        u.units = __reduce_add_sync(0xffffffffu, units) * kv_heads;
        if (u.chunk >= tried.most || u.units <= slots) return u;
        ++u.chunk;
    }
}

// Unit `want` (< units), by a whole warp.
__device__ __forceinline__ PrefixUnit prefix_unit(const PrefixGroups& all, int kv_heads, int chunk, int want) {
    const int lane = threadIdx.x & 31;
    PrefixUnit u = {};
    int before = 0;
    for (int g0 = 0; g0 < all.n_groups; g0 += 32) {
        const PrefixGroups x = all.from(g0);
        const int splits = pu_ceil(x.blocks, chunk), mine = x.tiles * splits * kv_heads;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += below;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + upto > want);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int at = __shfl_sync(0xffffffffu, before + upto - mine, src);
            u.group = g0 + src;
            u.splits = __shfl_sync(0xffffffffu, splits, src);
            u.tokens = __shfl_sync(0xffffffffu, x.tokens, src);
            u.slot = __shfl_sync(0xffffffffu, x.slot, src);
            const int in_group = __shfl_sync(0xffffffffu, x.count, src), first_row = __shfl_sync(0xffffffffu, x.start, src);
            const int rest = want - at, pair = pu_div(rest, u.splits);            // the unit's (tile, kv head)
            u.split = rest - pair * u.splits;
            u.tile = pu_div(pair, kv_heads);
            u.hk = pair - u.tile * kv_heads;
            u.first = at + u.tile * kv_heads * u.splits;
            u.start = first_row + u.tile * all.rows_per_tile;
            u.count = min(all.rows_per_tile, in_group - u.tile * all.rows_per_tile);
            return u;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return u;
}
