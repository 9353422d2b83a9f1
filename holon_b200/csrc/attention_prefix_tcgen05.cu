// Attention of rows that share their first pages over those pages' keys, head size 128 and pages of a multiple of 64 tokens:
// attention_prefix.cu's work on tcgen05 tensor cores.
//
// A tile is up to two groups of 128 query rows (rows of the step x query heads of the kv head); a persistent CTA, one an SM, takes
// units of it (prefix_units.cuh). Per group and 64 keys, as in the kernel for prompts: S = Q K^T (128 x 64 x 16, eight products,
// operands in shared memory, S in one of two 64-column buffers of tensor memory); softmax with a query row a thread, the weights go back
// over the S they came from; O += P V (128 x 128 x 16, four products, P from tensor memory). The running maximum may lag by 2^8
// before O is rescaled. No key is masked: shared pages are whole, and whole numbers of 64 keys.
// bfloat16 pages: keys and values come by TMA as the products want them. 8-bit pages: TMA brings the codes, and four warps turn them
// into bfloat16, scale and all (exactly), in the same layout. (Halves without the scale would convert in fewer steps and leave the scales to
// the softmax: a factor and a term a score, a factor a weight, in threads that have no registers left. Not built.)
// Barriers keep their phases from unit to unit; every role counts the tiles that it has seen.
//
// Measured, with 32 heads over 8 kv heads and with the rows' own keys behind it: 64 rows on 8,192 tokens of 8-bit pages 35.3 us (in the mma.sync
// kernel 71, row by row 139), 32 rows on 16,384 of bfloat16 35.3 us (71; 246). Of the first one's 35,000 cycles here about 6,000 go by before
// a unit is known and 2,400 before its first keys are there, 8 tiles take 2,400 each (24 products, 100 cycles apiece: more than their
// arithmetic, whatever their shape), and 3,800 the results (19 MB of all CTAs). bfloat16 tiles come every 1,650, HBM's rate.
// Between other kernels it takes 2 to 4 us more: its code comes from memory anew, so loops that can do without are not unrolled.
// Looking the unit up in one warp for all (the look-up twice in the code) made the launch 0.8 us slower.
#include "cache8.cuh"
#include "prefix_units.cuh"
#include "tcgen05.cuh"

#define PT_D 128
#define PT_BM 128                                 // query rows per group
#define PT_GROUPS 2
#define PT_BN 64
#define PT_Q_BYTES (PT_BM * PT_D * 2)             // 32 KB a group: two [128 x 64] swizzled blocks
#define PT_KV_BYTES (PT_BN * PT_D * 2)            // 16 KB: two [64 x 64] swizzled blocks
#define PT_RAW_BYTES (PT_BN * PT_D)               // 8 KB of codes
#define PT_RAW_STAGE (2 * PT_RAW_BYTES + 1024)    // keys, values, 64 + 64 scale bytes
#define PT_TMEM_COLS 512                          // per group: S0 [0, 64), S1 [64, 128), O [128, 256)
#define PT_RESCALE 8.0f
#define PT_MMA_WARP1 10                           // warps 1 and 10: Q K^T of the groups; 11: P V; 2 - 9: softmax; 0: loads; 12 - 15: codes to bfloat16
#define PT_CONVERTERS 4

template <bool KV8> struct Shape {
    static constexpr int THREADS = KV8 ? 512 : 384;
    static constexpr int STAGES = 3;              // of keys and values as the products read them
    static constexpr int RAW = KV8 ? 3 : 1;       // of codes (bfloat16: none, and no barrier of theirs is used)
    static constexpr int KV = PT_GROUPS * PT_Q_BYTES, RAWS = KV + STAGES * 2 * PT_KV_BYTES;
    static constexpr int BARS = RAWS + (KV8 ? RAW * PT_RAW_STAGE : 0);
    static constexpr int SMEM = BARS + 256 + 1024;
};

struct PrefixTcArgs {
    float *part_o, *part_ml;
    int4* part_at;
    const bf16* q;
    const unsigned char* kv;
    const int32_t *block_table, *members, *groups;
    int n_groups, table_stride, heads, kv_heads, pages, page_size;
    float scale_log2;
};

__device__ __forceinline__ void pt_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

// A warp's 32 query rows into rows r0 .. r0 + 31 of a group's operand: lane i says where row r0 + i begins among the queries
// (negative: zeros). Eight lanes read a row, four rows at a time (a row a lane would ask for 32 lines an instruction, 16 times).
__device__ __forceinline__ void load_queries(uint32_t q_s, const bf16* q, long mine, int r0) {
    const int lane = threadIdx.x & 31, sub = lane & 7;
    uint4 x[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long at = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3));
        const uint4* src = (const uint4*)(q + (at < 0 ? 0 : at));
        x[i][0] = at < 0 ? make_uint4(0, 0, 0, 0) : src[sub];
        x[i][1] = at < 0 ? make_uint4(0, 0, 0, 0) : src[8 + sub];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + i * 4 + (lane >> 3);
        const uint32_t to = q_s + r * 128 + ((sub ^ (r & 7)) << 4);
        st_shared16(to, x[i][0]);
        st_shared16(to + PT_Q_BYTES / 2, x[i][1]);
    }
    fence_async_smem();                                               // (the products read them through the async proxy)
}
__device__ __forceinline__ void st_global32(float* dst, const uint32_t* v) {      // 32 bytes: a whole sector a thread
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <bool KV8>
__global__ void __launch_bounds__(Shape<KV8>::THREADS, 1) prefix_tcgen05_kernel(const __grid_constant__ CUtensorMap map_kv, const PrefixTcArgs a) {
    extern __shared__ unsigned char smem_raw[];
    using H = Shape<KV8>;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_addr(smem_raw));
    const uint32_t q_s = base, kv_s = base + H::KV, bars = base + H::BARS;
    const uint32_t kv_full0 = bars, kv_empty0 = kv_full0 + 8 * H::STAGES, raw_full0 = kv_empty0 + 8 * H::STAGES, raw_empty0 = raw_full0 + 8 * H::RAW;
    // per group g and buffer i, at index (g * 2 + i): scores computed; weights written; weights read (O holds the tile)
    const uint32_t s_full0 = raw_empty0 + 8 * H::RAW, p_full0 = s_full0 + 32, p_empty0 = p_full0 + 32, o_full0 = p_empty0 + 32, q_full = o_full0 + 16, slot = q_full + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads, per_group = PT_BM / group, per_tile = PT_GROUPS * per_group;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (attention_rows.cu may begin with the rows' own keys)

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_kv) : "memory");
        for (int s = 0; s < H::STAGES; ++s) { mbar_init(kv_full0 + 8 * s, KV8 ? PT_CONVERTERS : 1); mbar_init(kv_empty0 + 8 * s, 1 + PT_GROUPS); }
        for (int s = 0; s < H::RAW; ++s) { mbar_init(raw_full0 + 8 * s, 1); mbar_init(raw_empty0 + 8 * s, PT_CONVERTERS); }
        for (int i = 0; i < 2 * PT_GROUPS; ++i) { mbar_init(s_full0 + 8 * i, 1); mbar_init(p_full0 + 8 * i, 4); mbar_init(p_empty0 + 8 * i, 1); }
        for (int g = 0; g < PT_GROUPS; ++g) mbar_init(o_full0 + 8 * g, 1);
        mbar_init(q_full, 4 * PT_GROUPS);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot), "r"(PT_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    const PrefixGroups known(a.groups, a.n_groups, per_tile);
    const PrefixUnits all = prefix_units(known, a.kv_heads, gridDim.x);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(tmem) : "r"(slot));

    int seen = 0, turn = 0, g_seen[PT_GROUPS] = {0, 0}, g_units[PT_GROUPS] = {0, 0};   // tiles and units before this one: of all, of a group's own
    bool ok = true;
    for (int w = blockIdx.x; w < all.units; w += gridDim.x, ++turn) {
        const PrefixUnit u = prefix_unit(known, a.kv_heads, all.chunk, w);
        const int first = u.split * all.chunk, tiles = min(u.tokens / PT_BN, first + all.chunk) - first;
        int g_rows[PT_GROUPS];                                        // query rows of each group
#pragma unroll
        for (int g = 0; g < PT_GROUPS; ++g) g_rows[g] = max(0, min(per_group, u.count - g * per_group)) * group;
        if (warp == 0 && u.hk == 0 && u.split == 0)
            for (int i = lane; i < u.count; i += 32)
                a.part_at[a.members[u.start + i]] = make_int4(u.first, u.splits, i / per_group * PT_BM + i % per_group * group, 0);

        if (warp == 0) {
            const int32_t* table = a.block_table + (size_t)u.slot * a.table_stride;
            int asked = 0;                                            // tiles whose copies are on their way or there
            for (int t0 = 0; t0 < tiles && ok; t0 += 32) {
                const int key = (first + t0 + lane) * PT_BN, pi = key / a.page_size, in = key - pi * a.page_size;     // this lane's tile
                int page = t0 + lane < tiles ? table[pi] : 0;
                const bool there = page >= 0 && page < a.pages;       // (a page that is not there: zeros)
                const int k_block = there ? page * 2 * a.kv_heads + u.hk : 2 * a.pages * a.kv_heads;
                const int v_block = there ? k_block + a.kv_heads : k_block;
                const size_t bytes = (size_t)a.page_size * (PT_D + 1);
                const unsigned char* k_scale = a.kv + (size_t)(there ? k_block : u.hk) * bytes + (size_t)a.page_size * PT_D + in;
                for (int i = 0; i < 32 && t0 + i < tiles; ++i) {
                    const int n = seen + t0 + i, s = n % (KV8 ? H::RAW : H::STAGES), round = n / (KV8 ? H::RAW : H::STAGES);
                    ok = __all_sync(0xffffffffu, mbar_wait((KV8 ? raw_empty0 : kv_empty0) + 8 * s, (round & 1) ^ 1, 1));
                    if (!ok) break;
                    asked = t0 + i + 1;
                    if (lane != i) continue;
                    if (KV8) {
                        const uint32_t full = raw_full0 + 8 * s, dst = base + H::RAWS + s * PT_RAW_STAGE;
                        mbar_expect_tx(full, 2 * PT_RAW_BYTES + 128);
                        tma_load_3d(dst, &map_kv, full, 0, in, k_block);
                        tma_load_3d(dst + PT_RAW_BYTES, &map_kv, full, 0, in, v_block);
                        pt_bulk_load(dst + 2 * PT_RAW_BYTES, k_scale, 64, full);
                        pt_bulk_load(dst + 2 * PT_RAW_BYTES + 64, k_scale + (size_t)a.kv_heads * bytes, 64, full);
                    } else {
                        const uint32_t full = kv_full0 + 8 * s, dst = kv_s + s * 2 * PT_KV_BYTES;
                        mbar_expect_tx(full, 2 * PT_KV_BYTES);
                        tma_load_3d(dst, &map_kv, full, 0, in, k_block);
                        tma_load_3d(dst + PT_KV_BYTES / 2, &map_kv, full, 64, in, k_block);
                        tma_load_3d(dst + PT_KV_BYTES, &map_kv, full, 0, in, v_block);
                        tma_load_3d(dst + PT_KV_BYTES + PT_KV_BYTES / 2, &map_kv, full, 64, in, v_block);
                    }
                }
            }
            // No copy may come after the CTA's end, whoever gave up before (else others wait for them, too).
            constexpr int RING = KV8 ? H::RAW : H::STAGES;
#pragma unroll 1
            for (int n = seen + max(0, asked - RING); n < seen + asked; ++n) ok &= mbar_wait((KV8 ? raw_full0 : kv_full0) + 8 * (n % RING), (n / RING) & 1, 13);
            ok = __all_sync(0xffffffffu, ok);
        } else if (KV8 && warp >= 12) {
            const int part = warp - 12, sub = lane & 7;
            for (int j = 0; j < tiles && ok; ++j) {
                const int n = seen + j, s = n % H::RAW, d = n % H::STAGES;
                ok = mbar_wait(raw_full0 + 8 * s, (n / H::RAW) & 1, 2) && mbar_wait(kv_empty0 + 8 * d, ((n / H::STAGES) & 1) ^ 1, 3);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t raw = base + H::RAWS + s * PT_RAW_STAGE, dst = kv_s + d * 2 * PT_KV_BYTES;
                // Eight lanes read four chunks of 16 codes of a row and of row ^ 5, and write them as bfloat16: no two of either in one
                // group of banks. Warps 0 and 1 take the first halves of keys' and of values' rows, 2 and 3 the second ones.
                const int ch = (part >> 1) * 4 + (sub & 3), v = part & 1;
                const unsigned char* scales = smem + H::RAWS + s * PT_RAW_STAGE + 2 * PT_RAW_BYTES + v * PT_BN;
                const uint32_t to0 = dst + v * PT_KV_BYTES + (part >> 1) * (PT_KV_BYTES / 2);
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                    const int row = i * 8 + ((lane >> 3) ^ (sub >> 2) * 5);
                    const uint4 c = ld_shared16(raw + v * PT_RAW_BYTES + row * 128 + ((ch ^ (row & 7)) << 4));
                    uint4 lo, hi;
                    c8_unpack16(c, c8_power(min((int)scales[row], 254) - 127), lo, hi);
                    st_shared16(to0 + row * 128 + (((2 * (ch & 3)) ^ (row & 7)) << 4), lo);
                    st_shared16(to0 + row * 128 + (((2 * (ch & 3) + 1) ^ (row & 7)) << 4), hi);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) { mbar_arrive(kv_full0 + 8 * d); mbar_arrive(raw_empty0 + 8 * s); }
            }
        } else if (warp == 1 || (warp >= PT_MMA_WARP1 && warp < 12)) {
            if (lane == 0) {
                // kind::f16, D float32, A and B bfloat16; N / 8 at bit 17, M / 16 at bit 24; bit 16: B is MN-major
                const uint32_t types = (1u << 4) | (1u << 7) | (1u << 10);
                const uint32_t idesc_qk = types | ((uint32_t)(PT_BN >> 3) << 17) | ((uint32_t)(PT_BM >> 4) << 24);
                const uint32_t idesc_pv = types | (1u << 16) | ((uint32_t)(PT_D >> 3) << 17) | ((uint32_t)(PT_BM >> 4) << 24);
                if (warp <= PT_MMA_WARP1) {                           // the scores of group 0 or 1
                    const int g = warp == 1 ? 0 : 1;
                    ok = mbar_wait(q_full, turn & 1, 4);
                    for (int j = 0; j < tiles && ok; ++j) {           // (a group without rows still paces the stages)
                        const int n = seen + j, s = n % H::STAGES;
                        ok = mbar_wait(kv_full0 + 8 * s, (n / H::STAGES) & 1, 5);
                        if (ok && g_rows[g] > 0) {
                            const int k = g_seen[g] + j, gb = g * 2 + (k & 1);
                            // S overwrites S and P of two tiles ago: wait until their P V has read them
                            ok = mbar_wait(p_empty0 + 8 * gb, ((k >> 1) & 1) ^ 1, 6);
                            if (!ok) break;
                            tc_fence_after();
                            const uint32_t k_src = kv_s + s * 2 * PT_KV_BYTES, s_t = tmem + g * 256 + (k & 1) * PT_BN;
#pragma unroll
                            for (int kk = 0; kk < PT_D / 16; ++kk) {  // d 0..63 in the first block, 64..127 in the second
                                const uint32_t blk = kk >> 2, within = (kk & 3) * 2;
                                tc_mma(s_t, tc_smem_desc(q_s + g * PT_Q_BYTES + blk * (PT_Q_BYTES / 2)) + within,
                                       tc_smem_desc(k_src + blk * (PT_KV_BYTES / 2)) + within, idesc_qk, kk != 0);
                            }
                            tc_commit(s_full0 + 8 * gb);
                        }
                        if (ok) tc_commit(kv_empty0 + 8 * s);         // the keys of the stage have been read (all three must arrive)
                    }
                } else {
                    for (int j = 0; j < tiles && ok; ++j) {
                        const int n = seen + j, s = n % H::STAGES;
                        ok = mbar_wait(kv_full0 + 8 * s, (n / H::STAGES) & 1, 7);
                        for (int g = 0; g < PT_GROUPS && ok; ++g) {   // O_g += P_g V
                            if (g_rows[g] == 0) continue;
                            const int k = g_seen[g] + j, gb = g * 2 + (k & 1);
                            ok = mbar_wait(p_full0 + 8 * gb, (k >> 1) & 1, 8);
                            if (!ok) break;
                            tc_fence_after();
                            const uint32_t v_src = kv_s + s * 2 * PT_KV_BYTES + PT_KV_BYTES;
                            const uint32_t o_t = tmem + g * 256 + 2 * PT_BN, p_t = tmem + g * 256 + (k & 1) * PT_BN;   // P lies over the first half of its own S
#pragma unroll
                            for (int kk = 0; kk < PT_BN / 16; ++kk)   // 16 keys a step: 8 columns along P, 16 rows down V
                                tc_mma_f16_ts(o_t, p_t + kk * 8, tc_smem_desc_mn(v_src + kk * 16 * 128, PT_KV_BYTES / 2), idesc_pv, (j | kk) != 0);
                            tc_commit(p_empty0 + 8 * gb);             // P has been read; O_g holds the tile
                            if (j == tiles - 1) tc_commit(o_full0 + 8 * g);
                        }
                        if (ok) tc_commit(kv_empty0 + 8 * s);         // the values of the stage have been read
                    }
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        } else if (warp >= 2 && warp < PT_MMA_WARP1) {
            const int g = (warp - 2) >> 2;                            // this warp's group of query rows
            const int quarter = warp & 3;                             // and its quarter of the TMEM lanes
            const int r = quarter * 32 + lane;                        // this thread's query row within the group
            const uint32_t lane_t = tmem + g * 256 + ((uint32_t)(quarter * 32) << 16);
            const uint32_t o_t = lane_t + 2 * PT_BN;
            float m_used = -INFINITY, l = 0.f;                        // in log2 units; the maximum may lag by PT_RESCALE
            if (g_rows[g] > 0) {
                long mine = -1;                                       // (one-token rows come first: a row's number is its token's)
                if (r < g_rows[g]) mine = ((long)a.members[u.start + g * per_group + r / group] * a.heads + u.hk * group + r % group) * PT_D;
                load_queries(q_s + g * PT_Q_BYTES, a.q, mine, quarter * 32);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            const uint64_t factor2 = pack2(a.scale_log2, a.scale_log2);
            if (g_rows[g] > 0) {
                for (int j = 0; j < tiles && ok; ++j) {
                    const int k = g_seen[g] + j, gb = g * 2 + (k & 1);
                    ok = mbar_wait(s_full0 + 8 * gb, (k >> 1) & 1, 9);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    uint32_t sr[2][32];
                    tc_ld32_nowait(lane_t + (k & 1) * PT_BN, sr[0]);
                    tc_ld32_nowait(lane_t + (k & 1) * PT_BN + 32, sr[1]);
                    tc_ld_wait();
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // four chains instead of one of 64
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(sr[c][i]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    const float mt = mx * a.scale_log2;
                    const bool grow = mt > m_used + PT_RESCALE || (m_used == -INFINITY && mt > -INFINITY);
                    if (__any_sync(0xffffffffu, grow)) {              // rescale what is summed (whole warp: the TMEM ops are collective)
                        const float m_new = grow ? mt : m_used;
                        const float f = m_used == -INFINITY ? 0.f : at_ex2(m_used - m_new);
                        if (j > 0) {
                            ok = mbar_wait(p_empty0 + 8 * (g * 2 + ((k - 1) & 1)), ((k - 1) >> 1) & 1, 10);   // O holds every tile before this one
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < PT_D / 32; ++c) {
                                uint32_t o[32];
                                tc_ld32(o_t + c * 32, o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc_st32(o_t + c * 32, o);
                            }
                        }
                        l *= f;
                        m_used = m_new;
                    }
                    const float off = m_used == -INFINITY ? 0.f : -m_used;
                    const uint64_t off2 = pack2(off, off);
                    uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};      // four chains of packed sums
                    uint32_t pk[32];                                  // 64 weights as pairs
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float x, y;
                            const uint64_t pair = pack2(__uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
                            unpack2(fma2(pair, factor2, off2), x, y);
                            x = at_ex2(x);
                            y = at_ex2(y);
                            sum2[(i >> 1) & 3] = add2(sum2[(i >> 1) & 3], pack2(x, y));
                            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
                            pk[c * 16 + i / 2] = *(const uint32_t*)&h;
                        }
                    float lo, hi;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), lo, hi);
                    l += lo + hi;
                    tc_st32(lane_t + (k & 1) * PT_BN, pk);            // P over the S it came from: 32 columns of pairs
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full0 + 8 * gb);
                }
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_full0 + 8 * g, g_units[g] & 1, 11));
                tc_fence_after();
                if (ok) {                                             // (the tensor-memory loads are warp-collective: no lane skips them)
                    const size_t at = (size_t)w * (PT_GROUPS * PT_BM) + g * PT_BM + r;
                    const bool mine = r < g_rows[g];
                    if (mine) *(float2*)(a.part_ml + at * 2) = make_float2(m_used, l);
#pragma unroll 1
                    for (int c = 0; c < PT_D / 32; ++c) {
                        uint32_t o[32];
                        tc_ld32(o_t + c * 32, o);
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) st_global32(a.part_o + at * PT_D + c * 32 + i, o + i);
                        }
                    }
                    tc_fence_before();
                }
            }
        }
        seen += tiles;
#pragma unroll
        for (int g = 0; g < PT_GROUPS; ++g)
            if (g_rows[g] > 0) { g_seen[g] += tiles; ++g_units[g]; }
        if (!__syncthreads_and((int)ok)) break;                       // a wait that gave up anywhere ends the walk everywhere
        tc_fence_after();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(PT_TMEM_COLS) : "memory");
    }
}

HB_DEFINE_STATUS_MIRROR(hb_attention_prefix_status_mirror)
extern "C" int hb_attention_prefix_status(unsigned int* status) {
    HB_CUDA(cudaDeviceSynchronize());
    HB_CUDA(cudaMemcpyFromSymbol(status, g_tc_status, sizeof(unsigned int)));
    const unsigned int zero = 0;
    HB_CUDA(cudaMemcpyToSymbol(g_tc_status, &zero, sizeof(unsigned int)));
    return 0;
}

template <bool KV8> static int launch(const PrefixTcArgs& a, int ctas, cudaStream_t s) {
    using H = Shape<KV8>;
    const uint64_t bytes = KV8 ? 1 : 2;
    CUtensorMap map;
    const cuuint64_t dims[3] = {PT_D, (cuuint64_t)a.page_size, (cuuint64_t)a.pages * 2 * a.kv_heads};
    const cuuint64_t strides[2] = {PT_D * bytes, a.page_size * (uint64_t)(PT_D + (KV8 ? 1 : 0)) * bytes};
    const cuuint32_t box[3] = {KV8 ? 128u : 64u, PT_BN, 1}, elem[3] = {1, 1, 1};
    const CUresult r = cuTensorMapEncodeTiled(&map, KV8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                                              const_cast<unsigned char*>(a.kv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) HB_REFUSE("attention_prefix: cuTensorMapEncodeTiled failed with %d", (int)r);
    auto kernel = prefix_tcgen05_kernel<KV8>;
    static unsigned long long prepared = 0;                           // devices that the kernel's limit is set on
    int device = 0;
    HB_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !(prepared >> device & 1)) {
        HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, H::SMEM));
        if (device < 64) prepared |= 1ull << device;
    }
    kernel<<<ctas, H::THREADS, H::SMEM, s>>>(map, a);
    HB_LAUNCH_CHECK("attention_prefix");
    return 0;
}

// hb_attention_prefix's work where head_dim is 128 and pages are multiples of 64 tokens (its checks are done).
int hb_attention_prefix_tcgen05(float* part_o, float* part_ml, int32_t* part_at, const void* q, const void* kv, int kv8, const int32_t* block_table,
                                int table_stride, const int32_t* members, const int32_t* groups,
                                int n_groups, int heads, int kv_heads, int pages, int page_size, float scale, int ctas, cudaStream_t s) {
    const PrefixTcArgs a = {part_o, part_ml, (int4*)part_at, (const bf16*)q, (const unsigned char*)kv, block_table, members,
                            groups, n_groups, table_stride, heads, kv_heads, pages, page_size, scale * 1.4426950408889634f};
    return kv8 ? launch<true>(a, ctas, s) : launch<false>(a, ctas, s);
}
