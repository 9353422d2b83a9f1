// Attention of rows that share their first pages over those pages' keys, which are read once for all of them: the queries
// that a kv head's group of heads has in a tile of rows are the rows of one matrix product. Leaves unnormalised partial
// results (maximum in log2 units, sum, weighted sum of values), which attention_rows.cu joins with each row's own keys.
// Any head size that is a multiple of 16 up to 256, any page size that the caches take; mma.sync m16n8k16 on bfloat16, codes turned
// into bfloat16 (exactly) as a tile is loaded. A persistent CTA of four warps takes 64 query rows against a unit's blocks of 64 keys.
// Bound by mma.sync and the loads that feed it (nothing overlaps a CTA's copies but the other CTAs of its SM): with the rows' own keys behind
// it 64 rows on 8,192 tokens take 71 us over 8-bit pages of 16 tokens (row by row 230), 32 rows on 16,384 71 us over bfloat16 ones (346).
// Tiles are loaded at one place in the code, four rows a thread at a time: all of a thread's rows at two places was code that took
// up to 15 us to come from memory (heads of 256, between other kernels), one row at a time 126 us in place of 71.
#include "attention_mma.cuh"
#include "cache8.cuh"
#include "prefix_units.cuh"

#define PX_ROWS 64                    // query rows a tile has at most (rows x heads a kv head)
#define PX_THREADS 128

struct PrefixArgs {
    float *part_o, *part_ml;
    int4* part_at;
    const bf16* q;
    const unsigned char* kv;
    const int32_t *block_table, *members, *groups;
    int n_groups, table_stride, heads, kv_heads, head_dim, pages, page_size;
    float scale_log2;
};

// Keys and values [j0, j0 + 64) of a kv head as bfloat16 tiles; keys from `hi` on become zeros.
template <int D_PAD, bool KV8>
__device__ __forceinline__ void load_shared_tile(uint32_t k_s, uint32_t v_s, const PrefixArgs& a, const int32_t* table, int hk, int j0, int hi) {
    constexpr int W = KV8 ? 16 : 8, CPR = D_PAD / W, STEP = PX_THREADS / CPR;      // numbers a chunk of 16 bytes of memory holds
    const int ch = threadIdx.x % CPR;
    if (ch * W >= a.head_dim) return;
    const int row_bytes = KV8 ? a.head_dim : 2 * a.head_dim;
    const size_t block = (size_t)a.page_size * (KV8 ? a.head_dim + 1 : 2 * a.head_dim), part = (size_t)a.kv_heads * block;
#pragma unroll 4
    for (int r = threadIdx.x / CPR; r < TILE_N; r += STEP) {
        const int j = j0 + r;
        bool valid = j < hi;
        size_t off = 0;
        int in = 0;
        if (valid) {
            const int pi = j / a.page_size, p = table[pi];
            valid = p >= 0 && p < a.pages;
            in = j - pi * a.page_size;
            off = (size_t)(valid ? p : 0) * 2 * part + (size_t)hk * block;
        }
        if constexpr (KV8) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                uint4 codes = make_uint4(0, 0, 0, 0), x, y;
                float scale = 0.f;
                if (valid) {
                    const unsigned char* b = a.kv + off + v * part;
                    codes = *(const uint4*)(b + (size_t)in * row_bytes + ch * 16);
                    scale = c8_power(min((int)b[(size_t)a.page_size * a.head_dim + in], 254) - 127);
                }
                c8_unpack16(codes, scale, x, y);
                const uint32_t t = v ? v_s : k_s;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(t + tile_off<D_PAD>(r, 2 * ch)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(t + tile_off<D_PAD>(r, 2 * ch + 1)), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w) : "memory");
            }
        } else {
            const unsigned char* src = a.kv + off + (valid ? (size_t)in * row_bytes + ch * 16 : 0);
            const uint32_t d = tile_off<D_PAD>(r, ch);
            cp_async16(k_s + d, src, valid);
            cp_async16(v_s + d, src + part, valid);
        }
    }
}

template <int D_PAD, bool KV8>
__global__ void __launch_bounds__(PX_THREADS) prefix_kernel(const PrefixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr uint32_t TILE_BYTES = TILE_N * D_PAD * 2;
    const uint32_t q_s = smem_u32(smem), kv_s = q_s + PX_ROWS * D_PAD * 2;          // two stages of keys and values
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads, per_tile = PX_ROWS / group, ksteps = a.head_dim >> 4;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // (attention_rows.cu may begin with the rows' own keys)
    const PrefixGroups known(a.groups, a.n_groups, per_tile);
    const PrefixUnits all = prefix_units(known, a.kv_heads, gridDim.x);
    const FragLanes f = frag_lanes<D_PAD>(lane);
    constexpr bool Q_IN_REGS = D_PAD <= 128;
    for (int w = blockIdx.x; w < all.units; w += gridDim.x) {
        const PrefixUnit u = prefix_unit(known, a.kv_heads, all.chunk, w);
        const int mrows = u.count * group;
        if (u.hk == 0 && u.split == 0 && threadIdx.x < u.count)
            a.part_at[a.members[u.start + threadIdx.x]] = make_int4(u.first, u.splits, (int)threadIdx.x * group, 0);
        __syncthreads();                                            // (the tiles are no longer read by the unit before)
        for (int i = threadIdx.x; i < PX_ROWS * (D_PAD / 8); i += PX_THREADS) {
            const int r = i / (D_PAD / 8), ch = i % (D_PAD / 8);
            const bool valid = r < mrows && ch * 8 < a.head_dim;
            const bf16* src = a.q;
            if (valid) src += ((size_t)a.members[u.start + r / group] * a.heads + u.hk * group + r % group) * a.head_dim + ch * 8;
            cp_async16(q_s + tile_off<D_PAD>(r, ch), src, valid);
        }
        cp_async_commit();
        const int32_t* table = a.block_table + (size_t)u.slot * a.table_stride;
        const int first = u.split * all.chunk, last = min((u.tokens + 63) / 64, first + all.chunk);
        uint32_t qf[Q_IN_REGS ? D_PAD / 16 : 1][4];
        float o[D_PAD / 8][4];
#pragma unroll
        for (int i = 0; i < D_PAD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (int tile = first - 1; tile < last; ++tile) {           // (the turn before the first tile only asks for it: one place loads)
            const uint32_t k_s = kv_s + ((tile - first) & 1) * 2 * TILE_BYTES, v_s = k_s + TILE_BYTES;
            if (tile >= first) {
                cp_async_wait<0>();
                __syncthreads();
            }
            if (tile + 1 < last) {
                const uint32_t next = kv_s + ((tile + 1 - first) & 1) * 2 * TILE_BYTES;
                load_shared_tile<D_PAD, KV8>(next, next + TILE_BYTES, a, table, u.hk, (tile + 1) * TILE_N, u.tokens);
            }
            cp_async_commit();
            if (tile < first || warp * 16 >= mrows) continue;       // (uniform per warp; the barrier is above)
            if (Q_IN_REGS && tile == first) {
#pragma unroll
                for (int ks = 0; ks < D_PAD / 16; ++ks)
                    if (ks < ksteps) ldmatrix_x4(qf[Q_IN_REGS ? ks : 0], q_s + warp * 16 * (D_PAD * 2) + f.a_row + ((ks * 32) ^ f.a_xor));
            }
            float s[8][4] = {};
#pragma unroll
            for (int ks = 0; ks < D_PAD / 16; ++ks) {
                if (ks < ksteps) {
                    uint32_t q4[4];
                    if (!Q_IN_REGS) ldmatrix_x4(q4, q_s + warp * 16 * (D_PAD * 2) + f.a_row + ((ks * 32) ^ f.a_xor));
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt) {
                        uint32_t kb[4];
                        ldmatrix_x4(kb, k_s + nt * 16 * (D_PAD * 2) + f.b_row + ((ks * 32) ^ f.b_xor));
                        mma_bf16(s[2 * nt], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : q4, kb[0], kb[1]);
                        mma_bf16(s[2 * nt + 1], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : q4, kb[2], kb[3]);
                    }
                }
            }
            if (tile * TILE_N + TILE_N > u.tokens) {
#pragma unroll
                for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (tile * TILE_N + nt * 8 + (lane & 3) * 2 + (e & 1) >= u.tokens) s[nt][e] = -INFINITY;
            }
            float c0, c1;
            softmax_step<8>(s, m0, m1, l0, l1, a.scale_log2, c0, c1);
            if (__any_sync(0xffffffffu, c0 != 1.f || c1 != 1.f)) {
#pragma unroll
                for (int i = 0; i < D_PAD / 8; ++i) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {                        // 16 keys a step
                const uint32_t p[4] = {pack_bf16(s[2 * kk][0], s[2 * kk][1]), pack_bf16(s[2 * kk][2], s[2 * kk][3]),
                                       pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
                for (int dt = 0; dt < D_PAD / 16; ++dt) {
                    if (dt < ksteps) {
                        uint32_t vb[4];
                        ldmatrix_x4_trans(vb, v_s + kk * 16 * (D_PAD * 2) + f.t_row + ((dt * 32) ^ f.t_xor));
                        mma_bf16(o[2 * dt], p, vb[0], vb[1]);
                        mma_bf16(o[2 * dt + 1], p, vb[2], vb[3]);
                    }
                }
            }
        }
        cp_async_wait<0>();
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const int c = (lane & 3) * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = warp * 16 + (lane >> 2) + 8 * h;
            if (r >= mrows) continue;
            const size_t slot = (size_t)w * PX_ROWS + r;
#pragma unroll
            for (int i = 0; i < D_PAD / 8; ++i)
                if (i * 8 < a.head_dim) *(float2*)(a.part_o + slot * a.head_dim + i * 8 + c) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            if (c == 0) *(float2*)(a.part_ml + slot * 2) = make_float2((h ? m1 : m0) * a.scale_log2, h ? l1 : l0);
        }
    }
}

template <int D_PAD, bool KV8> static int launch_prefix(const PrefixArgs& a, int ctas, cudaStream_t s) {
    auto kernel = prefix_kernel<D_PAD, KV8>;
    const int smem = (PX_ROWS + 4 * TILE_N) * D_PAD * 2;
    HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernel<<<ctas, PX_THREADS, smem, s>>>(a);
    HB_LAUNCH_CHECK("attention_prefix");
    return 0;
}

int hb_attention_prefix_tcgen05(float* part_o, float* part_ml, int32_t* part_at, const void* q, const void* kv, int kv8, const int32_t* block_table,
                                int table_stride, const int32_t* members, const int32_t* groups, int n_groups,
                                int heads, int kv_heads, int pages, int page_size, float scale, int ctas, cudaStream_t s);
static bool on_tcgen05(int head_dim, int page_size, int group) { return head_dim == 128 && page_size % 64 == 0 && group <= 128; }

extern "C" int hb_attention_prefix_plan(int head_dim, int page_size, int group, int* part_rows, int* tile_rows) {
    if (head_dim % 16 || head_dim > 256 || head_dim < 16 || group < 1 || page_size < 1) return 0;
    if (on_tcgen05(head_dim, page_size, group)) {
        *part_rows = 256;
        *tile_rows = 2 * (128 / group);
        return 1;
    }
    *part_rows = PX_ROWS;
    *tile_rows = PX_ROWS / group;
    return group > PX_ROWS ? 0 : head_dim > 128 ? 1 : 2;            // (above 128 a CTA's tiles take 160 KB)
}

extern "C" int hb_attention_prefix(float* part_o, float* part_ml, int32_t* part_at, const void* q, const void* kv, int kv8,
                                   const int32_t* block_table, int table_stride, const int32_t* members,
                                   const int32_t* groups, int n_groups, int heads, int kv_heads, int head_dim, int pages, int page_size, float scale,
                                   int ctas, hb_stream stream) {
    if (n_groups < 1 || ctas < 1) return 0;
    int part_rows, tile_rows;
    if (kv_heads < 1 || heads < 1 || heads % kv_heads || !hb_attention_prefix_plan(head_dim, page_size, heads / kv_heads, &part_rows, &tile_rows))
        HB_REFUSE("attention_prefix: %d heads, %d kv heads of %d", heads, kv_heads, head_dim);
    if (page_size < 16 || page_size % 16) HB_REFUSE("attention_prefix: page size %d is no multiple of 16", page_size);
    if (!(scale > 0.f)) HB_REFUSE("attention_prefix: the score scale must be positive");
    if (pages < 1 || (long)pages * 2 * kv_heads > 0x7ffffffel) HB_REFUSE("attention_prefix: %d pages of %d kv heads", pages, kv_heads);
    if (((uintptr_t)kv | (uintptr_t)q | (uintptr_t)part_at | (uintptr_t)groups) % 16 || (uintptr_t)part_o % 32 || (uintptr_t)part_ml % 8) HB_REFUSE("attention_prefix: tensors must start on 16 bytes");
    if (on_tcgen05(head_dim, page_size, heads / kv_heads))
        return hb_attention_prefix_tcgen05(part_o, part_ml, part_at, q, kv, kv8, block_table, table_stride, members, groups,
                                           n_groups, heads, kv_heads, pages, page_size, scale, ctas, (cudaStream_t)stream);
    const PrefixArgs a = {part_o, part_ml, (int4*)part_at, (const bf16*)q, (const unsigned char*)kv, block_table, members,
                          groups, n_groups, table_stride, heads, kv_heads, head_dim, pages, page_size, scale * 1.4426950408889634f};
    cudaStream_t s = (cudaStream_t)stream;
    if (kv8) return head_dim <= 64 ? launch_prefix<64, true>(a, ctas, s) : head_dim <= 128 ? launch_prefix<128, true>(a, ctas, s) : launch_prefix<256, true>(a, ctas, s);
    return head_dim <= 64 ? launch_prefix<64, false>(a, ctas, s) : head_dim <= 128 ? launch_prefix<128, false>(a, ctas, s) : launch_prefix<256, false>(a, ctas, s);
}
