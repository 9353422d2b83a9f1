// Attention of rows that bring one token each, over pages of 8-bit codes, and over the keys that rows which share their
// first pages hold behind those (pages of either kind).
//
// A CTA owns (row, kv head, split of the row's keys, up to eight of the kv head's query heads). A fifth warp brings tiles of keys by
// TMA; four warps take 32 keys each of every tile, keep their own running softmax and are merged in shared memory; the splits of a
// (row, kv head) are one thread-block cluster and are merged through distributed shared memory, in the order of the splits. With
// `skip` (tokens a row shares with others) the walk starts behind them, and the partial results that attention_prefix.cu left
// for the shared keys are added in the same merge.
//
// Both products have the heads as their eight columns: S^T = K Q^T (16 keys a product) and O^T = V^T P^T (16 numbers of the head), so
// that eight heads fill the shape and a lane's maxima and sums belong to the columns of its outputs; the weights pass from one
// product's result to the other's operand by a transposition of 8 x 8 blocks.
// 8-bit pages: codes become halves, which hold every code exactly. (mma.sync m16n8k32 on codes themselves: 9 executed instructions by
// counter, an m16n8k16 on halves 2.5, the conversion of four codes 2.5.) With k_j = 2^a_j K_j and
// v_j = 2^b_j V_j (K, V codes) and the head's query scaled into the halves' range by a power of two 2^-c,
//     u_j = (q 2^-c . K_j) 2^(a_j + c) scale log2(e) + b_j,   w_j = 2^(u_j - M),   O = sum w_j V_j,   l = sum w_j 2^-b_j
// with M the running maximum of u, not of the scores: the weights that meet the codes stay at most 2^14 whatever the values' scales
// are (14 is taken off M so that small weights are no subnormal halves), and l sums the softmax's own weights in the same units. Keys whose
// weights vanish in 32 bits (below 2^-126) would be missing in l: they are less than 2^-25 of it in all, for up to 2^20 keys, while the b of a
// head lie within 2^80 of one another (a value of zeros has b = -64: values up to 2^24 beside such). Where keys with values of (nearly) zeros
// take all but 2^-28 of the weight, the others' weights are subnormal halves with fewer bits.
// ldmatrix moves pairs of codes as it moves bfloat16: of a key a lane gets codes 4 c .. 4 c + 3 where the fragment wants columns 2 c,
// 2 c + 1, 2 c + 8, 2 c + 9, so queries are laid out in that order; of values it gets two neighbouring codes of two keys, one byte
// permutation pairs the keys, and the even numbers of the head are the product's rows 0 - 7, the odd ones its rows 8 - 15.
//
// Measured with 32 heads over 8 kv heads of 128, 8-bit pages of 64: 64 rows of 600 to 4,096 tokens 55.5 us (312 MB, 5.6 TB/s, 87% of
// what a copy reaches), 8 rows of 8,192 28.3 us (135 MB, 4.8 TB/s): bound by HBM and, below some 30 us, by a CTA's start (three loads that
// wait for one another, 1.8 us) and end. One row of 400 tokens 6.6 us: only start and end. Heads as columns and tiles by TMA in place of
// heads as padded rows and cp.async: 8 rows of 8,192 tokens 52.0 -> 28.8 us, 64 rows 144.5 -> 67.8; longest rows first 67.0 -> 54.8.
// Behind a shared beginning of 8,192 tokens (64 rows with up to 256 keys of their own) about 12 us, of which 3 weigh 19 MB of partial results.
#include <cuda_fp16.h>

#include "attention_mma.cuh"
#include "cache8.cuh"
#include "prefix_units.cuh"
#include "tcgen05.cuh"

#define AR_WARPS 4                    // that compute; one more loads
#define AR_THREADS (32 * AR_WARPS + 32)
#define AR_HEADS 8
#define AR_CLUSTER 16                 // splits at most
#define AR_BIAS 14.f
#define AR_BY_LENGTH 1024             // rows whose lengths a CTA has room to rank (what pays is the caller's to say)
#define AR_NK(D_PAD, KV8) ((KV8) || (D_PAD) <= 64 ? 2 : 1)
#define AR_STAGES(BYTES) ((BYTES) <= 16384 ? 4 : (BYTES) <= 32768 ? 3 : 2)

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 block of 16-bit numbers, transposed within the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *(uint32_t*)&v;
}
__device__ __forceinline__ void st_cluster_f32(const float* local, uint32_t rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(remote), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_f32x4(const float* local, uint32_t rank, const float4& v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// An untiled copy of a few bytes (16-byte boundaries and size), counted on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

struct RowsArgs {
    bf16* out;                     // [tokens, heads, head_dim]
    const bf16* q;
    const unsigned char* kv;
    const int32_t *block_table, *row_slot, *query_start, *kv_len;
    const float* sinks;
    const int32_t* skip;           // tokens a row shares (their partial results are in part_*), or null
    const float *part_o, *part_ml; // [units, part_rows, head_dim] and [units, part_rows, 2]
    const int4* part_at;           // per row: the first unit of kv head 0, units a kv head, where the row's heads start among a unit's part_rows
    int part_rows, part_units, table_stride, rows, heads, kv_heads, head_dim, pages, page_size, page_shift, box, window, splits, by_length;
    float scale_log2;
};

// A stage's tile of KEYS keys (FEW: 64, two stages: for rows of a few hundred keys, whose time is a CTA's start and end; an SM holds four
// such CTAs where it holds two of the others, bfloat16 heads of 128 three, 8-bit heads of 64 four in place of three, above 128 8-bit ones
// two in place of one and bfloat16 ones no more): keys, then values, each as column blocks [KEYS rows][SUB bytes] that TMA swizzles over SUB bytes.
template <int D_PAD, bool KV8, bool FEW> struct Tile {
    static constexpr int ROW = KV8 ? D_PAD : 2 * D_PAD;              // bytes of a key
    static constexpr int NK = FEW ? 1 : AR_NK(D_PAD, KV8), KEYS = 16 * AR_WARPS * NK;   // a warp takes NK times 16 keys of a tile
    static constexpr int SUB = ROW < 128 ? ROW : 128, NSUB = ROW / SUB, BLOCK = KEYS * SUB;
    static constexpr int PART = NSUB * BLOCK, STAGE = 2 * PART;
    static constexpr int STAGES = FEW ? 2 : AR_STAGES(STAGE);
    static constexpr int SUMS = (AR_WARPS * AR_HEADS * (D_PAD + 2)) * 4;      // what the warps leave, over the tiles
    static constexpr int BODY = STAGES * STAGE > SUMS ? STAGES * STAGE : SUMS;
    static constexpr int BARS = BODY + STAGES * 2 * KEYS;            // behind the tiles: a stage's scale bytes, then the barriers
    static constexpr int RECV = BARS + 16 * STAGES;                  // then what the other CTAs of a cluster send
    // CTAs an SM that registers are cut for: of the form for few keys what its 228 KB hold (1 KB of each is the system's, 1 KB goes to the
    // boundary), up to four; of the other three, of which two or three fit (8 rows of 8,192 keys 28.0 us in 128 registers, 28.5 in the 143 that two would leave).
    static constexpr int FIT = (228 * 1024) / (RECV + 2048), CTAS = D_PAD > 128 ? 1 : !FEW ? 3 : FIT < 4 ? FIT : 4;
};
// Byte offset of (row, 16-byte chunk) in a part of a tile: eight rows at one chunk lie in eight bank groups.
template <int D_PAD, bool KV8, bool FEW> __device__ __forceinline__ uint32_t tile_at(int row, int chunk) {
    using T = Tile<D_PAD, KV8, FEW>;
    if (T::SUB == 64) return (uint32_t)(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
    return (uint32_t)((chunk >> 3) * T::BLOCK + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// The loading warp: tiles [first, last) of (row, kv head). A tile is KEYS / box boxes of `box` keys that lie in one page each. Keys in
// pages that do not exist, and boxes behind the row's last key, are zeros (their scales: those of the first page).
template <int D_PAD, bool KV8, bool FEW>
__device__ __forceinline__ void load_tiles(const CUtensorMap* map, const RowsArgs& a, uint32_t base, const int32_t* table, int hk, int first, int last,
                                           int n) {
    using T = Tile<D_PAD, KV8, FEW>;
    const int lane = threadIdx.x & 31, boxes = T::KEYS / a.box, batch = 32 / boxes;
    const uint32_t full = base + T::BARS, empty = full + 8 * T::STAGES;
    const uint32_t bytes = T::STAGE + (KV8 ? 2 * T::KEYS : 0);
    const size_t block = (size_t)a.page_size * (a.head_dim + 1);
    int asked = 0;                                                   // tiles whose copies are on their way or there
    bool ok = true;
    for (int t0 = first; t0 < last && ok; t0 += batch) {
        const int key = t0 * T::KEYS + lane * a.box, pi = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size, in = key - pi * a.page_size;   // this lane's box
        const int page = lane < batch * boxes && key < n ? table[pi] : -1;
        const bool there = page >= 0 && page < a.pages;
        const int k_block = there ? page * 2 * a.kv_heads + hk : 2 * a.pages * a.kv_heads, v_block = there ? k_block + a.kv_heads : k_block;
        const unsigned char* k_scale = a.kv + (size_t)(there ? k_block : hk) * block + (size_t)a.page_size * a.head_dim + in;
        const unsigned char* v_scale = k_scale + (size_t)a.kv_heads * block;
        for (int i = 0; i < batch && t0 + i < last; ++i) {
            const int j = t0 + i - first, s = j % T::STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((j / T::STAGES) & 1) ^ 1, 1));
            if (!ok) break;
            asked = j + 1;
            if (lane == 0) mbar_expect_tx(full + 8 * s, bytes);
            __syncwarp();
            if (lane / boxes != i) continue;
            const uint32_t row = (lane % boxes) * a.box, dst = base + s * T::STAGE + row * T::SUB;
#pragma unroll
            for (int c = 0; c < T::NSUB; ++c) {                      // (columns past head_dim: zeros)
                tma_load_3d(dst + c * T::BLOCK, map, full + 8 * s, c * (KV8 ? T::SUB : T::SUB / 2), in, k_block);
                tma_load_3d(dst + T::PART + c * T::BLOCK, map, full + 8 * s, c * (KV8 ? T::SUB : T::SUB / 2), in, v_block);
            }
            if (KV8) {
                const uint32_t at = base + T::BODY + s * 2 * T::KEYS + row;
                bulk_load(at, k_scale, a.box, full + 8 * s);
                bulk_load(at + T::KEYS, v_scale, a.box, full + 8 * s);
            }
        }
    }
    // No copy may come after the CTA's end, whoever gave up before (else the computing warps wait for them, too).
#pragma unroll 1
    for (int j = max(0, asked - T::STAGES); j < asked; ++j) mbar_wait(full + 8 * (j % T::STAGES), (j / T::STAGES) & 1, 3);
}

// The B fragments of up to eight heads' queries at `q` (head_dim apart), head lane / 4; for codes as halves, each head divided by a
// power of two that brings its largest number near 2^6, which `up` undoes.
template <int D_PAD, bool KV8> struct Query {
    uint32_t f[D_PAD / 16][2];
    float up = 1.f;
    __device__ __forceinline__ void load(const bf16* q, int g, int head_dim) {
        const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
        const bf16* row = q + (size_t)(r < g ? r : 0) * head_dim;
        if constexpr (!KV8) {
#pragma unroll
            for (int ks = 0; ks < D_PAD / 16; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    f[ks][h] = r < g && ks * 16 < head_dim ? *(const uint32_t*)(row + ks * 16 + 8 * h + 2 * c) : 0u;
        } else {
            float m = 0.f;
#pragma unroll
            for (int ks = 0; ks < D_PAD / 16; ++ks) {
                const uint2 w = r < g && ks * 16 < head_dim ? *(const uint2*)(row + ks * 16 + 4 * c) : make_uint2(0u, 0u);
                const float2 x = __bfloat1622float2(*(const __nv_bfloat162*)&w.x), y = __bfloat1622float2(*(const __nv_bfloat162*)&w.y);
                m = fmaxf(fmaxf(m, fmaxf(c8_magnitude(x.x), c8_magnitude(x.y))), fmaxf(c8_magnitude(y.x), c8_magnitude(y.y)));
                f[ks][0] = w.x; f[ks][1] = w.y;
            }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const int e = min(max((int)(__float_as_uint(m) >> 23) - 127 - 6, -100), 121);
            const float down = c8_power(-e);
            up = c8_power(e);
#pragma unroll
            for (int ks = 0; ks < D_PAD / 16; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 x = __bfloat1622float2(*(const __nv_bfloat162*)&f[ks][h]);
                    f[ks][h] = pack_f16(x.x * down, x.y * down);
                }
        }
    }
};

__device__ __forceinline__ float column_max(float v) {              // over the eight lanes that hold a column
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// A computing warp's walk over tiles [first, last); leaves its sums over the tiles' memory: [warp][8][D_PAD] floats and
// [warp][g][2] (maximum in log2 units, sum), once every warp is done with the tiles.
template <int D_PAD, bool KV8, bool FEW>
__device__ __forceinline__ void walk(unsigned char* smem, uint32_t base, const RowsArgs& a, const bf16* q, int g, int first, int last, int lo, int n) {
    using T = Tile<D_PAD, KV8, FEW>;
    constexpr int NK = T::NK;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const uint32_t full = base + T::BARS, empty = full + 8 * T::STAGES;
    Query<D_PAD, KV8> query;
    query.load(q, g, a.head_dim);
    float up[2];                                                     // of heads 2 c, 2 c + 1
#pragma unroll
    for (int h = 0; h < 2; ++h) up[h] = __shfl_sync(0xffffffffu, query.up, 8 * c + 4 * h) * a.scale_log2;
    float o[D_PAD / 16][4];                                          // 16 numbers of the head x heads 2 c, 2 c + 1
#pragma unroll
    for (int i = 0; i < D_PAD / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int row = warp * 16 * NK + (lane & 15), ch = lane >> 4;   // ldmatrix: (rows 0-7, chunk), (8-15, chunk), (0-7, next), (8-15, next)

    for (int tile = first; tile < last; ++tile) {
        const int j = tile - first, stage = j % T::STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * stage, (j / T::STAGES) & 1, 2))) break;
        const int key0 = tile * T::KEYS + warp * 16 * NK;            // this warp's keys
        const uint32_t kt = base + stage * T::STAGE, vt = kt + T::PART;
        if (key0 < n && key0 + 16 * NK > lo) {
            float u[NK][4];                                          // keys r, r + 8 of each 16 x heads 2 c, 2 c + 1
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                u[kk][0] = u[kk][1] = u[kk][2] = u[kk][3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < D_PAD / 16; ks += KV8 ? 2 : 1) {
                    uint32_t x[4];
                    ldmatrix_x4(x, kt + tile_at<D_PAD, KV8, FEW>(row + 16 * kk, (KV8 ? ks : 2 * ks) + ch));
                    if constexpr (KV8) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t k[4] = {c8_halves(x[2 * h]), c8_halves(x[2 * h + 1]), c8_halves(x[2 * h] >> 16), c8_halves(x[2 * h + 1] >> 16)};
                            mma_f16(u[kk], k, query.f[ks + h][0], query.f[ks + h][1]);
                        }
                    } else {
                        mma_bf16(u[kk], x, query.f[ks][0], query.f[ks][1]);
                    }
                }
            }
            float drop[NK][2];                                       // 2^-b of this lane's keys
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    drop[kk][i] = 1.f;
                    if (KV8) {                                       // (a byte that is never written, in a page that is not there: codes of 0)
                        uint32_t kb, b;
                        const uint32_t at = base + T::BODY + stage * 2 * T::KEYS + warp * 16 * NK + kk * 16 + i * 8 + r;
                        asm volatile("ld.shared.u8 %0, [%1];\n" : "=r"(kb) : "r"(at));
                        asm volatile("ld.shared.u8 %0, [%1];\n" : "=r"(b) : "r"(at + T::KEYS));
                        kb = min(kb, 254u); b = min(max(b, (uint32_t)(C8_LOW + 127)), 254u);
                        const float ka = __uint_as_float(kb << 23), vb = (float)((int)b - 127);
                        drop[kk][i] = __uint_as_float((254u - b) << 23);
                        u[kk][2 * i] = fmaf(u[kk][2 * i], ka * up[0], vb);
                        u[kk][2 * i + 1] = fmaf(u[kk][2 * i + 1], ka * up[1], vb);
                    } else {
                        u[kk][2 * i] *= up[0];
                        u[kk][2 * i + 1] *= up[1];
                    }
                }
            if (key0 < lo || key0 + 16 * NK > n) {
                // Keys before `lo` and from `n` on: no score, and values that are zeros whatever their bytes say (a weight of zero
                // times no number is none). The next copy into this stage comes behind the fence.
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = key0 + kk * 16 + i * 8 + r;
                        if (key < lo || key >= n) u[kk][2 * i] = u[kk][2 * i + 1] = -INFINITY;
                    }
                for (int i = lane; i < 16 * NK * (T::ROW / 16); i += 32) {
                    const int at = i / (T::ROW / 16), key = key0 + at;
                    if (key < lo || key >= n)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(vt + tile_at<D_PAD, KV8, FEW>(warp * 16 * NK + at, i % (T::ROW / 16))), "r"(0u) : "memory");
                }
                fence_async_smem();
                __syncwarp();
            }
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = u[0][h];
#pragma unroll
                for (int i = 1; i < 2 * NK; ++i) mx = fmaxf(mx, u[i >> 1][2 * (i & 1) + h]);
                const float top = fmaxf(m[h], column_max(mx) - (KV8 ? AR_BIAS : 0.f)), off = top == -INFINITY ? 0.f : top;
                f[h] = ex2(m[h] - off);                              // (nothing yet: 2^(-inf) = 0)
                m[h] = top;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) {
                    float& w = u[i >> 1][2 * (i & 1) + h];
                    w = ex2(w - off);
                    sum = KV8 ? fmaf(w, drop[i >> 1][i & 1], sum) : sum + w;
                }
                l[h] = fmaf(l[h], f[h], sum);                        // this lane's keys; the column is joined at the end
            }
            if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {   // a running maximum moved: rescale what is summed
#pragma unroll
                for (int i = 0; i < D_PAD / 16; ++i) { o[i][0] *= f[0]; o[i][1] *= f[1]; o[i][2] *= f[0]; o[i][3] *= f[1]; }
            }
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                uint32_t p[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    p[i] = transposed(KV8 ? pack_f16(u[kk][2 * i], u[kk][2 * i + 1]) : pack_bf16(u[kk][2 * i], u[kk][2 * i + 1]));
#pragma unroll
                for (int d = 0; d < D_PAD / 16; d += KV8 ? 2 : 1) {
                    uint32_t x[4];
                    ldmatrix_x4_trans(x, vt + tile_at<D_PAD, KV8, FEW>(row + 16 * kk, (KV8 ? d : 2 * d) + ch));
                    if constexpr (KV8) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {                // two neighbouring codes of two keys -> pairs of keys: even numbers, odd ones
                            const uint32_t y0 = __byte_perm(x[2 * h], 0, 0x3120), y1 = __byte_perm(x[2 * h + 1], 0, 0x3120);
                            const uint32_t v[4] = {c8_halves(y0), c8_halves(y0 >> 16), c8_halves(y1), c8_halves(y1 >> 16)};
                            mma_f16(o[d + h], v, p[0], p[1]);
                        }
                    } else {
                        const uint32_t v[4] = {x[0], x[2], x[1], x[3]};
                        mma_bf16(o[d], v, p[0], p[1]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * stage);
    }
    l[0] = column_sum(l[0]); l[1] = column_sum(l[1]);
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * AR_WARPS) : "memory");   // every warp is done with the tiles: reuse them
    float* wo = (float*)smem;
#pragma unroll
    for (int i = 0; i < D_PAD / 16; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (2 * c + h >= g) continue;
            float* to = wo + (warp * AR_HEADS + 2 * c + h) * D_PAD + i * 16;
            if (KV8) *(float2*)(to + 2 * r) = make_float2(o[i][h], o[i][2 + h]);
            else { to[r] = o[i][h]; to[8 + r] = o[i][2 + h]; }
        }
    if (r == 0)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (2 * c + h < g) *(float2*)(wo + AR_WARPS * AR_HEADS * D_PAD + (warp * g + 2 * c + h) * 2) = make_float2(m[h], l[h]);
}

// How `pieces` partial results [pieces][g][2] (maximum in log2 units, sum) of each of g heads, and the `parts` ones of the shared keys
// that start at `part` (a head's are `stride` floats apart from split to split, neighbouring heads' lie side by side), are weighed:
// weights to w [g][pieces + parts], maximum and sum of the whole to whole [g][2]. A warp takes a head; no piece's order matters to
// the maximum, and the sums' order depends on the numbers alone.
__device__ __forceinline__ void weigh(float* w, float* whole, const float* ml, int pieces, int g, const float* part, size_t stride, int parts) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = pieces + parts;
    for (int r = warp; r < g; r += AR_THREADS / 32) {
        float top = -INFINITY;
        for (int i = lane; i < count; i += 32) {
            const float m = i < pieces ? ml[(i * g + r) * 2] : part[(i - pieces) * stride + r * 2];
            w[r * count + i] = m;                                    // (its own lane reads it again)
            top = fmaxf(top, m);
        }
        top = warp_max(top);
        const float off = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        for (int i = lane; i < count; i += 32) {
            const float l = i < pieces ? ml[(i * g + r) * 2 + 1] : part[(i - pieces) * stride + r * 2 + 1], f = ex2(w[r * count + i] - off);
            w[r * count + i] = f;
            sum = fmaf(l, f, sum);                                   // (a sum that is no number stays one)
        }
        sum = warp_sum(sum);
        if (lane == 0) { whole[2 * r] = top; whole[2 * r + 1] = sum; }
    }
}
__device__ __forceinline__ void add4(float4& x, float w, const float4& y) {
    x.x = fmaf(w, y.x, x.x); x.y = fmaf(w, y.y, x.y); x.z = fmaf(w, y.z, x.z); x.w = fmaf(w, y.w, x.w);
}

// The row whose own keys are `rank` rows' from the longest (of equal ones the first): where CTAs are more than run at once, the long
// ones start first, and the short ones fill the end of the launch.
__device__ __forceinline__ int row_by_length(unsigned char* smem, const RowsArgs& a, int rank) {
    int* own = (int*)smem;                                           // (the tiles' memory, before the first tile comes)
    __shared__ int found;
    for (int i = threadIdx.x; i < a.rows; i += AR_THREADS) {
        const int n = a.kv_len[i], from = max(a.skip ? a.skip[i] : 0, a.window > 0 ? n - a.window : 0);
        own[i] = n - max(0, from);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.rows; i += AR_THREADS) {
        const int mine = own[i];
        int before = 0;
        for (int j = 0; j < a.rows; ++j) before += own[j] > mine || (own[j] == mine && j < i);
        if (before == rank) found = i;
    }
    __syncthreads();
    return found;
}

// grid (kv_heads * ceil(group / 8), rows, splits), a cluster along z.
template <int D_PAD, bool KV8, bool FEW>
__global__ void __launch_bounds__(AR_THREADS, (Tile<D_PAD, KV8, FEW>::CTAS)) rows_kernel(const __grid_constant__ CUtensorMap map, const RowsArgs a) {
    extern __shared__ unsigned char smem_raw[];
    using T = Tile<D_PAD, KV8, FEW>;
    static_assert(T::SUMS + 4 * AR_HEADS * ((FEW ? AR_WARPS : AR_CLUSTER) + PU_MOST_PARTS) <= T::BODY, "the join's weights lie between the sums and `whole`");
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
    const bool cluster = !FEW && a.splits > 1;                      // (few keys: never cut, so no code for it)
    if (cluster) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");   // (this CTA runs: waited for before anybody writes here)
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
        for (int s = 0; s < T::STAGES; ++s) {
            mbar_init(base + T::BARS + 8 * s, 1);
            mbar_init(base + T::BARS + 8 * (T::STAGES + s), AR_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    const int group = a.heads / a.kv_heads, m_tiles = (group + AR_HEADS - 1) / AR_HEADS;
    const int hk = blockIdx.x / m_tiles, g0 = blockIdx.x % m_tiles * AR_HEADS, g = min(AR_HEADS, group - g0);
    const int split = FEW ? 0 : blockIdx.z, splits = FEW ? 1 : a.splits;
    const int b = a.by_length ? row_by_length(smem, a, blockIdx.y) : (int)blockIdx.y;
    const int n = a.kv_len[b], t = a.query_start[b], row_slot = a.row_slot[b];
    const int shared = a.skip ? a.skip[b] : 0;
    const int lo = max(shared, a.window > 0 ? max(0, n - a.window) : 0);          // the one query sits at position n - 1
    const int tile_lo = lo / T::KEYS, tile_hi = (n + T::KEYS - 1) / T::KEYS;
    const int per = max(0, tile_hi - tile_lo + splits - 1) / splits;
    const int first = tile_lo + split * per, last = min(tile_hi, first + per);
    if (a.by_length) fence_async_smem();                             // (what was written where the first tiles go)
    __syncthreads();
    if (threadIdx.x >= 32 * AR_WARPS)
        load_tiles<D_PAD, KV8, FEW>(&map, a, base, a.block_table + (size_t)row_slot * a.table_stride, hk, first, last, n);
    else
        walk<D_PAD, KV8, FEW>(smem, base, a, a.q + ((size_t)t * a.heads + hk * group + g0) * a.head_dim, g, first, last, lo, n);
    __syncthreads();
    // What the four warps left becomes one result a head, or, in a cluster, goes to the CTAs that combine it: each takes a share of
    // the numbers of all splits. The shared keys' partial results join the last step, and the sink.
    const float* wo = (const float*)smem;                           // [warp][8][D_PAD], then [warp][g][2]
    const float* wml = wo + AR_WARPS * AR_HEADS * D_PAD;
    float* weights = (float*)(smem + T::SUMS);                      // [g][pieces + parts]: room for PU_MOST_PARTS, which bounds the shared keys' units
    float* whole = (float*)(smem + T::BODY);                        // [8][2], over the scales, which are done
    float* recv_o = (float*)(smem + T::RECV);                       // [splits][share], then [splits][g][2]: what the others send
    const int total = g * a.head_dim, share = ((total + splits - 1) / splits + 3) & ~3;
    float* recv_ml = recv_o + splits * share;
    bf16* out = a.out + ((size_t)t * a.heads + hk * group + g0) * a.head_dim;
    int4 at = make_int4(0, 0, 0, 0);
    if (a.skip) asm volatile("griddepcontrol.wait;\n" ::: "memory");   // (this launch may have begun before the one that leaves them ended)
    if (shared > 0) {
        at = a.part_at[b];
        // Where a wait of that launch gave up, rows whose turn did not come have no entry, and what is there names anything.
        if (at.y < 1 || at.y > PU_MOST_PARTS || at.x < 0 || at.x > a.part_units - a.kv_heads * at.y || at.z < 0 || at.z > a.part_rows - group) {
            at = make_int4(0, 0, 0, 0);
            if (threadIdx.x == 0) tc_give_up(12);
        }
    }
    const size_t slot = (size_t)(at.x + hk * at.y) * a.part_rows + at.z + g0;
    const float* part_ml = shared > 0 ? a.part_ml + slot * 2 : nullptr;
    const float* part_o = shared > 0 ? a.part_o + slot * a.head_dim : nullptr;
    const size_t stride = (size_t)a.part_rows * a.head_dim;         // from one split's partial results to the next
    if (cluster) {
        weigh(weights, whole, wml, AR_WARPS, g, nullptr, 0, 0);
        __syncthreads();
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");   // every CTA of the cluster runs
        for (int i = threadIdx.x * 4; i < total; i += AR_THREADS * 4) {
            const int r = i / a.head_dim, d = i - r * a.head_dim, peer = i / share;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < AR_WARPS; ++w) add4(x, weights[r * AR_WARPS + w], *(const float4*)(wo + (w * AR_HEADS + r) * D_PAD + d));
            st_cluster_f32x4(recv_o + split * share + (i - peer * share), peer, x);
        }
        for (int i = threadIdx.x; i < splits * g; i += AR_THREADS) {
            const int peer = i / g, r = i - peer * g;
            st_cluster_f32(recv_ml + (split * g + r) * 2, peer, whole[2 * r]);
            st_cluster_f32(recv_ml + (split * g + r) * 2 + 1, peer, whole[2 * r + 1]);
        }
        __syncwarp();
        cluster_barrier();                                          // everything sent has arrived; nobody reads another's memory after it
    }
    const int pieces = cluster ? splits : AR_WARPS, count = pieces + at.y;
    const int from = cluster ? split * share : 0, upto = cluster ? min(total, from + share) : total;
    constexpr int AHEAD = FEW ? 8 : 16;
    float4 ahead[AHEAD];                                         // of a thread's first numbers, asked for before the weights are known
    {
        const int i = from + threadIdx.x * 4;
#pragma unroll
        for (int p = 0; p < AHEAD; ++p)
            ahead[p] = i < upto && p < at.y ? *(const float4*)(part_o + p * stride + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    weigh(weights, whole, cluster ? recv_ml : wml, pieces, g, part_ml, (size_t)a.part_rows * 2, at.y);
    __syncthreads();
    for (int i = from + threadIdx.x * 4; i < upto; i += AR_THREADS * 4) {
        const int r = i / a.head_dim, d = i - r * a.head_dim;
        const float* w = weights + r * count;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < pieces; ++p)
            add4(x, w[p], *(const float4*)(cluster ? recv_o + p * share + (i - from) : wo + (p * AR_HEADS + r) * D_PAD + d));
        int p0 = 0;
        if (i == from + (int)threadIdx.x * 4) {
#pragma unroll
            for (int p = 0; p < AHEAD; ++p) if (p < at.y) add4(x, w[pieces + p], ahead[p]);
            p0 = AHEAD;
        }
#pragma unroll 8
        for (int p = p0; p < at.y; ++p) add4(x, w[pieces + p], *(const float4*)(part_o + p * stride + i));
        float l = whole[2 * r + 1];
        if (a.sinks && l > 0.f) l += ex2(fmaf(a.sinks[hk * group + g0 + r], 1.4426950408889634f, -whole[2 * r]));   // the sink: a weight without a value
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;        // (a sum that is no number gives none)
        const uint2 v = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        *(uint2*)(out + i) = l > 0.f || l != l ? v : make_uint2(0u, 0u);
    }
}

template <int D_PAD, bool KV8, bool FEW> static size_t rows_smem(int splits, int group, int head_dim) {
    const int g = group < AR_HEADS ? group : AR_HEADS;
    const size_t recv = splits > 1 ? (size_t)(g * head_dim + 4 * splits + splits * g * 2) * 4 : 0;  // (a share is rounded up)
    return Tile<D_PAD, KV8, FEW>::RECV + recv + 1024;                    // (and the way to a boundary of 1,024 bytes)
}

template <int D_PAD, bool KV8, bool FEW>
static int launch_rows(RowsArgs* a, int rows, int splits, int group, int head_dim, int* capacity, cudaStream_t s) {
    using T = Tile<D_PAD, KV8, FEW>;
    auto kernel = rows_kernel<D_PAD, KV8, FEW>;
    const size_t smem = rows_smem<D_PAD, KV8, FEW>(splits, group, head_dim);
    static unsigned long long prepared = 0;                         // devices that the kernel's limits are set on
    int device = 0;
    HB_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !(prepared >> device & 1)) {
        HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem<D_PAD, KV8, FEW>(AR_CLUSTER, AR_HEADS, D_PAD)));
        HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (device < 64) prepared |= 1ull << device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = capacity ? dim3(1, 1, splits) : dim3(a->kv_heads * ((group + AR_HEADS - 1) / AR_HEADS), rows, splits);
    cfg.blockDim = dim3(AR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2] = {};
    cfg.attrs = attrs;
    if (splits > 1) {
        attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attrs[cfg.numAttrs].val.clusterDim.x = attrs[cfg.numAttrs].val.clusterDim.y = 1;
        attrs[cfg.numAttrs++].val.clusterDim.z = splits;
    }
    if (!capacity && a->skip) {                                     // behind attention_prefix, whose CTAs say when they have all begun
        attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (capacity) {
        if (splits > 1) HB_CUDA(cudaOccupancyMaxActiveClusters(capacity, kernel, &cfg));
        else HB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(capacity, kernel, AR_THREADS, smem));
        return 0;
    }
    a->box = a->page_size % 64 == 0 ? 64 : a->page_size % 32 == 0 ? 32 : 16;
    const uint64_t bytes = KV8 ? 1 : 2;
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)a->page_size, (cuuint64_t)a->pages * 2 * a->kv_heads};
    const cuuint64_t strides[2] = {head_dim * bytes, a->page_size * (uint64_t)(head_dim + (KV8 ? 1 : 0)) * bytes};
    const cuuint32_t box[3] = {(cuuint32_t)(T::SUB / bytes), (cuuint32_t)a->box, 1}, elem[3] = {1, 1, 1};
    const CUresult r = cuTensorMapEncodeTiled(&map, KV8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                                              const_cast<unsigned char*>(a->kv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                              T::SUB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) HB_REFUSE("attention_rows: cuTensorMapEncodeTiled failed with %d", (int)r);
    HB_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const CUtensorMap)map, (const RowsArgs)*a));
    return 0;
}
template <bool KV8, bool FEW> static int any_rows(RowsArgs* a, int rows, int splits, int group, int head_dim, int* capacity, cudaStream_t s) {
    if (head_dim <= 64) return launch_rows<64, KV8, FEW>(a, rows, splits, group, head_dim, capacity, s);
    if (head_dim <= 128) return launch_rows<128, KV8, FEW>(a, rows, splits, group, head_dim, capacity, s);
    return launch_rows<256, KV8, FEW>(a, rows, splits, group, head_dim, capacity, s);
}

HB_DEFINE_STATUS_MIRROR(hb_attention_rows_status_mirror)
extern "C" int hb_attention_rows_status(unsigned int* status) {
    HB_CUDA(cudaDeviceSynchronize());
    HB_CUDA(cudaMemcpyFromSymbol(status, g_tc_status, sizeof(unsigned int)));
    const unsigned int zero = 0;
    HB_CUDA(cudaMemcpyToSymbol(g_tc_status, &zero, sizeof(unsigned int)));
    return 0;
}

static int forms(int kv8, int few, RowsArgs* a, int rows, int splits, int group, int head_dim, int* capacity, cudaStream_t s) {
    if (kv8) return few ? any_rows<true, true>(a, rows, splits, group, head_dim, capacity, s) : any_rows<true, false>(a, rows, splits, group, head_dim, capacity, s);
    return few ? any_rows<false, true>(a, rows, splits, group, head_dim, capacity, s) : any_rows<false, false>(a, rows, splits, group, head_dim, capacity, s);
}

// Clusters of `splits` CTAs that run at once (splits 1: CTAs an SM); -1 where the sizes are refused.
extern "C" int hb_attention_rows_capacity(int kv8, int few, int head_dim, int group, int splits) {
    int n = 0;
    if (head_dim < 16 || head_dim > 256 || head_dim % 16 || group < 1 || splits < 1 || splits > AR_CLUSTER) return -1;
    if (forms(kv8, few, nullptr, 1, splits, group, head_dim, &n, 0) != 0) {
        (void)cudaGetLastError();
        return 0;
    }
    return n;
}

extern "C" int hb_attention_rows(void* out, const void* q, const void* kv, int kv8, const int32_t* block_table, int table_stride,
                                 const int32_t* row_slot, const int32_t* query_start, const int32_t* kv_len, int rows, int heads, int kv_heads,
                                 int head_dim, int pages, int page_size, float scale, int window, int splits, int few, int by_length, const float* sinks,
                                 const int32_t* skip, const float* part_o, const float* part_ml, const int32_t* part_at, int part_rows, int part_units,
                                 hb_stream stream) {
    if (rows == 0) return 0;
    if (head_dim % 16 || head_dim > 256 || head_dim < 16) HB_REFUSE("attention_rows: head_dim %d is no multiple of 16 up to 256", head_dim);
    if (kv_heads < 1 || heads < 1 || heads % kv_heads) HB_REFUSE("attention_rows: %d heads, %d kv heads", heads, kv_heads);
    if (page_size < 16 || page_size % 16) HB_REFUSE("attention_rows: page size %d is no multiple of 16", page_size);
    if (splits < 1 || splits > AR_CLUSTER) HB_REFUSE("attention_rows: %d splits (1 to 16, a cluster's size)", splits);
    if (few && splits > 1) HB_REFUSE("attention_rows: the form for few keys does not cut them (%d splits)", splits);
    if (!(scale > 0.f)) HB_REFUSE("attention_rows: the score scale must be positive");
    const int group = heads / kv_heads;
    if (rows > 65535) HB_REFUSE("attention_rows: %d rows", rows);
    if (pages < 1 || (long)pages * 2 * kv_heads > 0x7ffffffel) HB_REFUSE("attention_rows: %d pages of %d kv heads", pages, kv_heads);
    if (((uintptr_t)kv % 16) || (((uintptr_t)q | (uintptr_t)out) % 8)) HB_REFUSE("attention_rows: the cache must start on 16 bytes, q and out on 8");
    if (skip && (!part_o || !part_ml || !part_at || part_rows < group || part_units < 1 || window > 0)) HB_REFUSE("attention_rows: shared keys need their partial results, and no window");
    RowsArgs a = {(bf16*)out, (const bf16*)q, (const unsigned char*)kv, block_table, row_slot, query_start, kv_len, sinks, skip, part_o,
                  part_ml, (const int4*)part_at, part_rows, part_units, table_stride, rows, heads, kv_heads, head_dim, pages, page_size,
                  log2_exact(page_size), 0, window, splits, by_length && rows <= AR_BY_LENGTH, scale * 1.4426950408889634f};
    return forms(kv8, few, &a, rows, splits, group, head_dim, nullptr, (cudaStream_t)stream);
}
