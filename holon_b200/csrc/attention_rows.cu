// Attention of rows that bring one token each, over pages of 8-bit codes, and over the keys that rows which share their
// first pages hold behind those (pages of either kind). mma.sync m16n8k16, 32-bit accumulation and softmax.
//
// A CTA owns (row, kv head, split of the row's keys); the kv head's group of query heads is the 16-row M tile, so keys and
// values are read once per group. Its four warps take 16 keys each of every 64-key tile, keep their own running softmax and
// are merged in shared memory; the splits of a (row, kv head) are one thread-block cluster and are merged through
// distributed shared memory, in the order of the splits. With `skip` (tokens a row shares with others) the walk starts
// behind them, and the partial results that attention_prefix.cu left for the shared keys are added in the same merge.
//
// 8-bit pages: codes go to the matrix instructions as halves, which hold every code exactly. With k_j = 2^a_j K_j and
// v_j = 2^b_j V_j (K, V codes) and the head's query scaled into the halves' range by a power of two 2^-c,
//     u_j = (q 2^-c · K_j) 2^(a_j + c) scale log2(e) + b_j,   w_j = 2^(u_j - M),   O = sum w_j V_j,   l = sum w_j 2^-b_j
// with M the running maximum of u, not of the scores: the weights that meet the codes stay at most 2^14 whatever the values' scales
// are (14 is taken off M so that small weights are no subnormal halves), and l sums the softmax's own weights in the same units.
// ldmatrix moves pairs of codes as it moves bfloat16: a lane gets codes 4 c .. 4 c + 3 of a key where the fragment wants
// columns 2 c, 2 c + 1, 2 c + 8, 2 c + 9, so queries are laid out in that order; of values it gets two neighbouring codes of two keys,
// one byte permutation pairs the keys, and the even and the odd columns are two products.
#include <cuda_fp16.h>

#include "attention_mma.cuh"
#include "cache8.cuh"

#define AR_THREADS 128
#define AR_BIAS 14.f

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

struct RowsArgs {
    bf16* out;                     // [tokens, heads, head_dim]
    const bf16* q;
    const unsigned char* kv;
    const int32_t *block_table, *row_slot, *query_start, *kv_len;
    const float* sinks;
    const int32_t* skip;           // tokens a row shares (their partial results are in part_*), or null
    const float *part_o, *part_ml; // [units, part_rows, head_dim] and [units, part_rows, 2]
    const int4* part_at;           // per row: the first unit of kv head 0, units a kv head, the row's place among its tile's rows
    int part_rows, table_stride, heads, kv_heads, head_dim, pages, page_size, window, splits;
    float scale_log2;
};

// Byte offset of (row, 16-byte chunk) in a tile whose rows are ROW bytes: eight rows at one chunk lie in eight bank groups.
template <int ROW> __device__ __forceinline__ uint32_t row_off(int row, int chunk) {
    return (uint32_t)(row * ROW + ((ROW == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7)) << 4));
}
// Bytes of a tile's row: bfloat16 heads padded to 64, 128 or 256, codes to 64, 128 or 256.
template <int D_PAD, bool KV8> struct Tile {
    static constexpr int ROW = KV8 ? D_PAD : 2 * D_PAD;
    static constexpr int PART = TILE_N * ROW;                    // keys or values
    static constexpr int STAGE = 2 * PART + (KV8 ? 128 : 0);     // and 64 + 64 scale bytes
    static constexpr int Q = D_PAD > 128 ? D_PAD / 16 * 512 : 0; // fragments of the queries, where they do not stay in registers
    static constexpr int SUMS = (4 * 16 * D_PAD + 4 * 16 * 2 + 16 * D_PAD + 16 * 2) * 4;
    static constexpr int BYTES(int stages) { return Q + (stages * STAGE > SUMS ? stages * STAGE : SUMS); }
};

// Keys and values [tile * 64, tile * 64 + 64) of a kv head; keys outside [lo, hi) become zeros. `page`: the tile's page where
// a tile lies in one (page_size a multiple of 64), else every row looks its own up.
template <int D_PAD, bool KV8>
__device__ __forceinline__ void load_tile(uint32_t dst, const RowsArgs& a, const int32_t* table, int hk, int tile, int lo, int hi, bool in_page,
                                          int page) {
    using T = Tile<D_PAD, KV8>;
    constexpr int CPR = T::ROW / 16, STEP = AR_THREADS / CPR;
    const int bytes = KV8 ? a.head_dim : 2 * a.head_dim;            // of a row in memory
    const size_t block = (size_t)a.page_size * (KV8 ? a.head_dim + 1 : 2 * a.head_dim), part = (size_t)a.kv_heads * block;
    const int ch = threadIdx.x % CPR, r0 = threadIdx.x / CPR, j0 = tile * TILE_N;
    if (KV8 && threadIdx.x < 8) {                                   // the scales: 16 keys a thread (pages are multiples of 16 keys)
        const int j = j0 + (threadIdx.x & 3) * 16, v = threadIdx.x >> 2;
        bool valid = j + 16 > lo && j < hi;
        const int pi = j / a.page_size;
        const int p = !valid ? 0 : in_page ? page : table[pi];
        valid = valid && p >= 0 && p < a.pages;
        const size_t off = ((size_t)(valid ? p : 0) * 2 + v) * part + (size_t)hk * block + (size_t)a.page_size * a.head_dim + (valid ? j - pi * a.page_size : 0);
        cp_async16(dst + 2 * T::PART + v * 64 + (threadIdx.x & 3) * 16, a.kv + off, valid);
    }
    if (ch * 16 >= bytes) return;                                   // columns past head_dim are never read
    if (in_page) {
        const bool page_ok = page >= 0 && page < a.pages;
        const unsigned char* base = a.kv + (size_t)(page_ok ? page : 0) * 2 * part + (size_t)hk * block + ch * 16
                                    + (size_t)(j0 % a.page_size) * bytes;
#pragma unroll
        for (int r = r0; r < TILE_N; r += STEP) {
            const bool valid = page_ok && j0 + r >= lo && j0 + r < hi;
            const unsigned char* src = base + (valid ? (size_t)r * bytes : 0);
            const uint32_t d = dst + row_off<T::ROW>(r, ch);
            cp_async16(d, src, valid);
            cp_async16(d + T::PART, src + part, valid);
        }
        return;
    }
#pragma unroll
    for (int r = r0; r < TILE_N; r += STEP) {
        const int j = j0 + r;
        bool valid = j >= lo && j < hi;
        size_t off = 0;
        if (valid) {
            const int pi = j / a.page_size, p = table[pi];
            valid = p >= 0 && p < a.pages;
            off = (size_t)(valid ? p : 0) * 2 * part + (size_t)hk * block + (size_t)(j - pi * a.page_size) * bytes + ch * 16;
        }
        const uint32_t d = dst + row_off<T::ROW>(r, ch);
        cp_async16(d, a.kv + off, valid);
        cp_async16(d + T::PART, a.kv + off + part, valid);
    }
}

// The A fragments of up to 16 heads' queries at `q` (head_dim apart); for codes as halves, each head divided by a power of two
// that brings its largest number near 2^6, which `up0` and `up1` (lane/4, lane/4 + 8) undo.
template <int D_PAD, bool KV8>
__device__ __forceinline__ void load_q(uint32_t (&qf)[D_PAD > 128 ? 1 : D_PAD / 16][4], uint32_t q_s, const bf16* q, int g, int head_dim,
                                       float& up0, float& up1) {
    const int lane = threadIdx.x & 31, r0 = lane >> 2, c = lane & 3;
    float down[2] = {1.f, 1.f};
    up0 = up1 = 1.f;
    if (KV8) {
        float m[2] = {0.f, 0.f};
        for (int ks = 0; ks < head_dim >> 4; ++ks)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (r0 + 8 * h < g) {
                    const uint2 w = *(const uint2*)(q + (size_t)(r0 + 8 * h) * head_dim + ks * 16 + 4 * c);
                    const float2 x = __bfloat1622float2(*(const __nv_bfloat162*)&w.x), y = __bfloat1622float2(*(const __nv_bfloat162*)&w.y);
                    m[h] = fmaxf(fmaxf(m[h], fmaxf(c8_magnitude(x.x), c8_magnitude(x.y))), fmaxf(c8_magnitude(y.x), c8_magnitude(y.y)));
                }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 1));
            m[h] = fmaxf(m[h], __shfl_xor_sync(0xffffffffu, m[h], 2));
            const int e = min(max((int)(__float_as_uint(m[h]) >> 23) - 127 - 6, -100), 121);
            down[h] = c8_power(-e);
            (h ? up1 : up0) = c8_power(e);
        }
    }
    auto pair = [&](int r, int d, float f) -> uint32_t {             // numbers d, d + 1 of head r
        if (r >= g) return 0u;
        const uint32_t w = *(const uint32_t*)(q + (size_t)r * head_dim + d);
        if (!KV8) return w;
        const float2 x = __bfloat1622float2(*(const __nv_bfloat162*)&w);
        return pack_f16(x.x * f, x.y * f);
    };
    constexpr bool IN_REGS = D_PAD <= 128;
#pragma unroll
    for (int ks = 0; ks < D_PAD / 16; ++ks) {
        if (ks * 16 >= head_dim) break;
        const int lo = ks * 16 + (KV8 ? 4 * c : 2 * c), hi = lo + (KV8 ? 2 : 8);
        const uint32_t f[4] = {pair(r0, lo, down[0]), pair(r0 + 8, lo, down[1]), pair(r0, hi, down[0]), pair(r0 + 8, hi, down[1])};
        if (IN_REGS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[IN_REGS ? ks : 0][i] = f[i];
        } else if (threadIdx.x < 32) {                               // (every warp makes the same ones: the first stores them)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(q_s + (ks * 32 + lane) * 16), "r"(f[0]), "r"(f[1]), "r"(f[2]), "r"(f[3]) : "memory");
        }
    }
}

// One walk of the four warps over tiles [first, last) of (row, kv head); leaves each warp's sums in shared memory:
// [warp][16][D_PAD] floats and [warp][16][2] (maximum in log2 units, sum) at `smem` + Q.
template <int D_PAD, int STAGES, bool KV8>
__device__ __forceinline__ void walk(unsigned char* smem, const RowsArgs& a, const int32_t* table, const bf16* q, int hk, int g, int first, int last,
                                     int lo, int n) {
    using T = Tile<D_PAD, KV8>;
    const uint32_t q_s = smem_u32(smem), kv_s = q_s + T::Q;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool in_page = a.page_size % TILE_N == 0;
    const int per_page = in_page ? a.page_size / TILE_N : 1;
    auto page_of = [&](int tile) { return in_page && tile < last ? table[tile / per_page] : 0; };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        if (first + s < last) load_tile<D_PAD, KV8>(kv_s + s * T::STAGE, a, table, hk, first + s, lo, n, in_page, page_of(first + s));
        cp_async_commit();
    }
    int page_ahead = page_of(first + STAGES - 1);
    constexpr bool Q_IN_REGS = D_PAD <= 128;
    uint32_t qf[Q_IN_REGS ? D_PAD / 16 : 1][4];
    float up0, up1;
    load_q<D_PAD, KV8>(qf, q_s, q, g, a.head_dim, up0, up1);
    up0 *= a.scale_log2; up1 *= a.scale_log2;

    float o[D_PAD / 8][4];
#pragma unroll
    for (int i = 0; i < D_PAD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;      // rows lane/4 and lane/4 + 8
    const int ksteps = a.head_dim >> 4;
    // ldmatrix addresses. Keys: matrices (keys 0-7, chunk), (keys 8-15, chunk), (keys 0-7, next), (keys 8-15, next) for codes;
    // for bfloat16 (keys 0-7, chunk), (keys 0-7, next), (keys 8-15, chunk), (keys 8-15, next). Values, transposed: as codes' keys.
    const int key_row = warp * 16 + (lane & 7) + (KV8 ? (lane & 8) : (lane & 16) >> 1), key_ch = KV8 ? lane >> 4 : (lane >> 3) & 1;
    const int val_row = warp * 16 + (lane & 7) + (lane & 8), val_ch = lane >> 4;

    for (int tile = first; tile < last; ++tile) {
        const int stage = (tile - first) % STAGES;
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        if (tile + STAGES - 1 < last)
            load_tile<D_PAD, KV8>(kv_s + ((tile - first + STAGES - 1) % STAGES) * T::STAGE, a, table, hk, tile + STAGES - 1, lo, n, in_page, page_ahead);
        cp_async_commit();
        page_ahead = page_of(tile + STAGES);
        const int key0 = tile * TILE_N + warp * 16;                 // this warp's 16 keys
        if (key0 >= n || key0 + 16 <= lo) continue;                 // (uniform per warp; the barrier is above)
        const uint32_t kt = kv_s + stage * T::STAGE, vt = kt + T::PART;
        float s[2][4] = {};
        if constexpr (KV8) {
#pragma unroll
            for (int p = 0; p < D_PAD / 32; ++p) {                  // 32 numbers of the head
                if (2 * p < ksteps) {
                    uint32_t x[4];
                    ldmatrix_x4(x, kt + row_off<T::ROW>(key_row, 2 * p + key_ch));   // (past head_dim: whatever lies there, not used)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int ks = 2 * p + h;
                        if (ks < ksteps) {
                            uint32_t f[4];
                            if (!Q_IN_REGS) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(q_s + (ks * 32 + lane) * 16));
                            mma_f16(s[0], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : f, c8_halves(x[2 * h]), c8_halves(x[2 * h] >> 16));
                            mma_f16(s[1], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : f, c8_halves(x[2 * h + 1]), c8_halves(x[2 * h + 1] >> 16));
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < D_PAD / 16; ++ks) {
                if (ks < ksteps) {
                    uint32_t x[4], f[4];
                    if (!Q_IN_REGS) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(q_s + (ks * 32 + lane) * 16));
                    ldmatrix_x4(x, kt + row_off<T::ROW>(key_row, 2 * ks + key_ch));
                    mma_bf16(s[0], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : f, x[0], x[1]);
                    mma_bf16(s[1], Q_IN_REGS ? qf[Q_IN_REGS ? ks : 0] : f, x[2], x[3]);
                }
            }
        }
        float drop[2][2] = {{1.f, 1.f}, {1.f, 1.f}};                // 2^-b of this lane's keys
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            float ka[2] = {1.f, 1.f}, vb[2] = {0.f, 0.f};
            if (KV8) {                                              // (a byte below any that is written: a page that is not there, codes of 0)
                uint16_t kw, vw;
                const uint32_t at = vt + T::PART + warp * 16 + nt * 8 + (lane & 3) * 2;
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(kw) : "r"(at));
                asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(vw) : "r"(at + 64));
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t kb = e ? kw >> 8 : kw & 255, b = min(max(e ? vw >> 8 : vw & 255, C8_LOW + 127), 254);
                    ka[e] = __uint_as_float(kb << 23);
                    vb[e] = (float)((int)b - 127);
                    drop[nt][e] = __uint_as_float((254u - b) << 23);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = key0 + nt * 8 + (lane & 3) * 2 + (e & 1);
                const float u = fmaf(s[nt][e], ka[e & 1] * (e < 2 ? up0 : up1), vb[e & 1]);
                s[nt][e] = j >= lo && j < n ? u : -INFINITY;
            }
            mx0 = fmaxf(mx0, fmaxf(s[nt][0], s[nt][1]));
            mx1 = fmaxf(mx1, fmaxf(s[nt][2], s[nt][3]));
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float n0 = fmaxf(m0, mx0 - (KV8 ? AR_BIAS : 0.f)), n1 = fmaxf(m1, mx1 - (KV8 ? AR_BIAS : 0.f));
        const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;      // a row with nothing yet: 2^(-inf) = 0 below
        const float c0 = ex2(m0 - b0), c1 = ex2(m1 - b1);
        m0 = n0; m1 = n1;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = ex2(s[nt][e] - (e < 2 ? b0 : b1));
            sum0 += s[nt][0] * drop[nt][0] + s[nt][1] * drop[nt][1];
            sum1 += s[nt][2] * drop[nt][0] + s[nt][3] * drop[nt][1];
        }
        l0 = l0 * c0 + sum0; l1 = l1 * c1 + sum1;                   // per-lane partial sums; quads are joined at the end
        if (__any_sync(0xffffffffu, c0 != 1.f || c1 != 1.f)) {      // the running maximum moved: rescale what is summed
#pragma unroll
            for (int i = 0; i < D_PAD / 8; ++i) { o[i][0] *= c0; o[i][1] *= c0; o[i][2] *= c1; o[i][3] *= c1; }
        }
        uint32_t p[4];
        if constexpr (KV8) {
            p[0] = pack_f16(s[0][0], s[0][1]); p[1] = pack_f16(s[0][2], s[0][3]);
            p[2] = pack_f16(s[1][0], s[1][1]); p[3] = pack_f16(s[1][2], s[1][3]);
#pragma unroll
            for (int d = 0; d < D_PAD / 32; ++d) {                  // 32 columns: chunks 2 d and 2 d + 1
                if (2 * d < ksteps) {
                    uint32_t x[4];
                    ldmatrix_x4_trans(x, vt + row_off<T::ROW>(val_row, 2 * d + val_ch));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (2 * d + h < ksteps) {
                            const uint32_t y0 = __byte_perm(x[2 * h], 0, 0x3120), y1 = __byte_perm(x[2 * h + 1], 0, 0x3120);
                            mma_f16(o[4 * d + 2 * h], p, c8_halves(y0), c8_halves(y1));                    // even columns of the chunk
                            mma_f16(o[4 * d + 2 * h + 1], p, c8_halves(y0 >> 16), c8_halves(y1 >> 16));    // odd ones
                        }
                    }
                }
            }
        } else {
            p[0] = pack_bf16(s[0][0], s[0][1]); p[1] = pack_bf16(s[0][2], s[0][3]);
            p[2] = pack_bf16(s[1][0], s[1][1]); p[3] = pack_bf16(s[1][2], s[1][3]);
#pragma unroll
            for (int d = 0; d < D_PAD / 16; ++d) {
                if (d < ksteps) {
                    uint32_t x[4];
                    ldmatrix_x4_trans(x, vt + row_off<T::ROW>(val_row, 2 * d + val_ch));
                    mma_bf16(o[2 * d], p, x[0], x[1]);
                    mma_bf16(o[2 * d + 1], p, x[2], x[3]);
                }
            }
        }
    }
    cp_async_wait<0>();
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    __syncthreads();                                                // every warp is done with the tiles: reuse them
    float* wo = (float*)(smem + T::Q);
    float* wml = wo + 4 * 16 * D_PAD;
    const int r0 = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < D_PAD / 8; i += 2) {
        if (i * 8 < a.head_dim) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (r0 + 8 * h >= g) continue;
                float* row = wo + (warp * 16 + r0 + 8 * h) * D_PAD + i * 8;
                if (KV8) {
                    *(float4*)(row + 4 * c) = make_float4(o[i][2 * h], o[i + 1][2 * h], o[i][2 * h + 1], o[i + 1][2 * h + 1]);
                } else {
                    *(float2*)(row + 2 * c) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
                    *(float2*)(row + 8 + 2 * c) = make_float2(o[i + 1][2 * h], o[i + 1][2 * h + 1]);
                }
            }
        }
    }
    if (c == 0) {
        wml[(warp * 16 + r0) * 2] = m0; wml[(warp * 16 + r0) * 2 + 1] = l0;
        wml[(warp * 16 + r0 + 8) * 2] = m1; wml[(warp * 16 + r0 + 8) * 2 + 1] = l1;
    }
    __syncthreads();
}

// A running merge of partial results (maximum in log2 units, sum, weighted sum of one column), in the order of the calls.
struct Merge {
    float m = -INFINITY, l = 0.f, o = 0.f;
    __device__ __forceinline__ void add(float mi, float li, float oi) {
        if (mi == -INFINITY && li == 0.f) return;                   // (nothing seen; a sum that is no number stays one)
        const float top = fmaxf(m, mi), f = m == top ? 1.f : ex2(m - top), w = mi == top ? 1.f : ex2(mi - top);
        m = top; l = l * f + li * w; o = o * f + oi * w;
    }
};

// The result of one column of head `h`: what the splits left, the shared keys' partial results, the sink.
__device__ __forceinline__ float finished(Merge x, const RowsArgs& a, int b, int h, int hk, int in_group, int d, bool shares) {
    if (shares) {
        const int4 at = a.part_at[b];
        const int group = a.heads / a.kv_heads;
        for (int s = 0; s < at.y; ++s) {
            const size_t slot = (size_t)(at.x + hk * at.y + s) * a.part_rows + at.z * group + in_group;
            x.add(a.part_ml[slot * 2], a.part_ml[slot * 2 + 1], a.part_o[slot * a.head_dim + d]);
        }
    }
    if (a.sinks && x.l > 0.f) x.l += ex2(fmaf(a.sinks[h], 1.4426950408889634f, -x.m));   // the sink: a weight without a value
    return x.l > 0.f || x.l != x.l ? x.o / x.l : 0.f;               // (a sum that is no number gives none)
}

// grid (rows, kv_heads * m_tiles, splits), a cluster along z, 128 threads. m_tiles = ceil(group / 16).
template <int D_PAD, int STAGES, bool KV8>
__global__ void __launch_bounds__(AR_THREADS) rows_kernel(const RowsArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    using T = Tile<D_PAD, KV8>;
    const bool cluster = a.splits > 1;
    if (cluster) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");   // (this CTA runs: waited for before anybody writes here)
    const int b = blockIdx.x, split = blockIdx.z, splits = a.splits;
    const int group = a.heads / a.kv_heads, m_tiles = (group + 15) / 16;
    const int hk = blockIdx.y / m_tiles, g0 = blockIdx.y % m_tiles * 16, g = min(16, group - g0);
    const int n = a.kv_len[b], t = a.query_start[b];
    const int shared = a.skip ? a.skip[b] : 0;
    const int lo = max(shared, a.window > 0 ? max(0, n - a.window) : 0);          // the one query sits at position n - 1
    const int tile_lo = lo / TILE_N, tile_hi = (n + TILE_N - 1) / TILE_N;
    const int per = max(0, tile_hi - tile_lo + splits - 1) / splits;
    const int first = tile_lo + split * per, last = min(tile_hi, first + per);
    walk<D_PAD, STAGES, KV8>(smem, a, a.block_table + (size_t)a.row_slot[b] * a.table_stride,
                             a.q + ((size_t)t * a.heads + hk * group + g0) * a.head_dim, hk, g, first, last, lo, n);
    const float* wo = (const float*)(smem + T::Q);
    const float* wml = wo + 4 * 16 * D_PAD;
    const int total = g * a.head_dim, share = (total + splits - 1) / splits;
    bf16* out = a.out + ((size_t)t * a.heads + hk * group + g0) * a.head_dim;
    float* recv_o = (float*)(smem + T::BYTES(STAGES));              // [splits][share], then [splits][g][2]: what the others send
    float* recv_ml = recv_o + splits * share;
    if (cluster) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");   // every CTA of the cluster runs
    }
    for (int i = threadIdx.x; i < total; i += AR_THREADS) {
        const int r = i / a.head_dim, d = i - r * a.head_dim;
        Merge x;
#pragma unroll
        for (int w = 0; w < 4; ++w) x.add(wml[(w * 16 + r) * 2], wml[(w * 16 + r) * 2 + 1], wo[(w * 16 + r) * D_PAD + d]);
        if (!cluster) {
            out[i] = __float2bfloat16_rn(finished(x, a, b, hk * group + g0 + r, hk, g0 + r, d, shared > 0));
            continue;
        }
        const int peer = i / share;                                 // the CTA that combines this number
        st_cluster_f32(recv_o + split * share + (i - peer * share), peer, x.o);
        if (d == 0)
            for (int q = 0; q < splits; ++q) {
                st_cluster_f32(recv_ml + (split * g + r) * 2, q, x.m);
                st_cluster_f32(recv_ml + (split * g + r) * 2 + 1, q, x.l);
            }
    }
    if (!cluster) return;
    __syncwarp();
    cluster_barrier();                                              // everything sent has arrived; nobody reads another's memory after it
    for (int i = threadIdx.x; i < share; i += AR_THREADS) {
        const int e = split * share + i;
        if (e >= total) break;
        const int r = e / a.head_dim, d = e - r * a.head_dim;
        Merge x;
        for (int q = 0; q < splits; ++q) x.add(recv_ml[(q * g + r) * 2], recv_ml[(q * g + r) * 2 + 1], recv_o[q * share + i]);
        out[e] = __float2bfloat16_rn(finished(x, a, b, hk * group + g0 + r, hk, g0 + r, d, shared > 0));
    }
}

template <int D_PAD, int STAGES, bool KV8> static size_t rows_smem(int splits, int group, int head_dim) {
    const int g = group < 16 ? group : 16;
    const size_t recv = splits > 1 ? (size_t)(g * head_dim + splits + splits * g * 2) * 4 : 0;      // (a share is rounded up)
    return Tile<D_PAD, KV8>::BYTES(STAGES) + recv;
}

template <int D_PAD, int STAGES, bool KV8>
static int launch_rows(const RowsArgs* a, int rows, int splits, int group, int head_dim, int* capacity, cudaStream_t s) {
    auto kernel = rows_kernel<D_PAD, STAGES, KV8>;
    const size_t smem = rows_smem<D_PAD, STAGES, KV8>(splits, group, head_dim);
    HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem<D_PAD, STAGES, KV8>(16, 16, D_PAD)));
    if (splits > 8) HB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = capacity ? dim3(1, 1, splits) : dim3(rows, a->kv_heads * ((group + 15) / 16), splits);
    cfg.blockDim = dim3(AR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = splits;
    cfg.attrs = &attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    if (capacity) {
        if (splits > 1) HB_CUDA(cudaOccupancyMaxActiveClusters(capacity, kernel, &cfg));
        else HB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(capacity, kernel, AR_THREADS, smem));
        return 0;
    }
    HB_CUDA(cudaLaunchKernelEx(&cfg, kernel, *a));
    return 0;
}
template <bool KV8> static int any_rows(const RowsArgs* a, int rows, int splits, int group, int head_dim, int* capacity, cudaStream_t s) {
    if (head_dim <= 64) return launch_rows<64, 4, KV8>(a, rows, splits, group, head_dim, capacity, s);
    if (head_dim <= 128) return launch_rows<128, KV8 ? 4 : 2, KV8>(a, rows, splits, group, head_dim, capacity, s);
    return launch_rows<256, KV8 ? 3 : 2, KV8>(a, rows, splits, group, head_dim, capacity, s);
}

// Clusters of `splits` CTAs that run at once (splits 1: CTAs an SM); -1 where the sizes are refused.
extern "C" int hb_attention_rows_capacity(int kv8, int head_dim, int group, int splits) {
    int n = 0;
    if (head_dim < 16 || head_dim > 256 || head_dim % 16 || group < 1 || splits < 1 || splits > 16) return -1;
    if ((kv8 ? any_rows<true>(nullptr, 1, splits, group, head_dim, &n, 0) : any_rows<false>(nullptr, 1, splits, group, head_dim, &n, 0)) != 0) {
        (void)cudaGetLastError();
        return 0;
    }
    return n;
}

extern "C" int hb_attention_rows(void* out, const void* q, const void* kv, int kv8, const int32_t* block_table, int table_stride,
                                 const int32_t* row_slot, const int32_t* query_start, const int32_t* kv_len, int rows, int heads, int kv_heads,
                                 int head_dim, int pages, int page_size, float scale, int window, int splits, const float* sinks,
                                 const int32_t* skip, const float* part_o, const float* part_ml, const int32_t* part_at, int part_rows,
                                 hb_stream stream) {
    if (rows == 0) return 0;
    if (head_dim % 16 || head_dim > 256 || head_dim < 16) HB_REFUSE("attention_rows: head_dim %d is no multiple of 16 up to 256", head_dim);
    if (kv_heads < 1 || heads < 1 || heads % kv_heads) HB_REFUSE("attention_rows: %d heads, %d kv heads", heads, kv_heads);
    if (page_size < 1 || (kv8 && page_size % 16)) HB_REFUSE("attention_rows: page size %d is no multiple of 16", page_size);
    if (splits < 1 || splits > 16) HB_REFUSE("attention_rows: %d splits (1 to 16, a cluster's size)", splits);
    if (!(scale > 0.f)) HB_REFUSE("attention_rows: the score scale must be positive");
    const int group = heads / kv_heads;
    if ((long)kv_heads * ((group + 15) / 16) > 65535) HB_REFUSE("attention_rows: %d heads", heads);
    if (((uintptr_t)kv % 16) || (((uintptr_t)q | (uintptr_t)out) % 8)) HB_REFUSE("attention_rows: the cache must start on 16 bytes, q and out on 8");
    if (skip && (!part_o || !part_ml || !part_at || window > 0)) HB_REFUSE("attention_rows: shared keys need their partial results, and no window");
    const RowsArgs a = {(bf16*)out, (const bf16*)q, (const unsigned char*)kv, block_table, row_slot, query_start, kv_len, sinks, skip, part_o,
                        part_ml, (const int4*)part_at, part_rows, table_stride, heads, kv_heads, head_dim, pages, page_size, window, splits,
                        scale * 1.4426950408889634f};
    return kv8 ? any_rows<true>(&a, rows, splits, group, head_dim, nullptr, (cudaStream_t)stream)
               : any_rows<false>(&a, rows, splits, group, head_dim, nullptr, (cudaStream_t)stream);
}
