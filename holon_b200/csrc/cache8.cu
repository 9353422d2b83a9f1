// Writing the 8-bit cache, and reading it back.
//
// Write: q/k RMSNorm per head + rotation, as in rope_kv.cu, then every key and value row is scaled and rounded to codes
// (cache8.cuh). Everything before the one rounding is 32-bit: rounding a normed key to bfloat16 first would move about
// one code in thirty by a step.
// Read: a page's codes times their scales, as bfloat16 or 32-bit, either for a list of pages or for the pages that rows of
// several tokens attend over, which then hold zeros behind a row's last key.
#include "cache8.cuh"
#include "tcgen05.cuh"

template <typename TW> __device__ __forceinline__ float2 load_w2(const TW* w);
template <> __device__ __forceinline__ float2 load_w2<float>(const float* w) { return make_float2(w[0], w[1]); }
template <> __device__ __forceinline__ float2 load_w2<bf16>(const bf16* w) { return make_float2(to_f32(w[0]), to_f32(w[1])); }

// One warp per (token, head): query heads first, then key heads, then value heads; a row goes through shared memory. Any rotation, any
// head size, any alignment.
template <typename TW>
__global__ void __launch_bounds__(128) qk_norm_rope_kv_write8_kernel(
        bf16* __restrict__ q_out, const bf16* __restrict__ qkv, const int32_t* __restrict__ positions,
        const float* __restrict__ table, int rotary_dim, int max_positions, const TW* __restrict__ q_weight,
        const TW* __restrict__ k_weight, float eps, float offset, unsigned char* __restrict__ kv,
        const int32_t* __restrict__ write_index, int pages, int page_size, long units, int heads, int kv_heads, int head_dim,
        const bf16* __restrict__ bias) {
    extern __shared__ float smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int items = heads + 2 * kv_heads;
    const long unit = (long)blockIdx.x * (blockDim.x >> 5) + warp;
    if (unit >= units) return;                       // (a whole warp; nothing below waits for another one)
    const long t = unit / items;
    const int item = (int)(unit - t * items);
    float* y = smem + warp * head_dim;
    const bf16* src = qkv + ((size_t)t * (heads + 2 * kv_heads) + item) * head_dim;
    const bf16* add = bias ? bias + (size_t)item * head_dim : nullptr;
    const bool is_q = item < heads, is_v = item >= heads + kv_heads;
    int page = 0, off = 0;
    if (!is_q) {
        const int w = write_index[t];
        if (w < 0) return;
        page = w / page_size;
        off = w - page * page_size;
        if (page >= pages) return;
    }
    float ss = 0.f;
    for (int d = lane * 2; d < head_dim; d += 64) {
        float2 v = __bfloat1622float2(*(const __nv_bfloat162*)(src + d));
        if (add) { const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)(add + d)); v.x += a.x; v.y += a.y; }
        y[d] = v.x; y[d + 1] = v.y;
        ss += v.x * v.x + v.y * v.y;
    }
    const TW* weight = is_q ? q_weight : is_v ? nullptr : k_weight;
    if (weight) {
        const float rstd = rsqrtf(warp_sum(ss) / (float)head_dim + eps);
        for (int d = lane * 2; d < head_dim; d += 64) {
            const float2 w = load_w2<TW>(weight + d);
            y[d] *= rstd * (w.x + offset);
            y[d + 1] *= rstd * (w.y + offset);
        }
    }
    __syncwarp();
    if (!is_v && rotary_dim) {
        const int half = rotary_dim >> 1;
        int pos = positions[t];
        pos = pos < 0 ? 0 : (pos >= max_positions ? max_positions - 1 : pos);
        const float* cs = table + (size_t)pos * rotary_dim;
        for (int i = lane; i < half; i += 32) {
            const float a = y[i], b = y[i + half], c = cs[i], s = cs[half + i];
            y[i] = a * c - b * s;
            y[i + half] = b * c + a * s;
        }
        __syncwarp();
    }
    if (is_q) {
        bf16* dst = q_out + ((size_t)t * heads + item) * head_dim;
        for (int d = lane * 2; d < head_dim; d += 64) *(__nv_bfloat162*)(dst + d) = __floats2bfloat162_rn(y[d], y[d + 1]);
        return;
    }
    float largest = 0.f;
    for (int d = lane; d < head_dim; d += 32) largest = fmaxf(largest, c8_magnitude(y[d]));
    const int e = c8_exponent(warp_max(largest));
    const float inv = c8_power(-e);
    const size_t block = (size_t)page_size * (head_dim + 1);
    unsigned char* base = kv + (((size_t)page * 2 + is_v) * kv_heads + (item - heads - (is_v ? kv_heads : 0))) * block;
    for (int d = lane * 4; d < head_dim; d += 128)
        *(uint32_t*)(base + (size_t)off * head_dim + d) = c8_pack4(y[d] * inv, y[d + 1] * inv, y[d + 2] * inv, y[d + 3] * inv);
    if (lane == 0) base[(size_t)page_size * head_dim + off] = (unsigned char)(e + 127);
}

// The same with LANES lanes a (token, head), heads of up to 16 LANES numbers and rotations of a multiple of 16: a lane holds two
// chunks of 8, where the head turns the two that pair (chunk c of the first half of the turned numbers and c of the second), so
// that every access is 16 bytes wide, sums and maxima are shuffles and nothing goes through shared memory. 4,096 tokens of 32 + 8
// heads of 128: 90 us in the kernel above, 27.6 us here (92 MB, 3.3 TB/s). No unit is at its limit (66% of the issue slots, 22% of DRAM): it waits for
// its loads with 24 warps an SM, and every one of a token's heads loads the rotation's row and the gains and multiplies them anew.
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = __bfloat1622float2(*(const __nv_bfloat162*)&w[i]);
        f[2 * i] = p.x; f[2 * i + 1] = p.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *(uint32_t*)&p;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename TW> __device__ __forceinline__ void load8(const TW* w, float (&f)[8]);
template <> __device__ __forceinline__ void load8<bf16>(const bf16* w, float (&f)[8]) { unpack8(*(const uint4*)w, f); }
template <> __device__ __forceinline__ void load8<float>(const float* w, float (&f)[8]) {
    const float4 a = *(const float4*)w, b = *(const float4*)(w + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// Two numbers in one 64-bit register: an instruction of sm_100 does both (tcgen05.cuh has the names).
struct Eight {
    uint64_t v[4];
    __device__ __forceinline__ Eight() {}
    __device__ __forceinline__ explicit Eight(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pack2(f[2 * i], f[2 * i + 1]);
    }
    __device__ __forceinline__ void to(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(v[i], f[2 * i], f[2 * i + 1]);
    }
};
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <typename TW, int LANES>
__global__ void __launch_bounds__(256, 3) qk_norm_rope_kv_write8_lanes_kernel(
        bf16* __restrict__ q_out, const bf16* __restrict__ qkv, const int32_t* __restrict__ positions,
        const float* __restrict__ table, int rotary_dim, int max_positions, const TW* __restrict__ q_weight,
        const TW* __restrict__ k_weight, float eps, float offset, unsigned char* __restrict__ kv,
        const int32_t* __restrict__ write_index, int pages, int page_size, int page_shift, unsigned units, int heads, int kv_heads, int head_dim,
        const bf16* __restrict__ bias) {
    const unsigned items = heads + 2 * kv_heads, step = gridDim.x * (256 / LANES);
    const unsigned step_t = step / items, step_item = step - step_t * items;
    const int sub = threadIdx.x & (LANES - 1);
    const bool pairs = sub < rotary_dim >> 4, inside = sub < head_dim >> 4;      // (a value head's chunks are cut alike)
    const int c0 = pairs ? sub * 8 : rotary_dim + (sub - (rotary_dim >> 4)) * 16, c1 = pairs ? c0 + (rotary_dim >> 1) : c0 + 8;
    const bf16* first = qkv + (inside ? c0 : 0);
    const int apart = inside ? c1 - c0 : 0, width = (heads + 2 * kv_heads) * head_dim;
    // A unit's numbers, its position and its place in the cache are asked for a turn ahead: what a turn waits for is the rotation's row.
    uint4 na = make_uint4(0, 0, 0, 0), nb = na;
    int n_pos = 0, n_write = 0;
    const unsigned mine = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, warps_first = mine - (threadIdx.x & 31) / LANES;
    unsigned t = mine / items, item = mine - t * items;
    auto ask = [&](unsigned u) {
        if (u >= units) return;
        const bf16* src = first + (size_t)t * width + item * head_dim;
        if (inside) { na = *(const uint4*)src; nb = *(const uint4*)(src + apart); }
        if (rotary_dim) n_pos = positions[t];
        n_write = write_index[t];
    };
    // (every lane of a warp makes as many turns: the shuffles are the whole warp's)
    ask(mine);
    for (unsigned u0 = warps_first, u = mine; u0 < units; u0 += step, u += step) {
        const uint4 ra = na, rb = nb;
        const int write = n_write, head = (int)item;
        const unsigned token = t;
        const bool is_q = head < heads, is_v = head >= heads + kv_heads, turns = !is_v && pairs;
        bool live = inside && u < units;
        int pos = n_pos;
        float a[8], b[8], cs[8], sn[8];
        const TW* weight = is_q ? q_weight : is_v ? nullptr : k_weight;
        if (live && turns) {
            pos = pos < 0 ? 0 : (pos >= max_positions ? max_positions - 1 : pos);
            const float* row = table + (size_t)pos * rotary_dim + sub * 8;
            load8<float>(row, cs);
            load8<float>(row + (rotary_dim >> 1), sn);
        }
        t += step_t;
        item += step_item;
        if (item >= items) { item -= items; ++t; }
        ask(u + step);
        unpack8(ra, a);
        unpack8(rb, b);
        if (bias && live) {
            float x[8], y[8];
            load8<bf16>(bias + (size_t)head * head_dim + c0, x);
            load8<bf16>(bias + (size_t)head * head_dim + c1, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) { a[i] += x[i]; b[i] += y[i]; }
        }
        Eight pa(a), pb(b);
        if (__any_sync(0xffffffffu, weight != nullptr)) {
            uint64_t sums = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sums = fma2(pa.v[i], pa.v[i], fma2(pb.v[i], pb.v[i], sums));
            float s0, s1;
            unpack2(sums, s0, s1);
            float ss = inside ? s0 + s1 : 0.f;                       // (lanes behind the head's end take part with zeros)
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (weight && live) {
                const float rstd = rsqrtf(ss / (float)head_dim + eps);
                const uint64_t r2 = pack2(rstd, rstd), o2 = pack2(offset * rstd, offset * rstd);
                float wa[8], wb[8];
                load8<TW>(weight + c0, wa);                          // (few lines, which every unit reads: they are near)
                load8<TW>(weight + c1, wb);
                const Eight ga(wa), gb(wb);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    pa.v[i] = mul2(pa.v[i], fma2(ga.v[i], r2, o2));
                    pb.v[i] = mul2(pb.v[i], fma2(gb.v[i], r2, o2));
                }
            }
        }
        if (live && turns) {
            const Eight c(cs), n(sn);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t x = mul2(pb.v[i], n.v[i]), y = mul2(pa.v[i], n.v[i]);
                pa.v[i] = fma2(pa.v[i], c.v[i], x ^ 0x8000000080000000ull);      // a cos - b sin
                pb.v[i] = fma2(pb.v[i], c.v[i], y);
            }
        }
        pa.to(a);
        pb.to(b);
        if (live && is_q) {
            bf16* dst = q_out + ((size_t)token * heads + head) * head_dim;
            *(uint4*)(dst + c0) = pack8(a);
            *(uint4*)(dst + c1) = pack8(b);
        }
        if (!__any_sync(0xffffffffu, live && !is_q)) continue;
        float largest = 0.f, any = 0.f;                              // (a sum is finite unless a number is not, or the numbers nearly are not)
        if (inside) {
            uint64_t sums = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sums = add2(sums, add2(pa.v[i], pb.v[i]));
#pragma unroll
            for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fmaxf(fabsf(a[i]), fabsf(b[i])));
            float s0, s1;
            unpack2(sums, s0, s1);
            any = s0 + s1;
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        if (__any_sync(0xffffffffu, !(fabsf(any) < INFINITY))) {      // (rows with infinities or NaN: the largest finite one, and NaN for the others)
            largest = 0.f;
            if (inside)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    largest = fmaxf(largest, fmaxf(c8_magnitude(a[i]), c8_magnitude(b[i])));
                    if (fabsf(a[i]) == INFINITY) a[i] = __uint_as_float(0x7fc00000u);
                    if (fabsf(b[i]) == INFINITY) b[i] = __uint_as_float(0x7fc00000u);
                }
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        }
        if (live && !is_q && write >= 0) {
            const int page = page_shift >= 0 ? write >> page_shift : write / page_size, off = write - page * page_size;
            if (page < pages) {
                unsigned char* base = kv + (((size_t)page * 2 + is_v) * kv_heads + (head - heads - (is_v ? kv_heads : 0))) * ((size_t)page_size * (head_dim + 1));
                const int e = c8_exponent(largest);
                const uint64_t inv = pack2(c8_power(-e), c8_power(-e));
                Eight qa(a), qb(b);
#pragma unroll
                for (int i = 0; i < 4; ++i) { qa.v[i] = mul2(qa.v[i], inv); qb.v[i] = mul2(qb.v[i], inv); }
                qa.to(a);
                qb.to(b);
                unsigned char* row = base + (size_t)off * head_dim;
                *(uint2*)(row + c0) = make_uint2(c8_pack4_finite(a[0], a[1], a[2], a[3]), c8_pack4_finite(a[4], a[5], a[6], a[7]));
                *(uint2*)(row + c1) = make_uint2(c8_pack4_finite(b[0], b[1], b[2], b[3]), c8_pack4_finite(b[4], b[5], b[6], b[7]));
                if (sub == 0) base[(size_t)page_size * head_dim + off] = (unsigned char)(e + 127);
            }
        }
    }
}

extern "C" int hb_qk_norm_rope_kv_write8(void* q_out, const void* qkv, const int32_t* positions, const float* table,
                                         int rotary_dim, int max_positions, const void* q_weight, const void* k_weight,
                                         int weight_dtype, float eps, float offset, void* kv, const int32_t* write_index,
                                         int pages, int page_size, int tokens, int heads, int kv_heads, int head_dim,
                                         const void* bias, hb_stream stream) {
    if (tokens == 0) return 0;
    if (head_dim < 16 || head_dim % 16 || head_dim > 1024) HB_REFUSE("qk_norm_rope_kv_write8: head_dim %d is no multiple of 16 up to 1024", head_dim);
    if (!kv || !write_index) HB_REFUSE("qk_norm_rope_kv_write8: needs a cache and write_index");
    if (page_size < 16 || page_size % 16) HB_REFUSE("qk_norm_rope_kv_write8: page size %d is no multiple of 16", page_size);
    if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1))
        HB_REFUSE("qk_norm_rope_kv_write8: rotary_dim %d must be even and at most head_dim %d", rotary_dim, head_dim);
    if (rotary_dim && (!table || max_positions < 1)) HB_REFUSE("qk_norm_rope_kv_write8: a rotation needs its table");
    if ((q_weight == nullptr) != (k_weight == nullptr)) HB_REFUSE("qk_norm_rope_kv_write8: give both norm weights or none");
    if (kv_heads < 1 || heads < 1) HB_REFUSE("qk_norm_rope_kv_write8: %d heads, %d kv heads", heads, kv_heads);
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)bias | (uintptr_t)kv) % 4) HB_REFUSE("qk_norm_rope_kv_write8: tensors must start on 4 bytes");
    cudaStream_t s = (cudaStream_t)stream;
    const long units = (long)tokens * (heads + 2 * kv_heads);
#define HB_ARGS(TW) (bf16*)q_out, (const bf16*)qkv, positions, table, rotary_dim, max_positions, (const TW*)q_weight, (const TW*)k_weight, \
    eps, offset, (unsigned char*)kv, write_index, pages, page_size, units, heads, kv_heads, head_dim, (const bf16*)bias
    const bool aligned = ((uintptr_t)q_out | (uintptr_t)qkv | (uintptr_t)table | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)kv | (uintptr_t)bias) % 16 == 0;
    const bool lanes = aligned && rotary_dim % 16 == 0 && head_dim <= 256 && units < (1l << 31);
    const int width = !lanes ? 64 : head_dim <= 32 ? 2 : head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16;      // threads a unit; the general kernel: 4 units a block
    const long blocks = (units + 256 / width - 1) / (256 / width);
    if (blocks > 0x7fffffffl) HB_REFUSE("qk_norm_rope_kv_write8: %d tokens in one step", tokens);
    static int sms = 0;                                              // (three blocks an SM hold all of a step's tokens in turns)
    if (sms == 0) HB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, 0));
#define HB_LANES(TW, N) qk_norm_rope_kv_write8_lanes_kernel<TW, N><<<(unsigned)min(blocks, 3l * sms), 256, 0, s>>>( \
        (bf16*)q_out, (const bf16*)qkv, positions, table, rotary_dim, max_positions, (const TW*)q_weight, (const TW*)k_weight, eps, offset, \
        (unsigned char*)kv, write_index, pages, page_size, page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size), (unsigned)units, heads, kv_heads, head_dim, (const bf16*)bias)
#define HB_WRITE(TW) do { \
        if (!lanes) qk_norm_rope_kv_write8_kernel<TW><<<(unsigned)blocks, 128, 4 * head_dim * sizeof(float), s>>>(HB_ARGS(TW)); \
        else if (width == 2) HB_LANES(TW, 2); \
        else if (width == 4) HB_LANES(TW, 4); \
        else if (width == 8) HB_LANES(TW, 8); \
        else HB_LANES(TW, 16); \
    } while (0)
    if (weight_dtype == HB_BF16) HB_WRITE(bf16);
    else HB_WRITE(float);
#undef HB_WRITE
#undef HB_LANES
#undef HB_ARGS
    HB_LAUNCH_CHECK("qk_norm_rope_kv_write8");
    return 0;
}

// ---------------------------------------------------------------- reading back
template <typename T> __device__ __forceinline__ void store16(T* dst, const uint4& codes, float scale);
__device__ __forceinline__ void store32(void* dst, const uint4& a, const uint4& b) {             // 32 bytes in one store: a whole sector a lane
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}
template <> __device__ __forceinline__ void store16<bf16>(bf16* dst, const uint4& codes, float scale) {
    uint4 a, b;
    c8_unpack16(codes, scale, a, b);
    store32(dst, a, b);
}
template <> __device__ __forceinline__ void store16<float>(float* dst, const uint4& codes, float scale) {
    uint4 a, b;
    c8_unpack16(codes, scale, a, b);                 // (exact in bfloat16, so through it)
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) { f[2 * i] = w[i] << 16; f[2 * i + 1] = w[i] & 0xffff0000u; }
    store32(dst, make_uint4(f[0], f[1], f[2], f[3]), make_uint4(f[4], f[5], f[6], f[7]));
    store32(dst + 8, make_uint4(f[8], f[9], f[10], f[11]), make_uint4(f[12], f[13], f[14], f[15]));
}

// One (part, kv head) block of a page, blockIdx.y's, to `out`, 16 codes a thread and turn, four turns' loads at once; rows [skip, keep) as
// they are, the others as zeros, none from `upto` on. shift: log2 of the chunks of 16 codes a row, or -1.
#define RD_THREADS 128
#define RD_TURNS 4
template <typename T>
__device__ __forceinline__ void read_block(T* __restrict__ out, const unsigned char* __restrict__ kv, bool valid, int skip, int keep, int upto, int page_size, int head_dim, int shift) {
    const int per_row = head_dim >> 4, chunks = min(page_size, upto) * per_row;
    const size_t blk = blockIdx.y, codes_of = (size_t)page_size * head_dim;
    const unsigned char* b = kv + blk * (codes_of + page_size);
    for (int i0 = threadIdx.x; i0 < chunks; i0 += RD_THREADS * RD_TURNS) {
        uint4 codes[RD_TURNS];
        float scale[RD_TURNS];
#pragma unroll
        for (int k = 0; k < RD_TURNS; ++k) {
            const int i = i0 + k * RD_THREADS, r = shift >= 0 ? i >> shift : i / per_row;
            const bool take = valid && i < chunks && r >= skip && r < keep;
            codes[k] = take ? *(const uint4*)(b + (size_t)i * 16) : make_uint4(0, 0, 0, 0);
            scale[k] = take ? c8_power((int)b[codes_of + r] - 127) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < RD_TURNS; ++k)
            if (i0 + k * RD_THREADS < chunks) store16<T>(out + (size_t)(i0 + k * RD_THREADS) * 16, codes[k], scale[k]);
    }
}

template <typename T>
__global__ void __launch_bounds__(RD_THREADS) kv_read_kernel(T* __restrict__ out, const unsigned char* __restrict__ kv,
                                                             const int32_t* __restrict__ index, int pages, int page_size, int head_dim, int shift) {
    const int page = index[blockIdx.x];
    const bool valid = page >= 0 && page < pages;
    const size_t rows = (size_t)gridDim.y * page_size;
    read_block<T>(out + ((size_t)blockIdx.x * rows + (size_t)blockIdx.y * page_size) * head_dim, kv + (valid ? (size_t)page * rows * (head_dim + 1) : 0),
                  valid, 0, page_size, page_size, page_size, head_dim, shift);
}

// Rows row0 .. rows - 1: the keys and values that one of a row's new tokens sees, in a row: out [rows - row0, 2, kv_heads, length,
// head_dim]. Zeros stand before them from the last multiple of 64 on and behind them up to the next (attention kernels read whole
// tiles). The tables with which an attention kernel finds row b's keys as one page b - row0 are made, too: table [rows - row0], slots [rows].
// 6,144 tokens of 8 kv heads of 128: 8.5 us (38 MB, most of it to and from L2; page by page, without the way in a row, 8.5 us as well, and pages
// of 16 and 32 tokens then had to be attended to by the mma.sync kernel).
__global__ void __launch_bounds__(RD_THREADS) kv_read_rows_kernel(bf16* __restrict__ out, int32_t* __restrict__ table, int32_t* __restrict__ slots,
                                                                  const unsigned char* __restrict__ kv, const int32_t* __restrict__ block_table,
                                                                  int table_stride, const int32_t* __restrict__ row_slot,
                                                                  const int32_t* __restrict__ query_start, const int32_t* __restrict__ kv_len, int row0,
                                                                  int length, int pages, int page_size, int head_dim, int window, int shift) {
    const int r = blockIdx.z, i = blockIdx.x, b = row0 + r;
    if (threadIdx.x == 0 && blockIdx.y == 0 && i == 0) { table[r] = r; slots[b] = r; }
    const int n = kv_len[b], first = n - (query_start[b + 1] - query_start[b]);
    const int lo = window > 0 ? max(0, first - window + 1) : 0, at = i * page_size;
    if (at >= ((n + 63) & ~63) || at + page_size <= (lo & ~63)) return;
    const int page = at < n && at + page_size > lo ? block_table[(size_t)row_slot[b] * table_stride + i] : -1;
    const bool valid = page >= 0 && page < pages;
    const size_t rows = (size_t)gridDim.y * page_size;
    read_block<bf16>(out + (((size_t)r * gridDim.y + blockIdx.y) * length + at) * head_dim, kv + (valid ? (size_t)page * rows * (head_dim + 1) : 0),
                     valid, lo - at, n - at, length - at, page_size, head_dim, shift);
}

static int check_pages(const char* who, const void* out, const void* kv, int kv_heads, int page_size, int head_dim) {
    if (head_dim < 16 || head_dim % 16) HB_REFUSE("%s: head_dim %d is no multiple of 16", who, head_dim);
    if (page_size < 16 || page_size % 16) HB_REFUSE("%s: page size %d is no multiple of 16", who, page_size);
    if (kv_heads < 1 || (long)2 * kv_heads * page_size * head_dim > 0x7fffffffl) HB_REFUSE("%s: %d kv heads of %d in pages of %d", who, kv_heads, head_dim, page_size);
    if (2 * kv_heads > 65535) HB_REFUSE("%s: %d kv heads", who, kv_heads);
    if ((uintptr_t)out % 32 || (uintptr_t)kv % 16) HB_REFUSE("%s: out must start on 32 bytes, the cache on 16", who);
    return 0;
}
static int chunk_shift(int head_dim) {                // log2 of the chunks of 16 a row, or -1
    const int n = head_dim / 16;
    return (n & (n - 1)) == 0 ? __builtin_ctz(n) : -1;
}

extern "C" int hb_kv_read(void* out, int dtype, const void* kv, const int32_t* index, int count, int pages, int kv_heads, int page_size,
                          int head_dim, hb_stream stream) {
    if (count == 0) return 0;
    if (int rc = check_pages("kv_read", out, kv, kv_heads, page_size, head_dim)) return rc;
    const dim3 grid(count, 2 * kv_heads);
    const int shift = chunk_shift(head_dim);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == HB_BF16)
        kv_read_kernel<bf16><<<grid, RD_THREADS, 0, s>>>((bf16*)out, (const unsigned char*)kv, index, pages, page_size, head_dim, shift);
    else if (dtype == HB_F32)
        kv_read_kernel<float><<<grid, RD_THREADS, 0, s>>>((float*)out, (const unsigned char*)kv, index, pages, page_size, head_dim, shift);
    else HB_REFUSE("kv_read: no kernel for dtype %d", dtype);
    HB_LAUNCH_CHECK("kv_read");
    return 0;
}

extern "C" int hb_kv_read_rows(void* out, int32_t* table, int32_t* slots, const void* kv, const int32_t* block_table, int table_stride,
                               const int32_t* row_slot, const int32_t* query_start, const int32_t* kv_len, int row0, int rows, int length,
                               int pages, int kv_heads, int page_size, int head_dim, int window, hb_stream stream) {
    if (rows <= row0 || length < 1) return 0;
    if (int rc = check_pages("kv_read_rows", out, kv, kv_heads, page_size, head_dim)) return rc;
    if (length % 64) HB_REFUSE("kv_read_rows: %d tokens a row are no multiple of 64", length);
    if (rows - row0 > 65535) HB_REFUSE("kv_read_rows: %d rows", rows - row0);
    kv_read_rows_kernel<<<dim3((length + page_size - 1) / page_size, 2 * kv_heads, rows - row0), RD_THREADS, 0, (cudaStream_t)stream>>>(
        (bf16*)out, table, slots, (const unsigned char*)kv, block_table, table_stride, row_slot, query_start, kv_len, row0, length, pages,
        page_size, head_dim, window, chunk_shift(head_dim));
    HB_LAUNCH_CHECK("kv_read_rows");
    return 0;
}
