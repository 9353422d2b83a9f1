// Writing the 8-bit cache, and reading it back.
//
// Write: q/k RMSNorm per head + rotation, as in rope_kv.cu, then every key and value row is scaled and rounded to codes
// (cache8.cuh). Everything before the one rounding is 32-bit: rounding a normed key to bfloat16 first would move about
// one code in thirty by a step. Bound by reading qkv and writing q and the codes.
// Read: a page's codes times their scales, as bfloat16 or 32-bit, either for a list of pages or for the pages that rows of
// several tokens attend over, which then hold zeros behind a row's last key.
#include "cache8.cuh"

template <typename TW> __device__ __forceinline__ float2 load_w2(const TW* w);
template <> __device__ __forceinline__ float2 load_w2<float>(const float* w) { return make_float2(w[0], w[1]); }
template <> __device__ __forceinline__ float2 load_w2<bf16>(const bf16* w) { return make_float2(to_f32(w[0]), to_f32(w[1])); }

// One warp per (token, head): query heads first, then key heads, then value heads; a row goes through shared memory.
template <typename TW>
__global__ void __launch_bounds__(256) qk_norm_rope_kv_write8_kernel(
        bf16* __restrict__ q_out, const bf16* __restrict__ qkv, const int32_t* __restrict__ positions,
        const float* __restrict__ table, int rotary_dim, int max_positions, const TW* __restrict__ q_weight,
        const TW* __restrict__ k_weight, float eps, float offset, unsigned char* __restrict__ kv,
        const int32_t* __restrict__ write_index, int pages, int page_size, long units, int heads, int kv_heads, int head_dim,
        const bf16* __restrict__ bias) {
    extern __shared__ float smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int items = heads + (kv ? 2 * kv_heads : 0);
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

extern "C" int hb_qk_norm_rope_kv_write8(void* q_out, const void* qkv, const int32_t* positions, const float* table,
                                         int rotary_dim, int max_positions, const void* q_weight, const void* k_weight,
                                         int weight_dtype, float eps, float offset, void* kv, const int32_t* write_index,
                                         int pages, int page_size, int tokens, int heads, int kv_heads, int head_dim,
                                         const void* bias, hb_stream stream) {
    if (tokens == 0) return 0;
    if (head_dim < 16 || head_dim % 16 || head_dim > 1024) HB_REFUSE("qk_norm_rope_kv_write8: head_dim %d is no multiple of 16 up to 1024", head_dim);
    if (kv && (page_size < 16 || page_size % 16)) HB_REFUSE("qk_norm_rope_kv_write8: page size %d is no multiple of 16", page_size);
    if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1))
        HB_REFUSE("qk_norm_rope_kv_write8: rotary_dim %d must be even and at most head_dim %d", rotary_dim, head_dim);
    if (rotary_dim && !table) HB_REFUSE("qk_norm_rope_kv_write8: a rotation needs its table");
    if ((q_weight == nullptr) != (k_weight == nullptr)) HB_REFUSE("qk_norm_rope_kv_write8: give both norm weights or none");
    if (kv && !write_index) HB_REFUSE("qk_norm_rope_kv_write8: writing the cache needs write_index");
    if (kv_heads < 1 || heads < 1) HB_REFUSE("qk_norm_rope_kv_write8: %d heads, %d kv heads", heads, kv_heads);
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)bias | (uintptr_t)kv) % 4) HB_REFUSE("qk_norm_rope_kv_write8: tensors must start on 4 bytes");
    cudaStream_t s = (cudaStream_t)stream;
    const long units = (long)tokens * (heads + (kv ? 2 * kv_heads : 0));
    const int warps = 4;
    const long blocks = (units + warps - 1) / warps;
    if (blocks > 0x7fffffffl) HB_REFUSE("qk_norm_rope_kv_write8: %d tokens in one step", tokens);
#define HB_ARGS(TW) (bf16*)q_out, (const bf16*)qkv, positions, table, rotary_dim, max_positions, (const TW*)q_weight, (const TW*)k_weight, \
    eps, offset, (unsigned char*)kv, write_index, pages, page_size, units, heads, kv_heads, head_dim, (const bf16*)bias
    if (weight_dtype == HB_BF16)
        qk_norm_rope_kv_write8_kernel<bf16><<<(unsigned)blocks, warps * 32, warps * head_dim * sizeof(float), s>>>(HB_ARGS(bf16));
    else
        qk_norm_rope_kv_write8_kernel<float><<<(unsigned)blocks, warps * 32, warps * head_dim * sizeof(float), s>>>(HB_ARGS(float));
#undef HB_ARGS
    HB_LAUNCH_CHECK("qk_norm_rope_kv_write8");
    return 0;
}

// ---------------------------------------------------------------- reading back
template <typename T> __device__ __forceinline__ void store16(T* dst, const uint4& codes, float scale);
template <> __device__ __forceinline__ void store16<bf16>(bf16* dst, const uint4& codes, float scale) {
    uint4 a, b;
    c8_unpack16(codes, scale, a, b);
    *(uint4*)dst = a;
    *(uint4*)(dst + 8) = b;
}
template <> __device__ __forceinline__ void store16<float>(float* dst, const uint4& codes, float scale) {
    uint4 a, b;
    c8_unpack16(codes, scale, a, b);                 // (exact in bfloat16, so through it)
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) *(float2*)(dst + 2 * i) = __bfloat1622float2(*(const __nv_bfloat162*)&w[i]);
}

// One page, 16 codes a thread and turn; rows [0, keep) of every block as they are, the others as zeros.
template <typename T>
__device__ __forceinline__ void read_page(T* __restrict__ out, const unsigned char* __restrict__ kv, bool valid, int keep,
                                          int kv_heads, int page_size, int head_dim) {
    const int per_row = head_dim >> 4, chunks = 2 * kv_heads * page_size * per_row;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < chunks; i += gridDim.y * blockDim.x) {
        const int row = i / per_row, at = i - row * per_row, blk = row / page_size, r = row - blk * page_size;
        uint4 codes = make_uint4(0, 0, 0, 0);
        float scale = 0.f;
        if (valid && r < keep) {
            const unsigned char* b = kv + (size_t)blk * page_size * (head_dim + 1);
            codes = *(const uint4*)(b + (size_t)r * head_dim + at * 16);
            scale = c8_power((int)b[(size_t)page_size * head_dim + r] - 127);
        }
        store16<T>(out + (size_t)i * 16, codes, scale);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(T* __restrict__ out, const unsigned char* __restrict__ kv,
                                                      const int32_t* __restrict__ index, int pages, int kv_heads, int page_size, int head_dim) {
    const int page = index[blockIdx.x];
    const bool valid = page >= 0 && page < pages;
    const size_t rows = (size_t)2 * kv_heads * page_size;
    read_page<T>(out + (size_t)blockIdx.x * rows * head_dim, kv + (valid ? (size_t)page * rows * (head_dim + 1) : 0), valid, page_size,
                 kv_heads, page_size, head_dim);
}

// Rows row0 .. rows - 1: the pages that hold keys which one of a row's new tokens sees go to out, page i of row b at
// (b - row0) * stride + i, and the tables with which an attention kernel finds them there are made: table [rows - row0, stride]
// and slots [rows] (slots[b] = b - row0).
__global__ void __launch_bounds__(256) kv_read_rows_kernel(bf16* __restrict__ out, int32_t* __restrict__ table, int32_t* __restrict__ slots,
                                                           const unsigned char* __restrict__ kv, const int32_t* __restrict__ block_table,
                                                           int table_stride, const int32_t* __restrict__ row_slot,
                                                           const int32_t* __restrict__ query_start, const int32_t* __restrict__ kv_len, int row0,
                                                           int stride, int pages, int kv_heads, int page_size, int head_dim, int window) {
    const int r = blockIdx.z, i = blockIdx.x, b = row0 + r;
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        table[(size_t)r * stride + i] = r * stride + i;
        if (i == 0) slots[b] = r;
    }
    const int n = kv_len[b], first = n - (query_start[b + 1] - query_start[b]);
    const int lo = window > 0 ? max(0, first - window + 1) : 0;
    if (i * page_size >= n || (i + 1) * page_size <= lo) return;
    const int page = block_table[(size_t)row_slot[b] * table_stride + i];
    const bool valid = page >= 0 && page < pages;
    const size_t size = (size_t)2 * kv_heads * page_size;
    read_page<bf16>(out + ((size_t)r * stride + i) * size * head_dim, kv + (valid ? (size_t)page * size * (head_dim + 1) : 0), valid,
                    n - i * page_size, kv_heads, page_size, head_dim);
}

static int check_pages(const char* who, const void* out, const void* kv, int kv_heads, int page_size, int head_dim) {
    if (head_dim < 16 || head_dim % 16) HB_REFUSE("%s: head_dim %d is no multiple of 16", who, head_dim);
    if (page_size < 16 || page_size % 16) HB_REFUSE("%s: page size %d is no multiple of 16", who, page_size);
    if (kv_heads < 1 || (long)2 * kv_heads * page_size * head_dim > 0x7fffffffl) HB_REFUSE("%s: %d kv heads of %d in pages of %d", who, kv_heads, head_dim, page_size);
    if (((uintptr_t)out | (uintptr_t)kv) % 16) HB_REFUSE("%s: tensors must start on 16 bytes", who);
    return 0;
}
static unsigned slices(int kv_heads, int page_size, int head_dim) {      // blocks a page: about 1,024 chunks each
    const long chunks = (long)2 * kv_heads * page_size * (head_dim / 16);
    return (unsigned)min(65535l, (chunks + 1023) / 1024);
}

extern "C" int hb_kv_read(void* out, int dtype, const void* kv, const int32_t* index, int count, int pages, int kv_heads, int page_size,
                          int head_dim, hb_stream stream) {
    if (count == 0) return 0;
    if (int rc = check_pages("kv_read", out, kv, kv_heads, page_size, head_dim)) return rc;
    const dim3 grid(count, slices(kv_heads, page_size, head_dim));
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == HB_BF16)
        kv_read_kernel<bf16><<<grid, 256, 0, s>>>((bf16*)out, (const unsigned char*)kv, index, pages, kv_heads, page_size, head_dim);
    else if (dtype == HB_F32)
        kv_read_kernel<float><<<grid, 256, 0, s>>>((float*)out, (const unsigned char*)kv, index, pages, kv_heads, page_size, head_dim);
    else HB_REFUSE("kv_read: no kernel for dtype %d", dtype);
    HB_LAUNCH_CHECK("kv_read");
    return 0;
}

extern "C" int hb_kv_read_rows(void* out, int32_t* table, int32_t* slots, const void* kv, const int32_t* block_table, int table_stride,
                               const int32_t* row_slot, const int32_t* query_start, const int32_t* kv_len, int row0, int rows, int stride,
                               int pages, int kv_heads, int page_size, int head_dim, int window, hb_stream stream) {
    if (rows <= row0 || stride < 1) return 0;
    if (int rc = check_pages("kv_read_rows", out, kv, kv_heads, page_size, head_dim)) return rc;
    if (stride > table_stride) HB_REFUSE("kv_read_rows: %d pages a row, the block table has %d", stride, table_stride);
    if (rows - row0 > 65535) HB_REFUSE("kv_read_rows: %d rows", rows - row0);
    kv_read_rows_kernel<<<dim3(stride, slices(kv_heads, page_size, head_dim), rows - row0), 256, 0, (cudaStream_t)stream>>>(
        (bf16*)out, table, slots, (const unsigned char*)kv, block_table, table_stride, row_slot, query_start, kv_len, row0, stride, pages,
        kv_heads, page_size, head_dim, window);
    HB_LAUNCH_CHECK("kv_read_rows");
    return 0;
}
