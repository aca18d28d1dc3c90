// Rows into a cache held in 4 bits, and back out of it (packed.cuh has the format).
//
// kv_append_packed: four lanes hold a group, eight numbers each: minimum and maximum by two exchanges, one word of codes from
// every lane, the group's word from the first. Differences, quotients and roundings are IEEE float32, so that a row's bytes are a
// matter of its numbers alone. Bound by the bytes: the source rows are read once (16-byte pieces where they are aligned).
//
// kv_unpack: the rows of some requests as pages of the compute type, for kernels that read such pages (prompts in float32, head
// sizes that the packed prompt kernel does not take). One thread makes eight numbers of a row from a word.
#include "packed.cuh"

namespace ps {
namespace packed {

template <typename T> struct Eight;                      // eight numbers that a thread holds, as whole 16-byte pieces
template <> struct Eight<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&x)[8]) {
        const uint4 raw = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&x)[8]) {
        uint4 raw;
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&two);
        }
        *reinterpret_cast<uint4*>(p) = raw;
    }
};
template <> struct Eight<float> {
    static __device__ __forceinline__ void load(const float* p, float (&x)[8]) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
};

// thread = (token, k or v, head, group, part of the group); `aligned`: every part is whole 16-byte pieces of its row
template <typename T>
__global__ void __launch_bounds__(256)
append_kernel(const T* __restrict__ k_src, long long k_stride, const T* __restrict__ v_src, long long v_stride,
              const int* __restrict__ token_row, const int* __restrict__ positions, Pages pages, unsigned char* __restrict__ k_pool,
              unsigned char* __restrict__ v_pool, long long page_stride, int tokens, int planes, int n_kv_heads, int head_dim, int aligned) {
    pdl_prologue();
    k_src = pdl_fresh(k_src);
    v_src = pdl_fresh(v_src);
    const int groups = groups_of(head_dim), per_plane = n_kv_heads * groups * 4;
    const long long index = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool there = index < (long long)tokens * planes * per_plane;          // (the lanes of a group are there together)
    const long long row_index = there ? index / per_plane : 0;
    const int inside = there ? (int)(index - row_index * per_plane) : 0;
    const int t = (int)(row_index / planes), plane = planes == 2 ? (int)(row_index & 1) : (k_src ? 0 : 1);
    const int part = inside & 3, j = (inside >> 2) % groups, head = (inside >> 2) / groups;
    const int d = j * GROUP + part * 8;
    const int count = there ? min(8, head_dim - d) : 0;                          // numbers of this part that exist (may be negative)
    const T* src = (plane ? v_src + t * v_stride : k_src + t * k_stride) + head * head_dim + d;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (count == 8 && aligned) {
        Eight<T>::load(src, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) x[i] = to_float(src[i]);
    }
    float low = INFINITY, high = -INFINITY;
    bool bad = false;                                                            // (fminf and fmaxf pass NaN over)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < count) {
            low = fminf(low, x[i]);
            high = fmaxf(high, x[i]);
            bad |= x[i] != x[i];
        }
    if (bad) low = -INFINITY;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    if (!there) return;
    const int p = positions[t], page = pages.of(token_row[t], p);
    if (page < 0) return;
    low = bf16_below(low);
    float step = bf16_above(__fdiv_rn(__fsub_rn(high, low), 15.0f));
    uint32_t word = 0;
    if (isfinite(low) && isfinite(step)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float code = step > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], low), step)), 0.f), 15.f) : 0.f;
            if (i < count) word |= (uint32_t)(int)code << code_shift(i);
        }
    } else {
        low = step = __uint_as_float(0x7fff0000u);
    }
    const int page_size = 1 << pages.page_log2, row = p & (page_size - 1);
    unsigned char* slab = (plane ? v_pool : k_pool) + (long long)page * page_stride + (long long)head * slab_bytes(page_size, head_dim);
    reinterpret_cast<uint32_t*>(slab)[(row * 4 + part) * groups + j] = word;
    if (part == 0)
        reinterpret_cast<uint32_t*>(slab + page_size * groups * 16)[row * groups + j] =
            (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xffff0000u);
}

// thread = (item, position, k or v, head, word); out: pages [n_items * span / out_page, 2, kv heads, out_page, head_dim], item i's
// position p in page i * span / out_page + p / out_page. Positions from kv_len on are left as they are.
template <typename T>
__global__ void __launch_bounds__(256)
unpack_kernel(const unsigned char* __restrict__ k_pool, const unsigned char* __restrict__ v_pool, long long page_stride,
              const int* __restrict__ kv_len, const int* __restrict__ item_row, Pages pages, int span, T* __restrict__ out, int out_log2,
              int n_kv_heads, int head_dim, int aligned) {
    pdl_prologue();
    k_pool = pdl_fresh(k_pool);
    v_pool = pdl_fresh(v_pool);
    const int groups = groups_of(head_dim), words = groups * 4, per_row = 2 * n_kv_heads * words;
    const int item = blockIdx.y;
    const long long index = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long position64 = index / per_row;
    if (position64 >= span) return;
    const int p = (int)position64;
    if (p >= kv_len[item]) return;
    const int page = pages.of(item_row ? item_row[item] : item, p);
    if (page < 0) return;
    int rest = (int)(index - position64 * per_row);
    const int place = rest % words, plane = rest / words % 2, head = rest / words / 2;
    const int j = place % groups, d = j * GROUP + place / groups * 8;
    const int page_size = 1 << pages.page_log2, row = p & (page_size - 1);
    const unsigned char* slab = (plane ? v_pool : k_pool) + (long long)page * page_stride + (long long)head * slab_bytes(page_size, head_dim);
    const uint32_t word = reinterpret_cast<const uint32_t*>(slab)[row * words + place];
    const uint32_t scale = reinterpret_cast<const uint32_t*>(slab + page_size * groups * 16)[row * groups + j];
    const float step = step_of(scale), low = low_of(scale);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((word >> code_shift(i)) & 15u), step, low);
    const int out_size = 1 << out_log2;
    const long long out_page = (long long)item * (span >> out_log2) + (p >> out_log2);
    T* to = out + (((out_page * 2 + plane) * n_kv_heads + head) * out_size + (p & (out_size - 1))) * head_dim + d;
    const int count = head_dim - d;
    if (count >= 8 && aligned) {
        Eight<T>::store(to, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) to[i] = from_float<T>(x[i]);
    }
}

template <typename T>
int append(const void* k_src, long long k_stride, const void* v_src, long long v_stride, const int* token_row, const int* positions,
           const Pages& pages, void* k_pool, void* v_pool, long long page_stride, int tokens, int n_kv_heads, int head_dim, cudaStream_t s) {
    const int planes = (k_src ? 1 : 0) + (v_src ? 1 : 0);
    const long long threads = (long long)tokens * planes * n_kv_heads * groups_of(head_dim) * 4;
    if ((threads + 255) / 256 > 0x7fffffffll) return PS_ERR_UNSUPPORTED;
    constexpr int PER = 16 / (int)sizeof(T);
    const int aligned = !(((uintptr_t)k_src | (uintptr_t)v_src) & 15) && k_stride % PER == 0 && v_stride % PER == 0 && head_dim % 8 == 0;
    return launch_pdl(append_kernel<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, (const T*)k_src, k_stride, (const T*)v_src,
                      v_stride, token_row, positions, pages, (unsigned char*)k_pool, (unsigned char*)v_pool, page_stride, tokens, planes,
                      n_kv_heads, head_dim, aligned);
}

template <typename T>
int unpack(const void* k_pool, const void* v_pool, long long page_stride, const int* kv_len, const int* item_row, const Pages& pages, int n_items,
           int span, void* out, int out_page, int n_kv_heads, int head_dim, cudaStream_t s) {
    const long long threads = (long long)span * 2 * n_kv_heads * groups_of(head_dim) * 4;
    if ((threads + 255) / 256 > 0x7fffffffll) return PS_ERR_UNSUPPORTED;
    const int aligned = !((uintptr_t)out & 15) && head_dim % 8 == 0;
    return launch_pdl(unpack_kernel<T>, dim3((unsigned)((threads + 255) / 256), n_items), dim3(256), 0, s, (const unsigned char*)k_pool,
                      (const unsigned char*)v_pool, page_stride, kv_len, item_row, pages, span, (T*)out, log2_of(out_page), n_kv_heads, head_dim,
                      aligned);
}

}  // namespace packed
}  // namespace ps

// k_src / v_src: rows of n_kv_heads * head_dim numbers, k_stride / v_stride apart; either may be null (its plane stays as it is).
// token_row[t]: the row of block_table (bt_stride wide) with the pages of token t; a position below 0 or without a page is left out.
PS_EXPORT int ps_kv_append_packed(const void* k_src, long long k_stride, const void* v_src, long long v_stride, const int* token_row,
                                  const int* positions, const int* block_table, int bt_stride, void* k_pool, void* v_pool, int n_pages,
                                  long long page_stride, int tokens, int n_kv_heads, int head_dim, int page_size, int dtype, void* stream) {
    using namespace ps::packed;
    if (tokens <= 0 || (!k_src && !v_src)) return PS_OK;
    if (!token_row || !positions || !block_table || (k_src && !k_pool) || (v_src && !v_pool)) return PS_ERR_BAD_ARGUMENT;
    if (!sizes_ok(n_kv_heads, head_dim, page_size)) return PS_ERR_UNSUPPORTED;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    const Pages pages = {block_table, bt_stride, n_pages, log2_of(page_size)};
    if (dtype == PS_F32)
        return append<float>(k_src, k_stride, v_src, v_stride, token_row, positions, pages, k_pool, v_pool, page_stride, tokens, n_kv_heads,
                             head_dim, (cudaStream_t)stream);
    if (dtype == PS_BF16)
        return append<__nv_bfloat16>(k_src, k_stride, v_src, v_stride, token_row, positions, pages, k_pool, v_pool, page_stride, tokens,
                                     n_kv_heads, head_dim, (cudaStream_t)stream);
    return PS_ERR_UNSUPPORTED;
}

// kv_len / item_row: of the n_items items; span: positions that an item has room for in `out`, a multiple of out_page.
PS_EXPORT int ps_kv_unpack(const void* k_pool, const void* v_pool, int n_pages, long long page_stride, const int* kv_len, const int* block_table,
                           int bt_stride, const int* item_row, int n_items, int span, void* out, int out_page, int n_kv_heads, int head_dim,
                           int page_size, int dtype, void* stream) {
    using namespace ps::packed;
    if (n_items <= 0 || span <= 0) return PS_OK;
    if (!k_pool || !v_pool || !kv_len || !block_table || !out) return PS_ERR_BAD_ARGUMENT;
    if (!sizes_ok(n_kv_heads, head_dim, page_size) || n_items > 65535) return PS_ERR_UNSUPPORTED;
    if (out_page <= 0 || (out_page & (out_page - 1)) || span % out_page) return PS_ERR_BAD_ARGUMENT;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    const Pages pages = {block_table, bt_stride, n_pages, log2_of(page_size)};
    if (dtype == PS_F32)
        return unpack<float>(k_pool, v_pool, page_stride, kv_len, item_row, pages, n_items, span, out, out_page, n_kv_heads, head_dim,
                             (cudaStream_t)stream);
    if (dtype == PS_BF16)
        return unpack<__nv_bfloat16>(k_pool, v_pool, page_stride, kv_len, item_row, pages, n_items, span, out, out_page, n_kv_heads, head_dim,
                                     (cudaStream_t)stream);
    return PS_ERR_UNSUPPORTED;
}
