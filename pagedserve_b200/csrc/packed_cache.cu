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

__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// The codes of eight numbers as a word. Quotients by the reciprocal are within 2e-6 of the rounded ones: they name the same code unless one of them is
// near half a code, where the divisions decide. (The codes are 0 to 15 by themselves: low is not above a number, 15 steps from it not below.) Four codes add up to 16
// bits in float32, exactly.
__device__ __forceinline__ uint32_t word_of(const float (&x)[8], float low, float step) {
    if (!(step > 0.f)) return 0u;
    const float reciprocal = __frcp_rn(step);
    float code[8], off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float quotient = __fsub_rn(x[i], low) * reciprocal;
        code[i] = __fadd_rn(__fadd_rn(quotient, 12582912.f), -12582912.f);        // (1.5 * 2^23: the nearest whole number, ties to even)
        off = fmaxf(off, fabsf(quotient - code[i]));
    }
    if (!(off <= 0.4999f) || step < 1e-30f)
#pragma unroll
        for (int i = 0; i < 8; ++i) code[i] = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], low), step)), 0.f), 15.f);
    const float even = fmaf(fmaf(fmaf(code[6], 16.f, code[4]), 16.f, code[2]), 16.f, code[0]);
    const float odd = fmaf(fmaf(fmaf(code[7], 16.f, code[5]), 16.f, code[3]), 16.f, code[1]);
    return __byte_perm(__float_as_uint(even + 8388608.f), __float_as_uint(odd + 8388608.f), 0x5410);
}

// A token's parts (k or v, head, group, part of the group) over the threads of blockIdx.y = 0, 1, ..; `aligned`: every part is whole 16-byte pieces of its
// row.  What bounds it is instructions: 3,988 rows of 25 heads of 64 in float32 are 18.2 M of warps (285 a warp of 16 a token, whose last lanes have nothing
// to do), 15.6 us of all issue slots in 20.5 (30 with an index over the parts of all tokens, a division and a shift for every number, 26 without that index; several
// tokens a thread gained nothing).
template <typename T>
__global__ void __launch_bounds__(256)
append_kernel(const T* __restrict__ k_src, long long k_stride, const T* __restrict__ v_src, long long v_stride,
              const int* __restrict__ token_row, const int* __restrict__ positions, Pages pages, unsigned char* __restrict__ k_pool,
              unsigned char* __restrict__ v_pool, long long page_stride, int planes, int n_kv_heads, int head_dim, int aligned) {
    pdl_prologue();
    k_src = pdl_fresh(k_src);
    v_src = pdl_fresh(v_src);
    const int groups = groups_of(head_dim), per_plane = n_kv_heads * groups * 4, t = blockIdx.x;
    const int index = blockIdx.y * blockDim.x + threadIdx.x;
    const bool there = index < planes * per_plane;                               // (the lanes of a group are there together)
    const int second = planes == 2 && index >= per_plane ? 1 : 0, inside = there ? index - second * per_plane : 0;
    const int plane = planes == 2 ? second : (k_src ? 0 : 1);
    const int p = positions[t], table_row = token_row[t];
    const int part = inside & 3, head = (inside >> 2) / groups, j = (inside >> 2) - head * groups;
    const int d = j * GROUP + part * 8;
    const int count = there ? min(8, head_dim - d) : 0;                          // numbers of this part that exist (may be negative)
    const T* src = (plane ? v_src + t * v_stride : k_src + t * k_stride) + (head * head_dim + d);
    float x[8], low = INFINITY, high = -INFINITY;
    bool bad = false;                                                            // (minimum and maximum pass NaN over)
    if (count == 8) {
        if (aligned) {
            Eight<T>::load(src, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = to_float(src[i]);
        }
        low = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), fminf(x[6], x[7]));
        high = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
        float zero = 0.f;                                                        // 0, or NaN where a number is one or an infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) zero = fmaf(x[i], 0.f, zero);
        bad = zero != 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = 0.f;
            if (i < count) {
                x[i] = to_float(src[i]);
                low = fminf(low, x[i]);
                high = fmaxf(high, x[i]);
                bad |= x[i] != x[i];
            }
        }
    }
    if (bad) low = -INFINITY;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const int page = pages.of(table_row, p);                                     // (looked up while the numbers are on their way)
    if (!there || page < 0) return;
    low = bf16_below(low);
    float step = bf16_above(__fdiv_rn(__fsub_rn(high, low), 15.0f));
    uint32_t word = 0;
    if (isfinite(low) && isfinite(step)) {
        if (count < 8)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= count) x[i] = low;                                       // (code 0)
        word = word_of(x, low, step);
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

// The words of some positions (k or v, head, place in the row) over the threads of a CTA, blockIdx.y = item. A word waits for four reads in a row (length,
// row, page, the word): in bfloat16 four positions share the wait (64 requests of 1,000, 12 heads of 64: 76 us with one, 55 with two, 45 with four; its floor
// is 21), in float32, whose stores take longer than it, one has more CTAs under way (5 of 1,023, 25 heads of 64: 14.0, 15.3, 16.6; floor 8). out: pages
// [n_items * span / out_page, 2, kv heads, out_page, head_dim], item i's position p in page i * span / out_page + p / out_page. Positions from kv_len on
// are left as they are; those without a page, too, or (`fill`) become zeros.
template <typename T> struct Positions { static constexpr int TOGETHER = sizeof(T) == 2 ? 4 : 1; };
template <typename T>
__global__ void __launch_bounds__(256)
unpack_kernel(const unsigned char* __restrict__ k_pool, const unsigned char* __restrict__ v_pool, long long page_stride,
              const int* __restrict__ kv_len, const int* __restrict__ item_row, Pages pages, int span, T* __restrict__ out, int out_log2,
              int n_kv_heads, int head_dim, int aligned, int fill) {
    pdl_prologue();
    k_pool = pdl_fresh(k_pool);
    v_pool = pdl_fresh(v_pool);
    const int groups = groups_of(head_dim), words = groups * 4, per_row = 2 * n_kv_heads * words;
    constexpr int TOGETHER = Positions<T>::TOGETHER;
    const int item = blockIdx.y, first = blockIdx.x * TOGETHER, length = kv_len[item], table_row = item_row ? item_row[item] : item;
    const int page_size = 1 << pages.page_log2, out_size = 1 << out_log2;
    if (first >= length) return;
    int page[TOGETHER];
#pragma unroll
    for (int u = 0; u < TOGETHER; ++u) page[u] = first + u < length && first + u < span ? pages.of(table_row, first + u) : -1;
    for (int index = threadIdx.x; index < per_row; index += blockDim.x) {
        const int both = index / words, place = index - both * words, plane = both >= n_kv_heads ? 1 : 0, head = both - plane * n_kv_heads;
        const int part = place / groups, j = place - part * groups, d = j * GROUP + part * 8, count = head_dim - d;
        const unsigned char* slabs = (plane ? v_pool : k_pool) + (long long)head * slab_bytes(page_size, head_dim);
        uint32_t word[TOGETHER], scale[TOGETHER];
#pragma unroll
        for (int u = 0; u < TOGETHER; ++u) {
            word[u] = scale[u] = 0u;
            if (page[u] >= 0) {
                const int row = first + u & (page_size - 1);
                const unsigned char* slab = slabs + (long long)page[u] * page_stride;
                word[u] = reinterpret_cast<const uint32_t*>(slab)[row * words + place];
                scale[u] = reinterpret_cast<const uint32_t*>(slab + page_size * groups * 16)[row * groups + j];
            }
        }
#pragma unroll
        for (int u = 0; u < TOGETHER; ++u) {
            const int p = first + u;
            if (p >= length || p >= span || (page[u] < 0 && !fill)) continue;
            const float step = step_of(scale[u]), low = low_of(scale[u]);
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf((float)((word[u] >> code_shift(i)) & 15u), step, low);
            const long long out_page = (long long)item * (span >> out_log2) + (p >> out_log2);
            T* to = out + (((out_page * 2 + plane) * n_kv_heads + head) * out_size + (p & (out_size - 1))) * head_dim + d;
            if (count >= 8 && aligned) {
                Eight<T>::store(to, x);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < count) to[i] = from_float<T>(x[i]);
            }
        }
    }
}

template <typename T>
int append(const void* k_src, long long k_stride, const void* v_src, long long v_stride, const int* token_row, const int* positions,
           const Pages& pages, void* k_pool, void* v_pool, long long page_stride, int tokens, int n_kv_heads, int head_dim, cudaStream_t s) {
    const int planes = (k_src ? 1 : 0) + (v_src ? 1 : 0);
    const long long parts = (long long)planes * n_kv_heads * groups_of(head_dim) * 4;
    const int threads = parts >= 256 ? 256 : (int)((parts + 31) / 32 * 32);
    if ((parts + threads - 1) / threads > 65535) return PS_ERR_UNSUPPORTED;
    constexpr int PER = 16 / (int)sizeof(T);
    const int aligned = !(((uintptr_t)k_src | (uintptr_t)v_src) & 15) && k_stride % PER == 0 && v_stride % PER == 0 && head_dim % 8 == 0;
    return launch_pdl(append_kernel<T>, dim3(tokens, (unsigned)((parts + threads - 1) / threads)), dim3(threads), 0, s, (const T*)k_src, k_stride,
                      (const T*)v_src, v_stride, token_row, positions, pages, (unsigned char*)k_pool, (unsigned char*)v_pool, page_stride, planes,
                      n_kv_heads, head_dim, aligned);
}

template <typename T>
int unpack(const void* k_pool, const void* v_pool, long long page_stride, const int* kv_len, const int* item_row, const Pages& pages, int n_items,
           int span, void* out, int out_page, int n_kv_heads, int head_dim, int fill, cudaStream_t s) {
    const long long words = (long long)2 * n_kv_heads * groups_of(head_dim) * 4;
    if (words > 0x7fffffff) return PS_ERR_UNSUPPORTED;
    const long long rounds = (words + 255) / 256;
    const int threads = (int)(((words + rounds - 1) / rounds + 31) / 32 * 32);         // (as many in the last round as in the others)
    const int aligned = !((uintptr_t)out & 15) && head_dim % 8 == 0;
    return launch_pdl(unpack_kernel<T>, dim3((span + Positions<T>::TOGETHER - 1) / Positions<T>::TOGETHER, n_items), dim3(threads), 0, s, (const unsigned char*)k_pool,
                      (const unsigned char*)v_pool, page_stride, kv_len, item_row, pages, span, (T*)out, log2_of(out_page), n_kv_heads, head_dim,
                      aligned, fill);
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

// kv_len / item_row: of the n_items items; span: positions that an item has room for in `out`, a multiple of out_page; fill: zeros where there is no page.
PS_EXPORT int ps_kv_unpack(const void* k_pool, const void* v_pool, int n_pages, long long page_stride, const int* kv_len, const int* block_table,
                           int bt_stride, const int* item_row, int n_items, int span, void* out, int out_page, int n_kv_heads, int head_dim,
                           int page_size, int dtype, int fill, void* stream) {
    using namespace ps::packed;
    if (n_items <= 0 || span <= 0) return PS_OK;
    if (!k_pool || !v_pool || !kv_len || !block_table || !out) return PS_ERR_BAD_ARGUMENT;
    if (!sizes_ok(n_kv_heads, head_dim, page_size) || n_items > 65535) return PS_ERR_UNSUPPORTED;
    if (out_page <= 0 || (out_page & (out_page - 1)) || span % out_page) return PS_ERR_BAD_ARGUMENT;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    const Pages pages = {block_table, bt_stride, n_pages, log2_of(page_size)};
    if (dtype == PS_F32)
        return unpack<float>(k_pool, v_pool, page_stride, kv_len, item_row, pages, n_items, span, out, out_page, n_kv_heads, head_dim, fill,
                             (cudaStream_t)stream);
    if (dtype == PS_BF16)
        return unpack<__nv_bfloat16>(k_pool, v_pool, page_stride, kv_len, item_row, pages, n_items, span, out, out_page, n_kv_heads, head_dim, fill,
                                     (cudaStream_t)stream);
    return PS_ERR_UNSUPPORTED;
}
