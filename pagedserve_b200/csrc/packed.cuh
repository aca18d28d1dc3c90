// Keys and values held in 4 bits: the format of a cached row, and the steps that the kernels over it share.
//
// A row of one key/value head (head_dim numbers, at most 256) is cut into groups of 32; the last one may be short. A group keeps
//   low   its minimum, rounded down to bfloat16,
//   step  (maximum - low) / 15, rounded up to bfloat16,
//   16 bytes of codes, code = (x - low) / step rounded to the nearest whole number (ties to even), 0 where step is 0,
// and reads as low + code * step, which is within step / 2 of x. Rounding low down and step up keeps the whole group between codes 0
// and 15. A group with a NaN or an infinity, or whose range passes float32's, has NaN for step and low and reads as NaN throughout.
//
// A page of a head ("slab") holds the codes of its page_size rows, 16 bytes a group, then a word a group, row by row (step in the lower
// half, low in the upper one), and is rounded up to 16 bytes. The eight numbers 8t .. 8t + 7 of group j (of n) are one word, at place
// t * n + j of the row: the four lanes of an mma.sync quad that share a row of a fragment then find a part of every group each, side
// by side. Within the word the lower four codes are the numbers 0, 2, 4, 6, the upper four 1, 3, 5, 7: a mask of one code in either half gives two
// neighbouring numbers at once.
#pragma once

#include "common.cuh"

namespace ps {
namespace packed {

constexpr int GROUP = 32, MAX_HEAD = 256;

__host__ __device__ __forceinline__ int groups_of(int head_dim) { return (head_dim + GROUP - 1) / GROUP; }
__host__ __device__ __forceinline__ int slab_bytes(int page_size, int head_dim) {
    return (page_size * groups_of(head_dim) * 20 + 15) / 16 * 16;
}
// the code of number i (of 8) of a word starts at this bit
__host__ __device__ __forceinline__ int code_shift(int i) { return ((i >> 1) + ((i & 1) << 2)) * 4; }

__device__ __forceinline__ float step_of(uint32_t word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float low_of(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

// the bfloat16 number at or below x, and at or above it, as float32 (a NaN stays one; what passes the range becomes an infinity)
__device__ __forceinline__ float bf16_below(float x) {
    const uint32_t bits = __float_as_uint(x), cut = bits & 0xffff0000u;
    return __uint_as_float(cut + ((bits != cut && (bits >> 31)) ? 0x10000u : 0u));
}
__device__ __forceinline__ float bf16_above(float x) { return -bf16_below(-x); }

// The place of a token's row: its page, checked against the table's width and the pool's pages; -1: nowhere.
struct Pages {
    const int* block_table;
    int bt_stride;            // the table's width, too
    int n_pages;
    int page_log2;
    __device__ __forceinline__ int of(int row, int position) const {
        if (position < 0 || (position >> page_log2) >= bt_stride) return -1;
        const int page = block_table[(size_t)row * bt_stride + (position >> page_log2)];
        return page < n_pages ? page : -1;
    }
};

struct Cache {
    const unsigned char* k_pool;
    const unsigned char* v_pool;
    long long page_stride;
    Pages pages;
};

// One bfloat16 query against the keys that position p sees, in float32 from the codes, for kernels whose float16 operands do not hold them: lane l of the warp has
// number 32 j + l of every group (heads of up to 128), key after key. `out` from `to` on: bfloat16, or float32 where `wide`; `sink`: null, or the head's. Slow: a key is
// a chain of page, codes and score (about 0.4 us).
template <typename T>
__device__ __noinline__ void row_again(const T* q, void* out, long long to, int wide, const Cache cache, int table_row, long long head_at, int head_dim, int p,
                                       int window, float scale, float softcap, const float* sink, int lane) {
    const int groups = groups_of(head_dim), page_size = 1 << cache.pages.page_log2, shift = code_shift(lane & 7);
    const int last = min(p, (cache.pages.bt_stride << cache.pages.page_log2) - 1);
    float x[4], acc[4], m = -INFINITY, l = 0.f;
    if (sink) {
        m = *sink;
        l = 1.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = j * GROUP + lane;
        x[j] = d < head_dim ? to_float(q[d]) : 0.f;
        acc[j] = 0.f;
    }
    for (int key = p < 0 ? 0 : first_visible_key(p, window); key <= last; ++key) {
        const int page = cache.pages.of(table_row, key);
        if (page < 0) continue;
        const long long at = (long long)page * cache.page_stride + head_at;
        const int row = key & (page_size - 1);
        float s = 0.f, v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = 0.f;
            if (j < groups) {
                const int word = (row * 4 + (lane >> 3)) * groups + j, scale_at = page_size * groups * 4 + row * groups + j;
                const uint32_t *k = reinterpret_cast<const uint32_t*>(cache.k_pool + at), *w = reinterpret_cast<const uint32_t*>(cache.v_pool + at);
                const bool there = j * GROUP + lane < head_dim;                // (a number that is not there has no code)
                if (there) s = fmaf(fmaf((float)(k[word] >> shift & 15u), step_of(k[scale_at]), low_of(k[scale_at])), x[j], s);
                v[j] = fmaf((float)(w[word] >> shift & 15u), step_of(w[scale_at]), low_of(w[scale_at]));
            }
        }
        s = warp_sum(s) * scale;
        if (softcap > 0.f) s = softcap * tanhf(s / softcap);
        const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top, shrink = expf(m - base), w = expf(s - base);
        m = top;
        l = fmaf(l, shrink, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(acc[j], shrink, w * v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = j * GROUP + lane;
        const float result = l == 0.f ? acc[j] * 0.f : acc[j] / l;             // (no key at all: zero; a NaN stays one)
        if (d < head_dim) {
            if (wide) reinterpret_cast<float*>(out)[to + d] = result;
            else reinterpret_cast<T*>(out)[to + d] = from_float<T>(result);
        }
    }
}

inline bool sizes_ok(int n_kv_heads, int head_dim, int page_size) {
    return n_kv_heads > 0 && head_dim > 0 && head_dim <= MAX_HEAD && page_size > 0 && page_size <= 64 && !(page_size & (page_size - 1));
}
inline int log2_of(int page_size) { return 31 - __builtin_clz(page_size); }

}  // namespace packed
}  // namespace ps
