// Attention of single tokens over a cache held in 4 bits, on CUDA cores (packed.cuh has the cache's format): float32, and every
// head size up to 256.
//
// A key reads as low_j + step_j c in group j, so that
//   q . k = sum over j of step_j (q_j . c_j) + low_j sum(q_j)           (q_j, c_j: the numbers and codes of group j)
// and the weighted values are sum over keys of (p step_j) c + sum over keys of p low_j: a code is met by one multiply-add, the group's two numbers once a key.
// A code is put into the mantissa of a power of two (a value's into that of 16, by a rotation and a mask; two of a key's into those of 2^23, by a byte
// permutation each, for packed additions and multiply-adds) and moved to the middle of its range, c - 8, with low_j + 8 step_j in place of low_j:
// sums of 16 + c, eight times as large, cost the float32 results a digit (5 tokens, 512 keys, heads of 64: 2.4e-6 off, so 3e-7).  Scores, weights,
// sums: float32.
//
// A CTA has a token, a head (or two that share a key head, whose codes it then takes apart once) and a share of its keys: tiles of 32 keys aligned
// to absolute positions, one tile after another for each warp.  For the scores a lane has a key, for the values the numbers `lane` of every group.  The shares of a token and head are a
// thread-block cluster and merge through shared memory, in the order of the shares.
//
// What bounds it: instructions, two to four for every code of a key and of a value (5 tokens of up to 777 keys, the last 512 seen, 16
// heads of 64, capped scores, a sink: 7.6 us for 3.2 MB; 64 tokens of 1,024 keys, 12 heads of 64, 34), and for few
// tokens the chain of page, keys, weights and values of a tile: the values of 16 keys (2 groups a head) are on their way while the scores are formed (one
// token of 32,768 keys 56 us; with four at a time, asked for when they are due, 101).
#include "packed.cuh"

namespace ps {
namespace packed {

constexpr int WARPS = 4, TILE = 32;

// number i of a word as code - 8: `rotation` brings the code to bits 19 .. 22
__device__ __forceinline__ float centred(uint32_t word, int rotation) {
    return __uint_as_float((__funnelshift_l(word, word, rotation) & 0x00780000u) | 0x41800000u) - 24.f;
}
// bytes B and B + 2 of a word of codes, one a byte, as codes - 8: a byte put into the mantissa of 2^23, less 2^23 + 8
template <int B>
__device__ __forceinline__ unsigned long long centred_pair(uint32_t codes) {
    const float x = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7540 + B)), y = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7542 + B));
    return pair_add(pair_of(x, y), pair_of(-8388616.f, -8388616.f));
}

template <typename T, int NG, int R>
__global__ void __launch_bounds__(WARPS * 32)
tokens_kernel(const T* __restrict__ q, long long q_stride, void* __restrict__ out, long long out_stride, int wide,
              const unsigned char* __restrict__ k_pool, const unsigned char* __restrict__ v_pool, long long page_stride,
              const int* __restrict__ token_row, const int* __restrict__ positions, Pages pages, int n_heads, int n_kv_heads, int head_dim,
              int window, float scale, float softcap, const float* __restrict__ sink) {
    constexpr int NUMBERS = NG * GROUP, BATCH = NG * R <= 2 ? 16 : NG * R <= 4 ? 8 : 4;      // keys whose values are under way together
    __shared__ __align__(16) float q_s[R][NUMBERS];        // in the order of the cache's words
    __shared__ float sum_s[R * NG];                         // of each group's queries
    __shared__ __align__(16) float weight_s[WARPS][TILE][R * NG];
    __shared__ long long row_s[WARPS][TILE];
    __shared__ float acc_s[WARPS][R * NUMBERS], m_s[WARPS][R], l_s[WARPS][R];
    __shared__ float share_acc[R * NUMBERS], share_ml[R][2];
    pdl_prologue();
    q = pdl_fresh(q);
    k_pool = pdl_fresh(k_pool);
    v_pool = pdl_fresh(v_pool);
    const int ratio = n_heads / n_kv_heads, blocks = (ratio + R - 1) / R;
    const int t = blockIdx.x, g = blockIdx.y / blocks, first = blockIdx.y % blocks * R, share = blockIdx.z, shares = gridDim.z;
    const int h = g * ratio + first, heads = min(R, ratio - first);            // (what there is of R heads)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int p = positions[t], lo = p < 0 ? 0 : first_visible_key(p, window), table_row = token_row[t];
    const int last = min(p, (pages.bt_stride << pages.page_log2) - 1);          // (what is beyond the table has no page)
    for (int n = threadIdx.x; n < R * NUMBERS; n += WARPS * 32) {
        const int r = n / NUMBERS, i = n % NUMBERS, place = i >> 3, d = place % NG * GROUP + place / NG * 8 + (i & 7);
        q_s[r][i] = r < heads && d < head_dim ? to_float(q[t * q_stride + (h + r) * head_dim + d]) : 0.f;
    }
    __syncthreads();
    if (threadIdx.x < R * NG) {
        const int r = threadIdx.x / NG, j = threadIdx.x % NG;
        float sum = 0.f;
        for (int i = 0; i < NUMBERS; ++i)
            if ((i >> 3) % NG == j) sum += q_s[r][i];
        sum_s[threadIdx.x] = sum;
    }
    __syncthreads();
    float q_sum[R][NG];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NG; ++j) q_sum[r][j] = sum_s[r * NG + j];

    const int page_size = 1 << pages.page_log2, words_at = page_size * NG * 16;
    const long long head_at = (long long)g * slab_bytes(page_size, head_dim);
    const float scale_log2 = scale * 1.4426950408889634f;
    float m[R], l[R], acc[R][NG], lows[R][NG];             // acc: number `lane` of every group; l and lows: this lane's keys
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int j = 0; j < NG; ++j) acc[r][j] = lows[r][j] = 0.f;
    }
    const int my_rotation = (19 - code_shift(lane & 7)) & 31, my_part = lane >> 3;
    // (a key's entry of the block table is asked for a tile before, and not looked at until then: a comparison would wait for it)
    const int* table = pages.block_table + (size_t)table_row * pages.bt_stride;
    auto entry_of = [&](int tile) {
        const int key = tile * TILE + lane;
        return key >= lo && key <= last ? table[key >> pages.page_log2] : -1;
    };
    const int first_tile = lo / TILE + share * WARPS + warp;
    int entry = entry_of(first_tile);
    for (int tile = first_tile; tile * TILE <= last; tile += shares * WARPS) {
        const int key = tile * TILE + lane, page = entry < pages.n_pages ? entry : -1;
        entry = entry_of(tile + shares * WARPS);
        const long long at = page < 0 ? -1 : (long long)page * page_stride + head_at;
        const int row = key & (page_size - 1);
        // the values' words of the first keys, which the scores do not wait for
        __syncwarp();                                          // (the last tile's rows and weights are done with)
        row_s[warp][lane] = page < 0 ? -1 : at + row * NG * 16;
        __syncwarp();
        uint32_t value[BATCH][NG];
        auto load_values = [&](int k0) {
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const long long from = row_s[warp][k0 + k];
#pragma unroll
                for (int j = 0; j < NG; ++j) value[k][j] = from < 0 ? 0u : reinterpret_cast<const uint32_t*>(v_pool + from)[my_part * NG + j];
            }
        };
        load_values(0);
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = -INFINITY;
        if (page >= 0) {
            const uint4* codes = reinterpret_cast<const uint4*>(k_pool + at) + row * NG;
            const uint32_t* words = reinterpret_cast<const uint32_t*>(k_pool + at + words_at) + row * NG;
            unsigned long long dot[R][NG];                         // sums over even and over odd numbers
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int j = 0; j < NG; ++j) dot[r][j] = 0ull;
#pragma unroll
            for (int u = 0; u < NG; ++u) {
                const uint4 raw = codes[u];
                const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int place = u * 4 + w;
                    const uint32_t low = word[w] & 0x0f0f0f0fu, high = word[w] >> 4 & 0x0f0f0f0fu;       // numbers 0, 4, 1, 5 and 2, 6, 3, 7
                    const unsigned long long c0 = centred_pair<0>(low), c1 = centred_pair<0>(high), c2 = centred_pair<1>(low), c3 = centred_pair<1>(high);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(q_s[r] + place * 8), b = *reinterpret_cast<const ulonglong2*>(q_s[r] + place * 8 + 4);
                        dot[r][place % NG] = pair_fma(c3, b.y, pair_fma(c2, b.x, pair_fma(c1, a.y, pair_fma(c0, a.x, dot[r][place % NG]))));
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const uint32_t two = words[j];
                    float even, odd;
                    pair_split(dot[r][j], even, odd);
                    sum = fmaf(step_of(two), even + odd, fmaf(fmaf(8.f, step_of(two), low_of(two)), q_sum[r][j], sum));
                }
                s[r] = softcap > 0.f ? softcap * 1.4426950408889634f * tanhf(sum * (scale / softcap)) : sum * scale_log2;
            }
        }
        float shrink[R], weight[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float m_new = fmaxf(m[r], warp_max(s[r])), base = m_new == -INFINITY ? 0.f : m_new;
            shrink[r] = exp2f(m[r] - base);
            m[r] = m_new;
            weight[r] = page >= 0 ? exp2f(s[r] - base) : 0.f;
            l[r] = fmaf(l[r], shrink[r], weight[r]);
        }
        const uint32_t* words = reinterpret_cast<const uint32_t*>(v_pool + (page >= 0 ? at + words_at : 0)) + (page >= 0 ? row * NG : 0);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t two = page >= 0 ? words[j] : 0u;                       // (no page: weights of zero, and steps)
            const float step = step_of(two), middle = fmaf(8.f, step, low_of(two));
#pragma unroll
            for (int r = 0; r < R; ++r) {
                weight_s[warp][lane][r * NG + j] = weight[r] * step;
                lows[r][j] = fmaf(lows[r][j], shrink[r], weight[r] * middle);
                acc[r][j] *= shrink[r];
            }
        }
        __syncwarp();
#pragma unroll 1
        for (int k0 = 0; k0 < TILE; k0 += BATCH) {
            float number[BATCH][NG];
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
#pragma unroll
                for (int j = 0; j < NG; ++j) number[k][j] = centred(value[k][j], my_rotation);
            if (k0 + BATCH < TILE) load_values(k0 + BATCH);
#pragma unroll
            for (int k = 0; k < BATCH; ++k)
#pragma unroll
                for (int j = 0; j < NG; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][j] = fmaf(number[k][j], weight_s[warp][k0 + k][r * NG + j], acc[r][j]);
        }
    }
    // the warps' states, then the shares'
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = warp_sum(l[r]);
#pragma unroll
        for (int j = 0; j < NG; ++j) acc_s[warp][r * NUMBERS + j * GROUP + lane] = acc[r][j] + warp_sum(lows[r][j]);
        if (lane == 0) { m_s[warp][r] = m[r]; l_s[warp][r] = sum; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * NUMBERS; i += WARPS * 32) {
        const int r = i / NUMBERS;
        float top = -INFINITY, sum = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, m_s[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float by = exp2f(m_s[w][r] - base);
            total = fmaf(l_s[w][r], by, total);
            sum = fmaf(acc_s[w][i], by, sum);
        }
        share_acc[i] = sum;
        if (i % NUMBERS == 0) { share_ml[r][0] = top; share_ml[r][1] = total; }
    }
    if (shares > 1) cluster_sync_all();
    else __syncthreads();
    if (share == 0) {
        for (int i = threadIdx.x; i < heads * NUMBERS; i += WARPS * 32) {
            const int r = i / NUMBERS, d = i % NUMBERS;
            if (d >= head_dim) continue;
            const float sink_log2 = sink ? sink[h + r] * 1.4426950408889634f : -INFINITY;
            float all = sink_log2;
            for (int c = 0; c < shares; ++c) all = fmaxf(all, shares > 1 ? ld_cluster_f32(&share_ml[r][0], c) : share_ml[r][0]);
            const float ground = all == -INFINITY ? 0.f : all;
            float denominator = sink ? exp2f(sink_log2 - ground) : 0.f, sum = 0.f;
            for (int c = 0; c < shares; ++c) {
                const float by = exp2f((shares > 1 ? ld_cluster_f32(&share_ml[r][0], c) : share_ml[r][0]) - ground);
                denominator = fmaf(shares > 1 ? ld_cluster_f32(&share_ml[r][1], c) : share_ml[r][1], by, denominator);
                sum = fmaf(shares > 1 ? ld_cluster_f32(&share_acc[i], c) : share_acc[i], by, sum);
            }
            // (no key at all: zero; a NaN stays one)
            const float result = denominator == 0.f ? sum * 0.f : sum / denominator;
            const long long to = t * out_stride + (long long)(h + r) * head_dim + d;
            if (wide) reinterpret_cast<float*>(out)[to] = result;
            else reinterpret_cast<T*>(out)[to] = from_float<T>(result);
        }
    }
    if (shares > 1) cluster_sync_all();                     // the shares stay until they were read
}

template <typename T, int NG, int R>
int launch_tokens(const void* q, long long q_stride, void* out, long long out_stride, int wide, const void* k_pool, const void* v_pool,
                  long long page_stride, const int* token_row, const int* positions, const Pages& pages, int tokens, int n_heads, int n_kv_heads,
                  int head_dim, int window, float scale, float softcap, const float* sink, int shares, cudaStream_t s) {
    return launch_pdl_cluster(tokens_kernel<T, NG, R>, dim3(tokens, n_kv_heads * ((n_heads / n_kv_heads + R - 1) / R), shares),
                              dim3(WARPS * 32), 0, s, shares, (const T*)q, q_stride, out, out_stride, wide, (const unsigned char*)k_pool, (const unsigned char*)v_pool, page_stride, token_row, positions, pages,
                              n_heads, n_kv_heads, head_dim, window, scale, softcap, sink);
}

}  // namespace packed
}  // namespace ps

// q / out: rows of n_heads * head_dim numbers; token t stands at positions[t] (below 0: its row of `out` becomes zero) and reads the pages of
// row token_row[t] of block_table (bt_stride wide; what has no page is not seen).  window, softcap, sink as in ps_paged_attention_simt.
// out_dtype: that of q, or float32.  shares: 1, 2, 4 or 8 CTAs for the keys of a token and head.  together: 1, or (heads of up to 128) 2 query heads
// of a key head in a CTA.
PS_EXPORT int ps_packed_tokens_simt(const void* q, long long q_stride, void* out, long long out_stride, int out_dtype, const void* k_pool,
                                    const void* v_pool, int n_pages, long long page_stride, const int* token_row, const int* positions,
                                    const int* block_table, int bt_stride, int tokens, int n_heads, int n_kv_heads, int head_dim, int page_size,
                                    int window, float scale, float softcap, const float* sink, int shares, int together, int dtype, void* stream) {
    using namespace ps::packed;
    if (tokens <= 0) return PS_OK;
    if (!q || !out || !k_pool || !v_pool || !token_row || !positions || !block_table) return PS_ERR_BAD_ARGUMENT;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return PS_ERR_BAD_ARGUMENT;
    if (!sizes_ok(n_kv_heads, head_dim, page_size) || n_heads > 65535) return PS_ERR_UNSUPPORTED;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    if (shares != 1 && shares != 2 && shares != 4 && shares != 8) return PS_ERR_BAD_ARGUMENT;
    if ((dtype != PS_F32 && dtype != PS_BF16) || (out_dtype != dtype && out_dtype != PS_F32)) return PS_ERR_UNSUPPORTED;
    if ((together != 1 && together != 2) || (together > 1 && head_dim > 128)) return PS_ERR_BAD_ARGUMENT;
    if (dtype == PS_BF16 && head_dim <= 128) return PS_ERR_UNSUPPORTED;           // (ps_packed_tokens_mma)
    const Pages pages = {block_table, bt_stride, n_pages, log2_of(page_size)};
    const int wide = dtype == PS_BF16 && out_dtype == PS_F32;
#define PS_PACKED_TOKENS(T, NG, R)                                                                                                             \
    return launch_tokens<T, NG, R>(q, q_stride, out, out_stride, wide, k_pool, v_pool, page_stride, token_row, positions, pages, tokens, n_heads, \
                                   n_kv_heads, head_dim, window, scale, softcap, sink, shares, (cudaStream_t)stream)
#define PS_PACKED_TOKENS_F32(NG)                                     \
    case NG:                                                         \
        if (together == 2) PS_PACKED_TOKENS(float, NG, 2);           \
        PS_PACKED_TOKENS(float, NG, 1)
#define PS_PACKED_TOKENS_BOTH(NG)                                    \
    case NG:                                                         \
        if (dtype == PS_F32) PS_PACKED_TOKENS(float, NG, 1);         \
        PS_PACKED_TOKENS(__nv_bfloat16, NG, 1)
    switch (groups_of(head_dim)) {
        PS_PACKED_TOKENS_F32(1);
        PS_PACKED_TOKENS_F32(2);
        PS_PACKED_TOKENS_F32(3);
        PS_PACKED_TOKENS_F32(4);
        PS_PACKED_TOKENS_BOTH(5);
        PS_PACKED_TOKENS_BOTH(6);
        PS_PACKED_TOKENS_BOTH(7);
        PS_PACKED_TOKENS_BOTH(8);
    }
#undef PS_PACKED_TOKENS_BOTH
#undef PS_PACKED_TOKENS_F32
#undef PS_PACKED_TOKENS
    return PS_ERR_UNSUPPORTED;
}
