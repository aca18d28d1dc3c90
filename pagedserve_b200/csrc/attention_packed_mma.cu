// Attention of single tokens over a cache held in 4 bits on mma.sync, bfloat16 queries, head sizes up to 128 (packed.cuh has the format).
//
// The codes go to the tensor cores as they are, whole numbers in float16, and the groups' numbers are met by the scores and weights:
//   S_j = C_j q_j                              keys x queries, for each group j: mma.sync with the keys on the 16-row side, the query heads that
//                                              share the key head as its 8 columns
//   s   = sum over j of step_j S_j + low_j sum(q_j)
//   O_j = (C_j - 8)^T (p step_j)               numbers x queries: again on the 16-row side; the weights turn from the first product's result
//   o   = O_j + sum over keys of p (low_j + 8 step_j)             into the second's operand by movmatrix
// so that keys and values are met without a rounding; a weight times its step is rounded to float16 (2^-11 of itself).
//   * A mask puts two codes into float16 at once: bits 4 .. 7 of a half word under the exponent of 64 are 64 + c; bits 0 .. 3 under that of 1024 are
//     1024 + c. Keys take the first form (a shift a code), with low_j - 64 step_j in place of low_j; values take both, and one subtraction leaves
//     c - 8: their sums are long, and what 1024 p costs in float32 would show.
//   * Queries are scaled by a power of two to at most 512, which leaves a bfloat16 number as it is, or within 2^-33 of its row's largest.
//   * p step_j is at most 2^15: p is taken relative to the largest score so far, step_j to the exponent of the group's largest one less 5. Either moves only when a
//     score passes the former by 2^8 or a step the latter's power of two, so that hardly a tile pays for it. A product is then held to 2^-11 of itself or to 2^-30
//     of that of a weight of 1 and the largest step.
//   * A step other than zero below 2^-19 of the largest so far (its weight may be all there is, and float16 has no digits for it), or a group of a query below 2^-17
//     of its row: the token's heads are done again in float32 (row_again in packed.cuh), which is slow and right.
//
// A CTA has a token, a key head (8 or 16 of its query heads) and a share of the keys; a warp takes tiles of 16 keys, which it brings to shared
// memory itself (cp.async, a ring of its own, no barrier). Shares are a cluster and merge through shared memory.
//
// What bounds it: instructions, not bytes (the same time with one page that every token shares). A tile of 16 keys is about 640 instructions a warp at
// 128 numbers a head and 8 queries, half of them masks, shifts and sums on the ALU pipe, which issues every other clock (59 % of its slots on average, 73 % on the
// busiest SM; 63 % of all issue slots: a warp's own chain of scores, weights and products leaves the rest idle); its 32 mma.sync are not felt. 64 tokens of 4,099
// keys, 32 heads on 8 of 128: 103 us, 2.3 TB/s; 64 x 1,024, 12 heads of 64: 29 us; one token of 32,768: 26 us, 12 heads by 8 shares of 8 warps on 148 SMs. A
// page's number is asked for a tile before it is used and not compared until then, or its latency stands in the loop (110 us; one token 46, so 36 with 4 warps). A token
// that is done again takes 60 us for 129 keys and 480 for 1,024.
#include "packed.cuh"

namespace ps {
namespace packed {

constexpr int M_KEYS = 16;
constexpr float HEADROOM = 8.f;                            // log2 of how far a weight may be beyond 1 before its base moves
constexpr int LIFT = 5;                                    // log2 of what products of weights and steps are multiplied by
constexpr float LEAST_FACTOR = 6.103515625e-05f;           // 2^-14, float16's least number of eleven digits: a smaller factor of a step is not taken
constexpr int LEAST_EXPONENT = 27, MOST_EXPONENT = 253;    // biased: steps below 2^-100 count as that, those from 2^126 on (up to 4 of it)

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same on a sum that starts at zero
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t half_add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// two codes of a word as float16: 64 + c from bits 4 .. 7 of its halves, 1024 + c from bits 0 .. 3
__device__ __forceinline__ uint32_t sixty_four_plus(uint32_t x) { return (x & 0x00f000f0u) | 0x54005400u; }
__device__ __forceinline__ uint32_t thousand_plus(uint32_t x) { return (x & 0x000f000fu) | 0x64006400u; }
constexpr uint32_t LESS_72 = 0xd480d480u, LESS_1032 = 0xe408e408u;      // -72 and -1032 twice

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// NG words side by side
template <int NG>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[NG]) {
    if constexpr (NG == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int j = 0; j < NG; ++j) w[j] = reinterpret_cast<const uint32_t*>(p)[j];
    }
}

// a tile in the ring: codes of 16 keys, codes of 16 values, their scales
template <int NG, int M_WARPS>
struct Ring {
    static constexpr int CODES = M_KEYS * NG * 16, SCALES = M_KEYS * NG * 4, TILE_BYTES = 2 * (CODES + SCALES);
    static constexpr int STAGES = NG <= 2 ? 4 : 3;
    static constexpr int BYTES = M_WARPS * STAGES * TILE_BYTES;
};

template <int NG, int NQ, int M_WARPS>
__global__ void __launch_bounds__(M_WARPS * 32, (NG * NQ <= 4 ? 4 : 2) * 4 / M_WARPS)
tokens_mma_kernel(const __nv_bfloat16* __restrict__ q, long long q_stride, void* __restrict__ out, long long out_stride, int wide,
                  const unsigned char* __restrict__ k_pool, const unsigned char* __restrict__ v_pool, long long page_stride,
                  const int* __restrict__ token_row, const int* __restrict__ positions, Pages pages, int n_heads, int n_kv_heads, int head_dim,
                  int window, float scale, float softcap, const float* __restrict__ sink, int aligned) {
    using R = Ring<NG, M_WARPS>;
    constexpr int COLUMNS = 8 * NQ, NUMBERS = NG * GROUP;
    extern __shared__ __align__(16) unsigned char memory[];
    __shared__ float base_s[M_WARPS][COLUMNS], sum_s[M_WARPS][COLUMNS], share_base[COLUMNS], share_sum[COLUMNS];
    pdl_prologue();
    const __nv_bfloat16* queries = pdl_fresh(q);
    k_pool = pdl_fresh(k_pool);
    v_pool = pdl_fresh(v_pool);
    const int ratio = n_heads / n_kv_heads, blocks = (ratio + COLUMNS - 1) / COLUMNS;
    const int t = blockIdx.x, kv_head = blockIdx.y / blocks, first_query = blockIdx.y % blocks * COLUMNS, share = blockIdx.z, shares = gridDim.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int p = positions[t], lo = p < 0 ? 0 : first_visible_key(p, window), table_row = token_row[t];
    const int last = min(p, (pages.bt_stride << pages.page_log2) - 1);          // (what is beyond the table has no page)
    const int page_size = 1 << pages.page_log2;
    const long long head_at = (long long)kv_head * slab_bytes(page_size, head_dim);
    unsigned char* ring = memory + warp * R::STAGES * R::TILE_BYTES;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const bool by_tile = pages.page_log2 >= 4;                                   // a tile lies in one page

    // ---- a tile's bytes on their way. What is not visible or has no page is left as the ring holds it: its scales are not used.
    const int step_tiles = shares * M_WARPS;
    int tile = lo / M_KEYS + share * M_WARPS + warp;
    uint32_t paged = 0;                                                          // (by_tile) the stages whose tile has a page
    // (a tile's page is asked for a tile before, and not looked at until then: a comparison here would wait for it)
    const int* table = pages.block_table + (size_t)table_row * pages.bt_stride;
    auto page_of = [&](int which) { return by_tile && which * M_KEYS <= last ? table[which * M_KEYS >> pages.page_log2] : -1; };
    int next_page = page_of(tile);
    auto fetch = [&](int which, int stage) {
        const int key0 = which * M_KEYS, page = next_page < pages.n_pages ? next_page : -1;
        next_page = page_of(which + step_tiles);
        paged &= ~(1u << stage);
        if (key0 <= last) {
            const uint32_t to = ring_at + stage * R::TILE_BYTES;
            if (by_tile) {
                if (page >= 0) {
                    paged |= 1u << stage;
                    const long long at = (long long)page * page_stride + head_at;
                    const int row = key0 & (page_size - 1);
                    const unsigned char *k = k_pool + at, *v = v_pool + at;
#pragma unroll
                    for (int i = lane; i < M_KEYS * NG; i += 32) {
                        copy16(to + i * 16, k + (row * NG + i) * 16);
                        copy16(to + R::CODES + i * 16, v + (row * NG + i) * 16);
                    }
#pragma unroll
                    for (int i = lane; i < 8 * NG; i += 32) {
                        const int plane = i / (4 * NG), piece = i % (4 * NG);
                        copy16(to + 2 * R::CODES + i * 16, (plane ? v : k) + page_size * NG * 16 + row * NG * 4 + piece * 16);
                    }
                }
            } else {
#pragma unroll
                for (int i = lane; i < M_KEYS * NG; i += 32) {
                    const int key = key0 + i / NG, part = i % NG, own = key <= last ? pages.of(table_row, key) : -1;
                    if (own >= 0) {
                        const long long at = (long long)own * page_stride + head_at;
                        const int row = key & (page_size - 1);
                        const unsigned char *k = k_pool + at, *v = v_pool + at;
                        copy16(to + i * 16, k + (row * NG + part) * 16);
                        copy16(to + R::CODES + i * 16, v + (row * NG + part) * 16);
                        copy4(to + 2 * R::CODES + i * 4, k + page_size * NG * 16 + (row * NG + part) * 4);
                        copy4(to + 2 * R::CODES + R::SCALES + i * 4, v + page_size * NG * 16 + (row * NG + part) * 4);
                    }
                }
            }
        }
        copies_commit();
    };
#pragma unroll
    for (int s = 0; s < R::STAGES - 1; ++s) {
        fetch(tile + s * step_tiles, s);
    }

    // ---- queries: column g of every block of eight, numbers 32 j + 8 c .. + 7, scaled to float16
    uint32_t qf[NQ][NG][4];
    float q_sum[NQ][NG][2], factor[NQ][2];                      // of columns 2 c and 2 c + 1: what this thread's scores belong to
    uint32_t least = 0xffffffffu;                                // the smallest factor of a step other than 0, as bits
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int column = first_query + n * 8 + g;
        const __nv_bfloat16* row = queries + t * q_stride + ((long long)kv_head * ratio + column) * head_dim;
        float x[NG][8], part_largest[NG], largest = 0.f;
        bool strange = false;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int d = j * GROUP + c * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
            if (column < ratio && d < head_dim) {
                if (aligned) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(row + d);
                    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[j][2 * i] = __uint_as_float(w[i] << 16);
                        x[j][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (d + i < head_dim) x[j][i] = __bfloat162float(row[d + i]);
                }
            }
            part_largest[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                part_largest[j] = fmaxf(part_largest[j], fabsf(x[j][i]));
                strange |= !(fabsf(x[j][i]) <= 3.4028235e38f);
            }
            largest = fmaxf(largest, part_largest[j]);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            strange |= __shfl_xor_sync(0xffffffffu, (int)strange, o) != 0;
        }
#pragma unroll
        for (int j = 0; j < NG; ++j)
            if (part_largest[j] > 0.f && part_largest[j] < largest * 0x1p-17f && !strange) least = 0u;
        // 2^up brings the largest to [256, 512); a NaN or infinity stays one; (exponents from 1: below are denormals, which may as well stay small)
        int up = largest > 0.f && !strange ? 135 - max(1, (int)(__float_as_uint(largest) >> 23)) : 0;
        up = min(up, 126);
        const float by = __uint_as_float((uint32_t)(127 + up) << 23);
        float back = __uint_as_float((uint32_t)(127 - up) << 23);                 // (up from -119 to 126)
        float sums[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            sums[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[j][i] *= by;
                sums[j] += x[j][i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[n][j][i] = half_pair(x[j][2 * i], x[j][2 * i + 1]);
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], o);
        }
        const float unit = softcap > 0.f ? scale / softcap : scale * 1.4426950408889634f;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int from = (2 * c + b) * 4;                                     // a lane of column 2 c + b
            factor[n][b] = __shfl_sync(0xffffffffu, back, from) * unit;
#pragma unroll
            for (int j = 0; j < NG; ++j) q_sum[n][j][b] = __shfl_sync(0xffffffffu, sums[j], from);
        }
    }
    const float cap_log2 = softcap > 0.f ? softcap * 1.4426950408889634f : 0.f;

    float base[NQ][2], limit[NQ][2], l[NQ][2], lows[NQ][NG][2], o[NQ][NG][2][4];
    float unit_step[NG];                                         // 2^LIFT over the power of two of each group's largest step so far: what o is multiplied by
    auto reciprocal = [](int biased) { return __uint_as_float((uint32_t)(254 + LIFT - biased) << 23); };
#pragma unroll
    for (int j = 0; j < NG; ++j) unit_step[j] = reciprocal(LEAST_EXPONENT);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            limit[n][b] = -INFINITY;                             // what a score may reach before the base of the weights moves
            base[n][b] = l[n][b] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            lows[n][j][0] = lows[n][j][1] = 0.f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][j][b][i] = 0.f;
        }
    }
    // The keys of a tile stand in the fragments in this order, in which four rows of keys and four of values lie in different banks.
    const int row_a = g ^ (g >> 2 & 1), row_v = 2 * c ^ (c >> 1), row_w = (2 * c + 1) ^ (c >> 1);
    const uint32_t half_of = g < 4 ? 0x5410u : 0x7632u;

    int stage = 0;
    for (; tile * M_KEYS <= last; tile += step_tiles) {
        copies_wait<R::STAGES - 2>();
        __syncwarp();
        const bool whole = by_tile && (paged >> stage & 1u);
        fetch(tile + (R::STAGES - 1) * step_tiles, stage == 0 ? R::STAGES - 1 : stage - 1);      // (the stage that the last tile was in)
        const unsigned char* at = ring + stage * R::TILE_BYTES;
        stage = stage + 1 == R::STAGES ? 0 : stage + 1;
        const int key_a = tile * M_KEYS + row_a, key_b = key_a + 8;
        const bool full = whole && tile * M_KEYS >= lo && tile * M_KEYS + M_KEYS - 1 <= last;      // every key is seen
        bool seen_a = true, seen_b = true;
        if (!full) {
            seen_a = key_a >= lo && key_a <= last && (whole || (!by_tile && pages.of(table_row, key_a) >= 0));
            seen_b = key_b >= lo && key_b <= last && (whole || (!by_tile && pages.of(table_row, key_b) >= 0));
        }
        // ---- scores
        float s[NQ][4];
        {
            uint32_t wa[NG], wb[NG], za[NG], zb[NG];
            load_words<NG>(at + row_a * NG * 16 + c * NG * 4, wa);
            load_words<NG>(at + (row_a + 8) * NG * 16 + c * NG * 4, wb);
            load_words<NG>(at + 2 * R::CODES + row_a * NG * 4, za);
            load_words<NG>(at + 2 * R::CODES + (row_a + 8) * NG * 4, zb);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const uint32_t a0 = sixty_four_plus(wa[j] << 4), a2 = sixty_four_plus(wa[j]), a4 = sixty_four_plus(wa[j] >> 4),
                               a6 = sixty_four_plus(wa[j] >> 8);
                const uint32_t a1 = sixty_four_plus(wb[j] << 4), a3 = sixty_four_plus(wb[j]), a5 = sixty_four_plus(wb[j] >> 4),
                               a7 = sixty_four_plus(wb[j] >> 8);
                const float step_a = step_of(za[j]), step_b = step_of(zb[j]);
                const float low_a = fmaf(-64.f, step_a, low_of(za[j])), low_b = fmaf(-64.f, step_b, low_of(zb[j]));
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    float dot[4];
                    mma_f16_first(dot, a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
                    mma_f16(dot, a4, a5, a6, a7, qf[n][j][2], qf[n][j][3]);
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        s[n][b] = fmaf(step_a, dot[b], fmaf(low_a, q_sum[n][j][b], s[n][b]));
                        s[n][2 + b] = fmaf(step_b, dot[2 + b], fmaf(low_b, q_sum[n][j][b], s[n][2 + b]));
                    }
                }
            }
        }
        uint32_t za[NG], zb[NG];                                  // the values' scales; zero where there is no value
        load_words<NG>(at + 2 * R::CODES + R::SCALES + row_a * NG * 4, za);
        load_words<NG>(at + 2 * R::CODES + R::SCALES + (row_a + 8) * NG * 4, zb);
        bool moves = false;
        if (!full)
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                if (!seen_a) za[j] = 0u;
                if (!seen_b) zb[j] = 0u;
            }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            moves |= fmaxf(step_of(za[j]), step_of(zb[j])) * unit_step[j] >= (float)(4 << LIFT);        // (an exponent more than one above; false for NaN)
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = s[n][i] * factor[n][i & 1];
                if (cap_log2 > 0.f) x = cap_log2 * tanh_ex2(x);
                if (!full && !(i < 2 ? seen_a : seen_b)) x = -INFINITY;
                s[n][i] = x;
                moves |= x > limit[n][i & 1];
            }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int largest = (int)(__float_as_uint(fmaxf(0.f, fmaxf(step_of(za[j]), step_of(zb[j])))) >> 23);
                const int old = 254 + LIFT - (int)(__float_as_uint(unit_step[j]) >> 23);
                const int fresh = max(old, min(MOST_EXPONENT, __reduce_max_sync(0xffffffffu, largest)));
                const float shrink = __uint_as_float((uint32_t)max(0, 127 - (fresh - old)) << 23);
                unit_step[j] = reciprocal(fresh);
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[n][j][x][i] *= shrink;
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float top = fmaxf(s[n][b], s[n][2 + b]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    top = limit[n][b] == -INFINITY ? top : fmaxf(top, base[n][b]);
                    const float shrink = limit[n][b] == -INFINITY ? 0.f : ex2(base[n][b] - top);
                    limit[n][b] = top + HEADROOM;
                    base[n][b] = top == -INFINITY ? 0.f : top;
                    l[n][b] *= shrink;
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        lows[n][j][b] *= shrink;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            o[n][j][x][b] *= shrink;
                            o[n][j][x][2 + b] *= shrink;
                        }
                    }
                }
        }
        // ---- weights and values
        uint32_t v0[NG], v1[NG], v2[NG], v3[NG];
        load_words<NG>(at + R::CODES + row_v * NG * 16 + (g & 3) * NG * 4, v0);
        load_words<NG>(at + R::CODES + row_w * NG * 16 + (g & 3) * NG * 4, v1);
        load_words<NG>(at + R::CODES + (row_v + 8) * NG * 16 + (g & 3) * NG * 4, v2);
        load_words<NG>(at + R::CODES + (row_w + 8) * NG * 16 + (g & 3) * NG * 4, v3);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = ex2(s[n][i] - base[n][i & 1]);
                l[n][i & 1] += s[n][i];
            }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const uint32_t x = __byte_perm(v0[j], v1[j], half_of), y = __byte_perm(v2[j], v3[j], half_of), xs = x >> 8, ys = y >> 8;
            const uint32_t a0 = half_add(thousand_plus(x), LESS_1032), a1 = half_add(sixty_four_plus(x), LESS_72),
                           a2 = half_add(thousand_plus(y), LESS_1032), a3 = half_add(sixty_four_plus(y), LESS_72);
            const uint32_t a4 = half_add(thousand_plus(xs), LESS_1032), a5 = half_add(sixty_four_plus(xs), LESS_72),
                           a6 = half_add(thousand_plus(ys), LESS_1032), a7 = half_add(sixty_four_plus(ys), LESS_72);
            const float mid_a = fmaf(8.f, step_of(za[j]), low_of(za[j])), mid_b = fmaf(8.f, step_of(zb[j]), low_of(zb[j]));
            // (a step of 0 gets a factor of -2^-126, which is the largest of all as bits and makes weights of 0 in float16)
            const float by_a = fmaf(step_of(za[j]), unit_step[j], -0x1p-126f), by_b = fmaf(step_of(zb[j]), unit_step[j], -0x1p-126f);
            least = __vimin3_u32(__float_as_uint(by_a), __float_as_uint(by_b), least);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const uint32_t b0 = transposed(half_pair(s[n][0] * by_a, s[n][1] * by_a));
                const uint32_t b1 = transposed(half_pair(s[n][2] * by_b, s[n][3] * by_b));
#pragma unroll
                for (int b = 0; b < 2; ++b) lows[n][j][b] = fmaf(s[n][b], mid_a, fmaf(s[n][2 + b], mid_b, lows[n][j][b]));
                mma_f16(o[n][j][0], a0, a1, a2, a3, b0, b1);
                mma_f16(o[n][j][1], a4, a5, a6, a7, b0, b1);
            }
        }
    }
    copies_wait<0>();

    // ---- the warps' states: sums over the keys' lanes, then through shared memory
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l[n][b] += __shfl_xor_sync(0xffffffffu, l[n][b], x);
#pragma unroll
                for (int j = 0; j < NG; ++j) lows[n][j][b] += __shfl_xor_sync(0xffffffffu, lows[n][j][b], x);
            }
        }
    const bool strange = __any_sync(0xffffffffu, least < __float_as_uint(LEAST_FACTOR));
    __syncthreads();                                             // the rings are done with
    float* acc_s = reinterpret_cast<float*>(memory);             // [M_WARPS][COLUMNS][NUMBERS]
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int column = n * 8 + 2 * c + b;
            float* row = acc_s + (warp * COLUMNS + column) * NUMBERS;
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int d = j * GROUP + 8 * (g & 3) + (g >> 2) + 4 * x;
                    const float unit = __uint_as_float((254u << 23) - __float_as_uint(unit_step[j]));      // one over it
                    row[d] = fmaf(o[n][j][x][b], unit, lows[n][j][b]);
                    row[d + 2] = fmaf(o[n][j][x][2 + b], unit, lows[n][j][b]);
                }
            if (g == 0) {
                base_s[warp][column] = limit[n][b] == -INFINITY ? -INFINITY : base[n][b];
                sum_s[warp][column] = strange ? __uint_as_float(0x7fffffffu) : l[n][b];         // (a NaN: the row is done again)
            }
        }
    __syncthreads();
    float* share_acc = acc_s;                                    // the first warp's place: each number is read before it is written, by one thread
    for (int i = threadIdx.x; i < COLUMNS * NUMBERS; i += M_WARPS * 32) {
        const int column = i / NUMBERS;
        float top = base_s[0][column];
#pragma unroll
        for (int w = 1; w < M_WARPS; ++w) top = fmaxf(top, base_s[w][column]);
        const float ground = top == -INFINITY ? 0.f : top;
        float sum = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < M_WARPS; ++w) {
            const float by = ex2(base_s[w][column] - ground);
            sum = fmaf(acc_s[w * COLUMNS * NUMBERS + i], by, sum);
            total = fmaf(sum_s[w][column], by, total);
        }
        share_acc[i] = sum;
        if (i % NUMBERS == 0) {
            share_base[column] = top;
            share_sum[column] = total;
        }
    }
    if (shares > 1) cluster_sync_all();
    else __syncthreads();
    // the shares': each of them finishes a part of the numbers, a warp 32 of a query at a time
    for (int i = share * M_WARPS * 32 + threadIdx.x; i < COLUMNS * NUMBERS; i += shares * M_WARPS * 32) {
        const int column = i / NUMBERS, d = i % NUMBERS, query = first_query + column;
        if (query >= ratio) continue;
        const int h = kv_head * ratio + query;
        const float sink_log2 = sink ? sink[h] * 1.4426950408889634f : -INFINITY;
        float top = sink_log2, sum = 0.f;
        for (int x = 0; x < shares; ++x) top = fmaxf(top, shares > 1 ? ld_cluster_f32(&share_base[column], x) : share_base[column]);
        const float ground = top == -INFINITY ? 0.f : top;
        float total = sink ? ex2(sink_log2 - ground) : 0.f;
        for (int x = 0; x < shares; ++x) {
            const float by = ex2((shares > 1 ? ld_cluster_f32(&share_base[column], x) : share_base[column]) - ground);
            total = fmaf(shares > 1 ? ld_cluster_f32(&share_sum[column], x) : share_sum[column], by, total);
            sum = fmaf(shares > 1 ? ld_cluster_f32(&share_acc[i], x) : share_acc[i], by, sum);
        }
        if (total != total) {                                     // weights that are no numbers, or that float16 does not hold
            const Cache cache = {k_pool, v_pool, page_stride, pages};
            if (d < GROUP)                                        // (the warp that has the query's first numbers; read anew: no register keeps them in the loop)
                row_again(q + t * q_stride + (long long)h * head_dim, out, t * out_stride + (long long)h * head_dim, wide, cache, token_row[t],
                          (long long)kv_head * slab_bytes(page_size, head_dim), head_dim, positions[t], window, scale, softcap, sink ? sink + h : nullptr, lane);
            continue;
        }
        if (d >= head_dim) continue;
        // (no key at all: zero; a NaN stays one)
        const float result = total == 0.f ? sum * 0.f : sum / total;
        const long long to = t * out_stride + (long long)h * head_dim + d;
        if (wide) reinterpret_cast<float*>(out)[to] = result;
        else reinterpret_cast<__nv_bfloat16*>(out)[to] = __float2bfloat16_rn(result);
    }
    if (shares > 1) cluster_sync_all();                          // the shares stay until they were read
}

template <int NG, int NQ, int M_WARPS>
int launch_mma(const void* q, long long q_stride, void* out, long long out_stride, int wide, const void* k_pool, const void* v_pool,
               long long page_stride, const int* token_row, const int* positions, const Pages& pages, int tokens, int n_heads, int n_kv_heads,
               int head_dim, int window, float scale, float softcap, const float* sink, int shares, cudaStream_t s) {
    constexpr int COLUMNS = 8 * NQ, MERGE = M_WARPS * COLUMNS * NG * GROUP * 4;
    constexpr size_t SMEM = Ring<NG, M_WARPS>::BYTES > MERGE ? Ring<NG, M_WARPS>::BYTES : MERGE;
    auto kernel = tokens_mma_kernel<NG, NQ, M_WARPS>;
    static size_t raised[MAX_DEVICES] = {0};
    if (!ensure_dynamic_smem((const void*)kernel, SMEM, raised)) return PS_ERR_LAUNCH;
    const int ratio = n_heads / n_kv_heads, blocks = (ratio + COLUMNS - 1) / COLUMNS;
    const int aligned = !((uintptr_t)q & 15) && q_stride % 8 == 0 && head_dim % 8 == 0;
    return launch_pdl_cluster(kernel, dim3(tokens, n_kv_heads * blocks, shares), dim3(M_WARPS * 32), SMEM, s, shares, (const __nv_bfloat16*)q,
                              q_stride, out, out_stride, wide, (const unsigned char*)k_pool, (const unsigned char*)v_pool, page_stride, token_row,
                              positions, pages, n_heads, n_kv_heads, head_dim, window, scale, softcap, sink, aligned);
}

}  // namespace packed
}  // namespace ps

// As ps_packed_tokens_simt, for bfloat16 queries and head sizes up to 128.  wide: out is float32.
PS_EXPORT int ps_packed_tokens_mma(const void* q, long long q_stride, void* out, long long out_stride, int wide, const void* k_pool,
                                   const void* v_pool, int n_pages, long long page_stride, const int* token_row, const int* positions,
                                   const int* block_table, int bt_stride, int tokens, int n_heads, int n_kv_heads, int head_dim, int page_size,
                                   int window, float scale, float softcap, const float* sink, int shares, int warps, void* stream) {
    using namespace ps::packed;
    if (tokens <= 0) return PS_OK;
    if (!q || !out || !k_pool || !v_pool || !token_row || !positions || !block_table) return PS_ERR_BAD_ARGUMENT;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return PS_ERR_BAD_ARGUMENT;
    if (!sizes_ok(n_kv_heads, head_dim, page_size) || head_dim > 128 || n_heads > 65535) return PS_ERR_UNSUPPORTED;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    if ((shares != 1 && shares != 2 && shares != 4 && shares != 8) || (warps != 4 && warps != 8)) return PS_ERR_BAD_ARGUMENT;
    const Pages pages = {block_table, bt_stride, n_pages, log2_of(page_size)};
    const bool two = n_heads / n_kv_heads > 8;
#define PS_PACKED_MMA(NG, NQ, W)                                                                                                             \
    return launch_mma<NG, NQ, W>(q, q_stride, out, out_stride, wide, k_pool, v_pool, page_stride, token_row, positions, pages, tokens,       \
                                 n_heads, n_kv_heads, head_dim, window, scale, softcap, sink, shares, (cudaStream_t)stream)
#define PS_PACKED_MMA_GROUPS(NG)                         \
    case NG:                                             \
        if (two && warps == 8) PS_PACKED_MMA(NG, 2, 8);  \
        if (two) PS_PACKED_MMA(NG, 2, 4);                \
        if (warps == 8) PS_PACKED_MMA(NG, 1, 8);         \
        PS_PACKED_MMA(NG, 1, 4)
    switch (groups_of(head_dim)) {
        PS_PACKED_MMA_GROUPS(1);
        PS_PACKED_MMA_GROUPS(2);
        PS_PACKED_MMA_GROUPS(3);
        PS_PACKED_MMA_GROUPS(4);
    }
#undef PS_PACKED_MMA_GROUPS
#undef PS_PACKED_MMA
    return PS_ERR_UNSUPPORTED;
}
