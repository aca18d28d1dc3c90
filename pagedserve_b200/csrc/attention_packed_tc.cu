// Causal attention of prompt portions over a cache held in 4 bits on tcgen05 tensor cores (bfloat16 queries, head sizes up to 128; packed.cuh
// has the cache's format).
//
// One CTA per (block of 256 query tokens of one request, head, share of the keys), tiles of 128 keys aligned to absolute positions. The block is two
// tiles of 128 queries that take turns: while the rows of one form their weights, the tensor cores work for the other.
//   warps 0..3   a key and its value a thread: codes and scales come to registers ahead of their tile, become 32 (low + code * step) (one rounding to
//                float16, 2^-11 of the number, an eighth of bfloat16's: two bfloat16 roundings, of keys and of values, made the result twice as inexact
//                as its own) and go to the swizzled tile, 16 bytes a word of codes
//   warps 4, 13  issue of S = Q K^T and O += P V for the first and the second query tile (4: TMEM allocation, too)
//   warps 5..12  a thread per query row: the query to its tile, then softmax: maximum, weights (float16, to TMEM), sum. The base of a row's weights moves,
//                and O with it, only when a score is beyond it by 2^8, which float16 has room for
// Weights are 2^7 times what their base gives, so that one is held to 2^-11 of itself or to 2^-32 of its row's largest; their sum has them unrounded. A sink joins
// the sum at the end.
// A tile's keys go through in two halves of 64, whose scores have columns of their own: P of a half takes the place of its scores, P V of the half is
// issued and then the scores of the same half of the next tile (MMAs run in the order of their issue), while the rows work on the other half.
// Queries are scaled row by row by a power of two, which leaves a number of a bfloat16 row as it is, or within 2^-33 of the row's largest: 2^-13 of any group whose
// largest is 2^-20 of that. Keys and values are all scaled by 2^5, which puts ordinary ones into the middle of float16's range. A step or a low of 2^-22 or more
// (2^-17 once scaled) is a float16 number then, of eight digits on a grid of 2^-24, and so low + code * step, on that grid too, is rounded to 2^-11 of itself or not at
// all. A block that needs a group with a smaller step or low other than zero, with a number beyond 1,875 (60,000 once scaled) or a NaN, a key without a page, or a query
// with a smaller group other than zero, forms its rows again in float32 from the codes (row_again in packed.cuh), which is slow and right.
// Few blocks of many keys: a cluster's CTAs share the key tiles out, leave O, bases and sums in shared memory and join a part of the rows each; a block of
// few keys takes fewer of them, and the others end at once.
//
// What bounds it: per 128 keys and 256 queries the rows' instructions are about 2,500 clocks, 2,048 of them exponentials, and at head size 128 the makers' about 2,500
// (keys and values), the products' 2,050; a tile takes about 5,000 there, with 54 % of the issue slots and 42 % of the tensor pipe used: the roles wait for one another,
// and which of the waits it is has not been measured. Then about 12,000 clocks from a CTA's start to its first weights, four dependent reads (lengths, row, page,
// codes) and the first passes through everything. Two prompts of 1,024 (12 heads of 64) 25.1 us; three portions of 683 and fewer queries
// behind up to 8,192 keys (16 heads on 4 of 128) 170 us, 0.62 PFLOP/s. Rows that are formed again take a warp 0.4 us a key: 250 us for a prompt of 129, 7.5 ms where
// all blocks of two prompts of 1,024 do. The way there at those two: an MMA issued behind `lane == 0`, or predicated, takes 70 to 97
// clocks, behind elect.sync 45 (190 -> 182 us at head size 128, one query tile 68 -> 54); the queries by the rows' warps, which wait anyway, instead of the
// makers (26.8 -> 25.6, 182 -> 170). Two threads a row, 32 scores each, were slower (30 us, 190: a meeting of the two each half, and 80 registers a thread), and so were six
// makers with halves of rows (27, 211: the groups' numbers twice, a page for each).
#include <type_traits>

#include "packed.cuh"

namespace ps {
namespace packedtc {

using namespace packed;

constexpr int BQ = 128, BKEY = 128, MAKERS = 128, THREADS = MAKERS + 64 + 2 * BQ;
constexpr uint64_t WAIT_LIMIT_NS = 200ull * 1000 * 1000;
constexpr float CACHE_SCALE = 32.f, MOST = 60000.f;                // what keys and values are multiplied by on their way into float16; the largest there
constexpr uint32_t LEAST_BITS = 0x3480u;                           // 2^-22 in bfloat16: steps and lows from there on are float16 numbers once scaled

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t timer_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
// false: the wait ran out, or another role of this CTA gave up
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    // (the timer is read only after many tries: a read takes longer than most waits)
#pragma unroll 1
    for (int spin = 0; spin < 2048; ++spin)
        if (mbar_try_wait(bar, parity)) return true;
    const uint64_t start = timer_ns();
    while (true) {
#pragma unroll 1
        for (int spin = 0; spin < 64; ++spin)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (timer_ns() - start > WAIT_LIMIT_NS) { *abort_flag = 1; return false; }
    }
}
__device__ __forceinline__ uint64_t desc_sw128(uint32_t smem_addr, uint32_t lbo_bytes) {
    uint64_t desc = (uint64_t)((smem_addr >> 4) & 0x3FFF);
    desc |= (uint64_t)((lbo_bytes >> 4) & 0x3FFF) << 16;
    desc |= (uint64_t)(1024 >> 4) << 32;
    desc |= (uint64_t)1 << 46;
    desc |= (uint64_t)2 << 61;
    return desc;
}
// one lane of a warp, chosen by the instruction that the compiler knows to choose one (behind `lane == 0` it moves an MMA's operands one by one:
// 70 to 97 clocks an MMA; in this branch 45, at N = 64)
__device__ __forceinline__ bool elect_one() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
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
__device__ __forceinline__ uint32_t half_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// the byte of a tile ([HD / 64][128 rows][128 bytes], swizzled) at which the eight numbers from d on of a row stand
__device__ __forceinline__ uint32_t tile_byte(int row, int d) {
    return (uint32_t)((d >> 6) * (128 * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4));
}
// a word of codes as eight float16 numbers low + code * step
__device__ __forceinline__ uint4 numbers_of(uint32_t word, uint32_t step, uint32_t low) {
    const uint32_t next = word >> 8;
    uint4 v;                                                       // codes 1024 + c and 64 + c, less those: whole numbers, exactly
    v.x = half_fma(half_add((word & 0x000f000fu) | 0x64006400u, 0xe400e400u), step, low);
    v.y = half_fma(half_add((word & 0x00f000f0u) | 0x54005400u, 0xd400d400u), step, low);
    v.z = half_fma(half_add((next & 0x000f000fu) | 0x64006400u, 0xe400e400u), step, low);
    v.w = half_fma(half_add((next & 0x00f000f0u) | 0x54005400u, 0xd400d400u), step, low);
    return v;
}

template <int HD>
struct Layout {
    static constexpr int KV_STAGES = 2, KCH = HD / 64, Q_BYTES = BQ * HD * 2, KV_BYTES = BKEY * HD * 2, STAGE_BYTES = 2 * KV_BYTES;
    // two query tiles, the stages, barriers (256 bytes), then a few words
    static constexpr size_t SMEM = 2 * Q_BYTES + (size_t)KV_STAGES * STAGE_BYTES + 1024 + 256 + 16;
    static constexpr int PART_ROW = HD + 4;                         // pitch of a share's O rows: eight neighbouring rows on eight groups of four banks
    // TMEM: scores of either tile (P takes their place), then O of either
    static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
};
constexpr float HEADROOM = 8.f;                                     // log2 of how far a weight may be beyond 1 before its base moves
constexpr float LIFT = 7.f;                                         // log2 of what weights are multiplied by: float16's largest is above 2^(LIFT + HEADROOM)

template <int HD, bool CAPPED>
__global__ void __launch_bounds__(THREADS, 1)
prompts_kernel(const __nv_bfloat16* __restrict__ q, long long q_stride, void* __restrict__ out, long long out_stride, Cache cache,
               const int* __restrict__ q_start, const int* __restrict__ kv_len, const int* __restrict__ item_row, int n_items, int n_heads,
               int n_kv_heads, int head_dim, int window, float scale, float softcap, SoftmaxExtras extras, int aligned_q, int aligned_out,
               int most, int* __restrict__ status) {
    using L = Layout<HD>;
    constexpr int KV_STAGES = L::KV_STAGES, GROUPS_MOST = HD / GROUP;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = base;                // two tiles
    unsigned char* kv_s = base + 2 * L::Q_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(kv_s + (size_t)KV_STAGES * L::STAGE_BYTES);
    uint64_t* q_full = bars;                  // [2] rows -> MMA
    uint64_t* k_full = q_full + 2;            // [KV_STAGES] makers -> MMA
    uint64_t* k_empty = k_full + KV_STAGES;   // [KV_STAGES] MMA -> makers
    uint64_t* v_full = k_empty + KV_STAGES;   // [KV_STAGES] makers -> MMA
    uint64_t* v_empty = v_full + KV_STAGES;   // [KV_STAGES] MMA -> makers
    uint64_t* s_full = v_empty + KV_STAGES;   // [2 query tiles][2 halves] MMA -> rows: the half's scores are complete
    uint64_t* p_ready = s_full + 4;           // [2][2] rows -> MMA: P of the half is in TMEM, O is in its units
    uint64_t* o_done = p_ready + 4;           // [2] MMA -> rows: P V of a half is complete
    uint64_t* o_full = o_done + 2;            // [2] MMA -> rows: O is complete (o_done could be a phase or two behind where no one waited for it)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* strange_s = reinterpret_cast<uint32_t*>(reinterpret_cast<unsigned char*>(bars) + 256);    // whether the rows are to be formed again

    pdl_prologue();
    q = pdl_fresh(q);
    cache.k_pool = pdl_fresh(cache.k_pool);
    cache.v_pool = pdl_fresh(cache.v_pool);
    int block = blockIdx.y, item = -1, qb = 0;                    // late blocks see most keys: they come first
    for (int i = 0; i < n_items; ++i) {
        const int blocks = (q_start[i + 1] - q_start[i] + 2 * BQ - 1) / (2 * BQ);
        if (block < blocks) { item = i; qb = blocks - 1 - block; break; }
        block -= blocks;
    }
    if (item < 0) return;
    const int h = blockIdx.x, g = h / (n_heads / n_kv_heads), share = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int qs = q_start[item], q_len = q_start[item + 1] - qs;
    const int pos0 = kv_len[item] - q_len + qb * 2 * BQ;              // position of the block's first query
    const int rows = min(2 * BQ, q_len - qb * 2 * BQ), tok0 = qs + qb * 2 * BQ;
    const int hi = pos0 + rows - 1, lo = pos0 < 0 ? 0 : first_visible_key(pos0, window);
    // the share's run of the block's key tiles: `most` of them or fewer, while the cluster's CTAs last; one without a share is done
    const int kb_all = lo / BKEY, kb_count = max(hi, 0) / BKEY - kb_all + 1, shares = min((int)gridDim.z, (kb_count + most - 1) / most);
    if (share >= shares) return;
    const int kb_first = kb_all + kb_count * share / shares, kb_last = kb_all + kb_count * (share + 1) / shares - 1;
    // those of them that a query tile's rows see (a second tile without rows: none)
    auto first_of = [&](int x) {
        const int p = pos0 + x * BQ;
        return x * BQ >= rows ? kb_last + 1 : max(kb_first, (p < 0 ? 0 : first_visible_key(p, window)) / BKEY);
    };
    auto last_of = [&](int x) { return min(kb_last, max(pos0 + min(rows, (x + 1) * BQ) - 1, 0) / BKEY); };
    const int table_row = item_row ? item_row[item] : item;
    const int page_size = 1 << cache.pages.page_log2, groups = groups_of(head_dim);
    const long long head_at = (long long)g * slab_bytes(page_size, head_dim);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < KV_STAGES; ++s) {
            mbar_init(&k_full[s], MAKERS / 32); mbar_init(&k_empty[s], 2);
            mbar_init(&v_full[s], MAKERS / 32); mbar_init(&v_empty[s], 2);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&q_full[x], BQ / 32);
            for (int half = 0; half < 2; ++half) {
                mbar_init(&s_full[2 * x + half], 1);
                mbar_init(&p_ready[2 * x + half], BQ / 32);
            }
            mbar_init(&o_done[x], 1);
            mbar_init(&o_full[x], 1);
        }
        *strange_s = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)L::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const float sink_log2 = extras.sink ? extras.sink[h] * 1.4426950408889634f : -INFINITY;
    // one arrival for a whole warp
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    // eight numbers of a query row's result, from d on
    auto store8 = [&](int place, int d, const float (&v)[8]) {
        const long long to = (long long)(tok0 + place) * out_stride + (long long)h * head_dim + d;
        if (aligned_out && d + 8 <= head_dim) {
            if (extras.wide) {
                float4* at = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + to);
                at[0] = make_float4(v[0], v[1], v[2], v[3]);
                at[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                uint4 pack;
                uint32_t* two = reinterpret_cast<uint32_t*>(&pack);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    two[i] = *reinterpret_cast<const uint32_t*>(&b);
                }
                *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + to) = pack;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < head_dim) store_result(reinterpret_cast<__nv_bfloat16*>(out), to + i, v[i], extras);
        }
    };
    // what a share leaves of its rows, over the tiles: O, then the bases and the sums of the weights
    float* part_s = reinterpret_cast<float*>(base);
    float *part_m = part_s + 2 * BQ * L::PART_ROW, *part_l = part_m + 2 * BQ;

    if (warp < 4) {
        // ------------------------------------------------ makers: thread r has key r of every tile and its value
        const int r = threadIdx.x;
        uint4 k_codes[GROUPS_MOST], v_codes[GROUPS_MOST];
        uint32_t k_scales[GROUPS_MOST], v_scales[GROUPS_MOST];
        bool strange = false;
        uint32_t least = 0xffffffffu;                              // the smallest step and low other than 0 (bits of their sizes, less 1), either in its half
        long long page_at = -1;                                    // of the key whose numbers are asked for (below 0: not needed, or no page)
        int page_row = 0;
        // A key's entry of the block table is asked for a tile before its codes, and not looked at until then: a comparison would wait for it.
        const int* table = cache.pages.block_table + (size_t)table_row * cache.pages.bt_stride;
        auto needed = [&](int kb) { return kb * BKEY + r >= lo && kb * BKEY + r <= hi; };
        auto entry_of = [&](int kb) {
            const int at = (kb * BKEY + r) >> cache.pages.page_log2;
            return needed(kb) && at < cache.pages.bt_stride ? table[at] : -1;
        };
        int entry = entry_of(kb_first);
        auto locate = [&](int kb) {
            const int page = entry < cache.pages.n_pages ? entry : -1;
            entry = entry_of(kb + 1);
            strange |= needed(kb) && page < 0;
            page_row = (kb * BKEY + r) & (page_size - 1);
            page_at = page < 0 ? -1 : (long long)page * cache.page_stride + head_at;
        };
        auto fetch = [&](const unsigned char* pool, uint4 (&codes)[GROUPS_MOST], uint32_t (&scales)[GROUPS_MOST]) {
            const unsigned char* at = pool + page_at;
#pragma unroll
            for (int j = 0; j < GROUPS_MOST; ++j) {
                const bool there = page_at >= 0 && j < groups;
                codes[j] = there ? *reinterpret_cast<const uint4*>(at + (page_row * groups + j) * 16) : make_uint4(0, 0, 0, 0);
                scales[j] = there ? *reinterpret_cast<const uint32_t*>(at + page_size * groups * 16 + (page_row * groups + j) * 4) : 0u;
            }
        };
        // a row of a tile: place p of the codes (part p / groups of group p % groups) becomes eight numbers; what is not there becomes zeros
        auto make = [&](unsigned char* tile, const uint4 (&codes)[GROUPS_MOST], const uint32_t (&scales)[GROUPS_MOST]) {
            uint32_t step[GROUPS_MOST], low[GROUPS_MOST];
#pragma unroll
            for (int j = 0; j < GROUPS_MOST; ++j) {
                const float a = step_of(scales[j]) * CACHE_SCALE, b = low_of(scales[j]) * CACHE_SCALE;
                strange |= !(fmaxf(fabsf(b), fabsf(fmaf(15.f, a, b))) <= MOST);
                least = __viaddmin_u16x2(scales[j] & 0x7fff7fffu, 0xffffffffu, least);         // (0 less 1 is the largest of all)
                step[j] = half_pair(a, a);
                low[j] = half_pair(b, b);
            }
            auto put = [&](auto count) {
                constexpr int NG = decltype(count)::value;
#pragma unroll
                for (int p = 0; p < 4 * NG; ++p) {
                    const uint4& four = codes[p >> 2];
                    const uint32_t word = (p & 3) == 0 ? four.x : (p & 3) == 1 ? four.y : (p & 3) == 2 ? four.z : four.w;
                    *reinterpret_cast<uint4*>(tile + tile_byte(r, (p % NG) * GROUP + p / NG * 8)) = numbers_of(word, step[p % NG], low[p % NG]);
                }
#pragma unroll
                for (int d = NG * GROUP; d < HD; d += 8) *reinterpret_cast<uint4*>(tile + tile_byte(r, d)) = make_uint4(0, 0, 0, 0);
            };
            if constexpr (GROUPS_MOST == 2) {
                if (groups == 2) put(std::integral_constant<int, 2>());
                else put(std::integral_constant<int, 1>());
            } else {
                if (groups == 4) put(std::integral_constant<int, 4>());
                else put(std::integral_constant<int, 3>());
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        locate(kb_first);
        fetch(cache.k_pool, k_codes, k_scales);
        fetch(cache.v_pool, v_codes, v_scales);
        uint32_t it = 0;
        for (int kb = kb_first; kb <= kb_last; ++kb, ++it) {
            const int s = it % KV_STAGES;
            const uint32_t free = ((it / KV_STAGES) & 1) ^ 1;
            unsigned char* tile = kv_s + (size_t)s * L::STAGE_BYTES;
            if (kb < kb_last) locate(kb + 1);
            if (!mbar_wait(&k_empty[s], free, abort_flag)) { if (lane == 0) atomicExch(status, 51); break; }
            make(tile, k_codes, k_scales);
            arrive(&k_full[s]);
            if (kb < kb_last) fetch(cache.k_pool, k_codes, k_scales);
            if (!mbar_wait(&v_empty[s], free, abort_flag)) { if (lane == 0) atomicExch(status, 52); break; }
            make(tile + L::KV_BYTES, v_codes, v_scales);
            arrive(&v_full[s]);
            if (kb < kb_last) fetch(cache.v_pool, v_codes, v_scales);
        }
        strange |= (least & 0xffffu) < LEAST_BITS - 1u || (least >> 16) < LEAST_BITS - 1u;
        if (__any_sync(0xffffffffu, strange) && lane == 0) atomicExch(strange_s, 1u);
    } else if (warp == 4 || warp == 13) {
        // ------------------------------------------------ MMA issuers, one for each query tile
        // D f32, A/B f16: S = Q K^T both K-major, N = 64; O = P V with A from TMEM and B MN-major (bit 16), N = HD
        constexpr uint32_t idesc_qk = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
        constexpr uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
        const int x = warp == 4 ? 0 : 1, first = first_of(x), last = last_of(x);
        const uint32_t s_at = tmem_base + L::S_COL + x * 128, o_at = tmem_base + L::O_COL + x * HD;
        const uint64_t q_desc = desc_sw128(smem_u32(q_s + x * L::Q_BYTES), 16);
        auto waits = [&](uint64_t* bar, uint32_t parity, int code) {
            const bool there = mbar_wait(bar, parity, abort_flag);
            if (!there) atomicExch(status, code);
            tc_fence_after();
            return there;
        };
        auto scores = [&](int kb, int half) {                      // (64 rows of a tile are 8,192 bytes)
            const uint64_t k_desc = desc_sw128(smem_u32(kv_s + (size_t)((kb - kb_first) % KV_STAGES) * L::STAGE_BYTES) + half * 8192, 16);
#pragma unroll
            for (int c = 0; c < L::KCH; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_ss(s_at + half * 64, q_desc + c * (BQ * 128 / 16) + 2 * k, k_desc + c * (BKEY * 128 / 16) + 2 * k, idesc_qk, (c | k) ? 1u : 0u);
            umma_commit(&s_full[2 * x + half]);
        };
        if (elect_one()) {
            bool ok = true;
            uint32_t taken = 0;                                        // key tiles of this query tile whose weights were taken
            for (int kb = kb_first - 1; kb <= kb_last && ok; ++kb) {   // weights of tile kb, scores of kb + 1
                const uint32_t it = (uint32_t)(kb - kb_first);
                const bool weighs = kb >= first && kb <= last, next = kb + 1 <= kb_last, asks = kb + 1 >= first && kb + 1 <= last;
                if (next) ok = waits(&k_full[(it + 1) % KV_STAGES], ((it + 1) / KV_STAGES) & 1, 54);
                if (ok && kb + 1 == first) ok = waits(&q_full[x], 0, 53);
                if (ok && kb >= kb_first) ok = waits(&v_full[it % KV_STAGES], (it / KV_STAGES) & 1, 57);
#pragma unroll 1
                for (int half = 0; half < 2 && ok; ++half) {
                    if (weighs) {
                        ok = waits(&p_ready[2 * x + half], taken & 1, 56);
                        if (!ok) break;
                        const uint64_t v_desc = desc_sw128(smem_u32(kv_s + (size_t)(it % KV_STAGES) * L::STAGE_BYTES) + L::KV_BYTES + half * 8192, BKEY * 128);
#pragma unroll
                        for (int k = 0; k < 4; ++k)                    // 16 keys = 2,048 bytes of V, 8 columns of P
                            umma_ts(o_at, s_at + half * 64 + 8 * k, v_desc + (uint64_t)((2048 * k) >> 4), idesc_pv, (taken | (uint32_t)half | (uint32_t)k) ? 1u : 0u);
                        umma_commit(&o_done[x]);
                        if (kb == last && half == 1) umma_commit(&o_full[x]);
                    }
                    if (asks) scores(kb + 1, half);
                }
                if (ok && weighs) ++taken;
                // (a tile that this query tile does not see is given back as soon as it is there)
                if (ok && kb >= kb_first) umma_commit(&v_empty[it % KV_STAGES]);
                if (ok && next) umma_commit(&k_empty[(it + 1) % KV_STAGES]);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------ rows
        const int quarter = warp & 3, x = (warp - 5) >> 2;
        const int r = quarter * 32 + lane, place = x * BQ + r, pos = pos0 + place;
        const int first = first_of(x), last = last_of(x);
        const int lo_row = pos < 0 ? 0 : first_visible_key(pos, window);
        const int pos_first = pos0 + x * BQ, pos_last = pos0 + min(rows, (x + 1) * BQ) - 1;
        const int lo_all = pos_last < 0 ? 0 : first_visible_key(pos_last, window);        // the first key that every row of the tile sees
        const uint32_t s_at = tmem_base + ((uint32_t)(quarter * 32) << 16) + L::S_COL + x * 128;
        const uint32_t o_at = tmem_base + ((uint32_t)(quarter * 32) << 16) + L::O_COL + x * HD;
        // in log2 units: the base of the weights (of keys alone: beside a sink far above them they would be lost), what a score may reach
        float base_m = 0.f, limit = -INFINITY, l_run = 0.f;
        bool ok = first <= last;
        // the row's query, scaled by a power of two, to its tile
        float factor;
        {
            const __nv_bfloat16* row = q + (long long)(tok0 + place) * q_stride + (long long)h * head_dim;
            float most = 0.f, group_most[GROUPS_MOST];
            bool odd = false;
            uint4 raw[HD / 8];                                     // the whole row at once: its loads are under way together
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (place < rows && 8 * i < head_dim) {
                    if (aligned_q) {
                        raw[i] = *reinterpret_cast<const uint4*>(row + 8 * i);
                    } else {
                        const unsigned short* at = reinterpret_cast<const unsigned short*>(row + 8 * i);
                        auto number = [&](int j) -> uint32_t { return 8 * i + j < head_dim ? at[j] : 0u; };
                        raw[i] = make_uint4(number(0) | number(1) << 16, number(2) | number(3) << 16, number(4) | number(5) << 16, number(6) | number(7) << 16);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                float& largest = group_most[i / 4];
                if (i % 4 == 0) largest = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float lo_half = fabsf(__uint_as_float(w[j] << 16)), hi_half = fabsf(__uint_as_float(w[j] & 0xffff0000u));
                    largest = max3(largest, lo_half, hi_half);
                    odd |= !(lo_half <= 3.4028235e38f) || !(hi_half <= 3.4028235e38f);
                }
            }
#pragma unroll
            for (int j = 0; j < GROUPS_MOST; ++j) most = fmaxf(most, group_most[j]);
            bool small = false;
#pragma unroll
            for (int j = 0; j < GROUPS_MOST; ++j) small |= group_most[j] > 0.f && group_most[j] < most * 0x1p-20f;
            if (small && !odd) *strange_s = 1u;
            // 2^up brings the largest to [256, 512); a NaN or infinity stays one
            const int up = most > 0.f && !odd ? min(121, 135 - max(1, (int)(__float_as_uint(most) >> 23))) : 0;
            const float by = __uint_as_float((uint32_t)(127 + up) << 23);
            factor = __uint_as_float((uint32_t)(127 - up) << 23) * (1.f / CACHE_SCALE);      // (of queries and keys; up is -119 to 121)
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = half_pair(__uint_as_float(w[j] << 16) * by, __uint_as_float(w[j] & 0xffff0000u) * by);
                *reinterpret_cast<uint4*>(q_s + x * L::Q_BYTES + tile_byte(r, 8 * i)) = make_uint4(v[0], v[1], v[2], v[3]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(&q_full[x]);
        }
        // (not 0: minus infinity times it is to stay that)
        const float unit_scale = CAPPED ? 1.0f : fmaxf(scale * 1.4426950408889634f * factor, 1e-37f);
        const unsigned long long unit2 = pair_of(unit_scale, unit_scale);
        uint32_t n = 0;                                            // halves so far
        for (; first * 2 + (int)n < 2 * (last + 1) && ok; ++n) {
            const int half = n & 1, key0 = first * BKEY + (int)n * 64;
            if (!mbar_wait(&s_full[2 * x + half], (n >> 1) & 1, abort_flag)) { ok = false; if (lane == 0) atomicExch(status, 59); break; }
            tc_fence_after();
            uint32_t sr[64];
            tmem_ld32(s_at + half * 64, sr);
            tmem_ld32(s_at + half * 64 + 32, sr + 32);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if constexpr (CAPPED) {
#pragma unroll
                for (int j = 0; j < 64; ++j) sr[j] = __float_as_uint(cap_special(__uint_as_float(sr[j]) * factor, extras));
            }
            if (key0 + 63 > pos_first || key0 < lo_all || (x + 1) * BQ > rows) {
                const int first_ok = place < rows ? lo_row - key0 : 64, last_ok = place < rows ? pos - key0 : -1;
#pragma unroll
                for (int j = 0; j < 64; ++j)
                    if (j < first_ok || j > last_ok) sr[j] = 0xff800000u;        // -inf
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 64; j += 2) mx[(j >> 1) & 3] = max3(mx[(j >> 1) & 3], __uint_as_float(sr[j]), __uint_as_float(sr[j + 1]));
            const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * unit_scale;
            if (__any_sync(0xffffffffu, top > limit)) {
                const bool has = limit > -INFINITY, moves = top > limit;
                const float fresh = moves ? (has ? fmaxf(top, base_m) : top) : base_m, corr = !moves ? 1.f : (has ? ex2(base_m - fresh) : 0.f);
                base_m = fresh;
                if (moves) limit = fresh + HEADROOM;
                l_run *= corr;
                // No P V may be under way: that of the half before has to be done (that of the one before it is: this half's scores followed it).
                if (n > 0) {
                    if (!mbar_wait(&o_done[x], (n - 1) & 1, abort_flag)) { ok = false; if (lane == 0) atomicExch(status, 60); break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        uint32_t orr[16];
                        tmem_ld16(o_at + c, orr);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int j = 0; j < 16; ++j) orr[j] = __float_as_uint(__uint_as_float(orr[j]) * corr);
                        tmem_st16(o_at + c, orr);
                    }
                }
            }
            // weights 2^(s - base + LIFT)
            const unsigned long long less = pair_of(LIFT - base_m, LIFT - base_m);
            unsigned long long sum_a = 0ull, sum_b = 0ull;
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                uint32_t pr[16];
#pragma unroll
                for (int j = c; j < c + 32; j += 4) {
                    float p[4];
                    pair_split(pair_fma(pair_of(__uint_as_float(sr[j]), __uint_as_float(sr[j + 1])), unit2, less), p[0], p[1]);
                    pair_split(pair_fma(pair_of(__uint_as_float(sr[j + 2]), __uint_as_float(sr[j + 3])), unit2, less), p[2], p[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = ex2(p[i]);
                    sum_a = pair_add(sum_a, pair_of(p[0], p[1]));
                    sum_b = pair_add(sum_b, pair_of(p[2], p[3]));
                    pr[(j - c) >> 1] = half_pair(p[0], p[1]);
                    pr[((j - c) >> 1) + 1] = half_pair(p[2], p[3]);
                }
                tmem_st16(s_at + half * 64 + (c >> 1), pr);
            }
            float even, odd;
            pair_split(pair_add(sum_a, sum_b), even, odd);
            l_run += even + odd;
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            arrive(&p_ready[2 * x + half]);
        }
        if (ok && !mbar_wait(&o_full[x], 0, abort_flag)) { ok = false; if (lane == 0) atomicExch(status, 61); }
        tc_fence_after();
        if (shares > 1) {
            // (every row has waited for its O: no product reads the tiles any more, and what the makers made is all taken)
            asm volatile("bar.sync 1, %0;" ::"n"(2 * BQ) : "memory");
            part_m[place] = limit > -INFINITY ? base_m : -INFINITY;
            part_l[place] = l_run;
        }
        const float all = extras.sink ? l_run + ex2(sink_log2 - base_m + LIFT) : l_run, inv = all == 0.f ? 0.f : 1.f / (CACHE_SCALE * all);
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
            uint32_t orr[16];
            if (ok) {
                tmem_ld16(o_at + c, orr);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) orr[i] = 0u;          // (the share has no key that the tile sees)
            }
            if (shares > 1) {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<uint4*>(part_s + place * L::PART_ROW + c + i) = make_uint4(orr[i], orr[i + 1], orr[i + 2], orr[i + 3]);
            } else if (ok && place < rows) {
#pragma unroll
                for (int d = 0; d < 16; d += 8) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(orr[d + i]) * inv;
                    store8(place, c + d, v);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)L::TMEM_COLS) : "memory");
    }
    uint32_t strange = *strange_s;
    if (shares > 1) {
        __syncwarp();
        cluster_sync_all();
        for (int other = 0; other < shares; ++other) strange |= ld_cluster_u32(strange_s, other);
    }
    if (strange) {
        for (int r = share * (THREADS / 32) + warp; r < rows; r += shares * (THREADS / 32))
            row_again(q + (long long)(tok0 + r) * q_stride + (long long)h * head_dim, out, (long long)(tok0 + r) * out_stride + (long long)h * head_dim, extras.wide,
                      cache, table_row, head_at, head_dim, pos0 + r, window, scale, softcap, extras.sink ? extras.sink + h : nullptr, lane);
    } else if (shares > 1) {
        // a part of the rows each, eight numbers a thread
        constexpr int PIECES = HD / 8;
        const int first = rows * share / shares, count = rows * (share + 1) / shares - first;
        for (int i = threadIdx.x; i < count * PIECES; i += THREADS) {
            const int place = first + i / PIECES, d = i % PIECES * 8;
            if (d >= head_dim) continue;
            float top = sink_log2, v[8];
            for (int other = 0; other < shares; ++other) top = fmaxf(top, ld_cluster_f32(part_m + place, other));
            const float ground = top == -INFINITY ? 0.f : top;
            float total = extras.sink ? ex2(sink_log2 - ground + LIFT) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
            for (int other = 0; other < shares; ++other) {
                const float by = ex2(ld_cluster_f32(part_m + place, other) - ground);
                const float4 a = ld_cluster_f32x4(part_s + place * L::PART_ROW + d, other), b = ld_cluster_f32x4(part_s + place * L::PART_ROW + d + 4, other);
                const float one[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                total = fmaf(ld_cluster_f32(part_l + place, other), by, total);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = fmaf(one[j], by, v[j]);
            }
            const float inv = total == 0.f ? 0.f : 1.f / (CACHE_SCALE * total);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
            store8(place, d, v);
        }
    }
    if (shares > 1) {
        __syncwarp();
        cluster_sync_all();                                        // the shares stay until they were read
    }
}

template <int HD, bool CAPPED>
int launch(const void* q, long long q_stride, void* out, long long out_stride, int wide, const Cache& cache, const int* q_start, const int* kv_len,
           const int* item_row, int n_items, int max_blocks, int n_heads, int n_kv_heads, int head_dim, int window, float scale, float softcap,
           const float* sink, int shares, int most, int* status, cudaStream_t s) {
    auto kernel = prompts_kernel<HD, CAPPED>;
    static size_t raised[MAX_DEVICES] = {0};
    if (!ensure_dynamic_smem((const void*)kernel, Layout<HD>::SMEM, raised)) return PS_ERR_LAUNCH;
    const int aligned_q = !((uintptr_t)q & 15) && q_stride % 8 == 0 && head_dim % 8 == 0;
    const int aligned_out = !((uintptr_t)out & 15) && out_stride % 8 == 0 && head_dim % 8 == 0;
    return launch_pdl_cluster(kernel, dim3(n_heads, max_blocks, shares), dim3(THREADS), Layout<HD>::SMEM, s, shares, (const __nv_bfloat16*)q, q_stride, out, out_stride, cache,
                      q_start, kv_len, item_row, n_items, n_heads, n_kv_heads, head_dim, window, scale, softcap, softmax_extras(scale, softcap, sink, wide),
                      aligned_q, aligned_out, most, status);
}

}  // namespace packedtc
}  // namespace ps

// q / out: the step's flat rows of n_heads * head_dim numbers; item i's tokens are rows q_start[i] .. q_start[i + 1], the last ones of kv_len[i], its
// pages row item_row[i] of block_table (bt_stride wide).  max_blocks >= sum over the items of ceil(tokens / 256).  wide: out is float32.
// shares: CTAs (a cluster) that share a block's keys out, 1, 2, 4 or 8; most: tiles of 128 keys from which on a block takes another of them.
PS_EXPORT int ps_packed_prompts_tc(const void* q, long long q_stride, void* out, long long out_stride, int wide, const void* k_pool, const void* v_pool,
                                   int n_pages, long long page_stride, const int* q_start, const int* kv_len, const int* block_table, int bt_stride,
                                   const int* item_row, int n_items, int max_blocks, int n_heads, int n_kv_heads, int head_dim, int page_size,
                                   int window, float scale, float softcap, const float* sink, int shares, int most, int* status, void* stream) {
    using namespace ps::packedtc;
    if (n_items <= 0 || max_blocks <= 0) return PS_OK;
    if (!q || !out || !k_pool || !v_pool || !q_start || !kv_len || !block_table || !status) return PS_ERR_BAD_ARGUMENT;
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || max_blocks > 65535) return PS_ERR_BAD_ARGUMENT;
    if (!ps::packed::sizes_ok(n_kv_heads, head_dim, page_size) || head_dim > 128) return PS_ERR_UNSUPPORTED;
    if ((shares != 1 && shares != 2 && shares != 4 && shares != 8) || most <= 0) return PS_ERR_BAD_ARGUMENT;
    if (page_stride % 16 || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) return PS_ERR_UNSUPPORTED;
    const Cache cache = {(const unsigned char*)k_pool, (const unsigned char*)v_pool, page_stride, {block_table, bt_stride, n_pages, ps::packed::log2_of(page_size)}};
    auto run = head_dim <= 64 ? (softcap > 0.f ? launch<64, true> : launch<64, false>) : (softcap > 0.f ? launch<128, true> : launch<128, false>);
    return run(q, q_stride, out, out_stride, wide, cache, q_start, kv_len, item_row, n_items, max_blocks, n_heads, n_kv_heads, head_dim, window, scale,
               softcap, sink, shares, most, status, (cudaStream_t)stream);
}
