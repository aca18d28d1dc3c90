// Log probabilities of given tokens straight from the head's product (bfloat16): the logits are read where they are formed, out of tensor memory,
// and never stored (logprobs.cu says what is computed; 2,047 rows of 50,257 logits are 412 MB, 63 us to write and 63 to read).
//
// product     pairs of CTAs on tiles of 256 rows x 256 tokens as in gemm_tc.cu (tcgen05 cta_group::2, TMA, two accumulators in TMEM). A pair keeps
//             to its 256 rows and walks a strip of the vocabulary, so that the sums of a row stay in the registers of its four threads (each takes
//             every fourth 32 tokens of a tile); a strip leaves m, S and W of its part of a row.  A warp reads 32 tokens of its rows in about
//             2,300 clocks, most of them waits for results, so that with two threads a row the reading was longer than the product.
// sample      for the most likely tokens, the logits of every s-th token (about 2,048 of them, more for vocabularies and lists beyond 50,257 and 32: what lies beyond
//             the bound is to fit a row's list) are formed first, by the ordinary product: the `top`-th
//             largest of them is a bound that the row's `top` largest reach, less 2^-16 of itself, since another product may add in another order.
//             The product sends what lies beyond it (about 25 * top of 50,257) to a list of its row: a number larger than the bound, or equal to it
//             up to the sampled token that set it, so that whatever is not in the list comes behind all that is.  A thread holds up to 16 of them in
//             shared memory before it takes places in the list, all rows of a warp together (an atomic addition for each number cost a microsecond's
//             wait: 326 us of 445; one for each row that had eight, 157 of 266 us with 20 alternatives).
// join        a CTA a row adds the strips' sums up, ranks the list, and writes the results.  A row whose list did not hold all (an order of tokens that
//             fools the sample), or fewer than `top`, has its logits formed again there, token by token.
//
// What bounds it, 2,047 rows of 768 on 50,257 tokens (158 GFLOP, 96 us at a cuBLAS product's measured rate): without alternatives the tensor pipe, 91 % of the time
// active, 94 us (112 with the MMAs issued behind `lane == 0` instead of elect.sync); with 5 of them 157, with 20 183. One by one, in front of cold caches: the product
// 100 without alternatives and 127 with 5 (five stages for six, tensor memory read twice, numbers on their way to the lists: the tensor pipe 68 % active), the sample's
// product 18 and ranking 16, the join 17 (without alternatives 11). Up to about 256 rows (42 us; without alternatives 21) the table's 77 MB and four kernels one
// behind another.
#include <cuda.h>

#include "logprobs.cuh"

namespace ps {
namespace headlp {

using namespace logprob;

constexpr int NT = 256, CHUNK = NT * PER, CAPACITY = capacity<NT>();

constexpr int BM = 128, BN = 256, BK = 64, TEAMS = 4, ROW_THREADS = 128 * TEAMS, HEAD_THREADS = 64 + ROW_THREADS;
constexpr int STAGE_BYTES = BM * BK * 2 + (BN / 2) * BK * 2;
constexpr int HELD = 16;                                           // entries that a row's thread holds before it sends them to the row's list
// stages of the operands, fewer where rows hold entries
template <bool TOP> constexpr int stages() { return TOP ? 5 : 6; }
template <bool TOP> constexpr size_t smem_bytes() { return (size_t)stages<TOP>() * STAGE_BYTES + 1024 + 256 + (TOP ? ROW_THREADS * HELD * 8 : 0); }
constexpr int LIST = 2048;                                        // entries of a row's list
constexpr uint64_t WAIT_LIMIT_NS = 200ull * 1000 * 1000;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {               // arrivals of the other CTA too
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t timer_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
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
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(smem_u32(p)));
    return remote;
}
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr) {                           // K-major, 128-byte swizzle
    uint64_t desc = (uint64_t)((smem_addr >> 4) & 0x3FFF);
    desc |= (uint64_t)1 << 16;
    desc |= (uint64_t)(1024 >> 4) << 32;
    desc |= (uint64_t)1 << 46;
    desc |= (uint64_t)2 << 61;
    return desc;
}
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// one lane of a warp, chosen by the instruction that the compiler knows to choose one: an MMA's operands are then formed once for the warp
__device__ __forceinline__ bool elect_one() {
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {                                  // arrives at this place in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
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
__device__ __forceinline__ unsigned long long pair_ex2(unsigned long long x) {
    float lo, hi;
    pair_split(x, lo, hi);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(lo));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(hi));
    return pair_of(lo, hi);
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// What the three kernels hand on, of each row: partial sums of its threads in every strip, the target's logit, and with alternatives the list.
struct Scratch {
    float* sums;                     // [rows, TEAMS * strips, 3]: m, S, W
    float* given;                    // [rows]
    unsigned long long* list;        // [rows, LIST]: (logit, token)
    int* count;                      // [rows]: entries that were to be written
    float* limit;                    // [rows]: the bound, and
    int* limit_index;                // [rows] the token behind the sampled one that set it
};

// The sample: logits of tokens 0, s, 2 s, .. of a row (n of them, ld apart). One CTA a row.
__global__ void __launch_bounds__(NT)
sample_kernel(const float* __restrict__ logits, long long ld, int n, int every, int top, Scratch out) {
    __shared__ unsigned long long entry_s[CAPACITY], kept_s[MOST_TOP];
    __shared__ uint32_t group_s[GROUPS], limit_s, bound_s;
    __shared__ int count_s;
    pdl_prologue();
    logits = pdl_fresh(logits);
    const long long r = blockIdx.x;
    const int tid = threadIdx.x;
    const List list = {entry_s, kept_s, &count_s, &limit_s, group_s, &bound_s};
    if (tid == 0) { count_s = 0; limit_s = 0; }
    __syncthreads();
    for (int chunk = 0; chunk < n; chunk += CHUNK) {
        float x[PER], big = -INFINITY;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int i = chunk + u * NT + tid;
            x[u] = i < n ? logits[r * ld + i] : -INFINITY;
            big = fmaxf(big, x[u]);
        }
        consider<NT>(list, x, big, top, [&](int u) { const int i = chunk + u * NT + tid; return i < n ? i : -1; });
    }
    __syncthreads();
    rank<NT>(list, top);
    if (tid == top - 1) {
        const unsigned long long entry = entry_s[tid];
        const float value = value_of(order_in(entry));
        const bool number = order_in(entry) > 1u;
        out.limit[r] = number ? value * (value > 0.f ? 1.f - 0x1p-16f : 1.f + 0x1p-16f) : INFINITY;
        out.limit_index[r] = index_in(entry) * every + 1;
        out.count[r] = number ? 0 : LIST + 1;                     // (fewer numbers than `top` in the sample: the row is done again)
    }
}

template <bool TOP>
__global__ void __launch_bounds__(HEAD_THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const int* __restrict__ targets, int M, int N,
               int K, int strips, int tiles_per_strip, Scratch out, int* __restrict__ status) {
    constexpr int STAGES = stages<TOP>();
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + (size_t)STAGES * STAGE_BYTES);       // [STAGES] TMA -> MMA
    uint64_t* empty = full + STAGES;                                                          // [STAGES] MMA -> TMA
    uint64_t* acc_full = empty + STAGES;                                                      // [2] MMA -> rows
    uint64_t* acc_empty = acc_full + 2;                                                       // [2] rows -> MMA
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)blockIdx.x & 1, pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int tiles_n = (N + BN - 1) / BN, units = ((M + 2 * BM - 1) / (2 * BM)) * strips, num_kb = (K + BK - 1) / BK;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * ROW_THREADS / 32); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2u * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_prologue();

    // the tiles of a unit: rows (unit / strips) * 256 .., tokens of tiles [first, last) of its strip
    auto first_tile = [&](int unit) { return unit % strips * tiles_per_strip; };
    auto last_tile = [&](int unit) { return min(tiles_n, first_tile(unit) + tiles_per_strip); };

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int unit = pair; unit < units && ok; unit += pairs) {
                const int m0 = unit / strips * 2 * BM + rank * BM;
                for (int tile = first_tile(unit); tile < last_tile(unit) && ok; ++tile)
                    for (int kb = 0; kb < num_kb; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { ok = false; atomicExch(status, 42); break; }
                        unsigned char* dst = tiles + (size_t)s * STAGE_BYTES;
                        if (rank == 0) mbar_expect_tx(&full[s], 2 * STAGE_BYTES);             // (both CTAs' copies count there)
                        tma_load_pair(dst, &map_x, kb * BK, m0, in_first_cta(&full[s]));
                        tma_load_pair(dst + BM * BK * 2, &map_w, kb * BK, tile * BN + rank * (BN / 2), in_first_cta(&full[s]));
                    }
            }
            // the CTA stays until the first CTA's last commits have arrived in its shared memory
            for (int n = 0; n < STAGES && ok; ++n, ++it)
                if (!mbar_wait(&empty[it % STAGES], ((it / STAGES) & 1) ^ 1, abort_flag)) { ok = false; atomicExch(status, 43); }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            // D = f32, A = B = bf16, both K-major, N = 256, M = 256 of the pair
            constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((2 * BM) >> 4) << 24);
            uint32_t it = 0, local = 0;
            bool ok = true;
            for (int unit = pair; unit < units && ok; unit += pairs)
                for (int tile = first_tile(unit); tile < last_tile(unit) && ok; ++tile, ++local) {
                    const int buf = local & 1;
                    if (!mbar_wait(&acc_empty[buf], ((local >> 1) & 1) ^ 1, abort_flag)) { ok = false; atomicExch(status, 44); break; }
                    tc_fence_after();
                    for (int kb = 0; kb < num_kb; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (!mbar_wait(&full[s], (it / STAGES) & 1, abort_flag)) { ok = false; atomicExch(status, 45); break; }
                        tc_fence_after();
                        const uint32_t at = smem_u32(tiles + (size_t)s * STAGE_BYTES);
                        const uint64_t desc_a = umma_desc(at), desc_b = umma_desc(at + BM * BK * 2);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_pair(tmem_base + (uint32_t)(buf * BN), desc_a + 2 * k, desc_b + 2 * k, idesc, (kb | k) ? 1u : 0u);
                        commit_pair(&empty[s]);
                    }
                    if (ok) commit_pair(&acc_full[buf]);
                }
        }
    } else {
        // ---- rows: lane l of quarter q is row 32 q + l of the CTA's 128; team t takes tokens 32 t + 128 i .. + 31 of a tile
        const int quarter = warp & 3, team = (warp - 2) >> 2;
        uint32_t local = 0;
        bool ok = true;
        // a thread's entries, its own column of the array (8-byte places side by side: no bank conflicts)
        unsigned long long* held = reinterpret_cast<unsigned long long*>(tiles + (size_t)STAGES * STAGE_BYTES + 256) + (threadIdx.x - 64);
        int holds = 0;
        auto send = [&](long long m) {
            if (holds) {
                const int place = atomicAdd(out.count + m, holds);
                for (int i = 0; i < holds; ++i)
                    if (place + i < LIST) out.list[m * LIST + place + i] = held[i * ROW_THREADS];
                holds = 0;
            }
        };
        targets = pdl_fresh(targets);
        for (int unit = pair; unit < units && ok; unit += pairs) {
            const long long m = (long long)(unit / strips) * 2 * BM + rank * BM + quarter * 32 + lane;
            const bool there = m < M;
            const int target = there ? targets[m] : -1;
            const float limit = TOP && there ? pdl_fresh(out.limit)[m] : INFINITY;
            const int limit_index = TOP && there ? pdl_fresh(out.limit_index)[m] : 0;
            Sums mine = {-INFINITY, 0.f, 0.f};
            for (int tile = first_tile(unit); tile < last_tile(unit); ++tile, ++local) {
                const int buf = local & 1;
                if (!mbar_wait(&acc_full[buf], (local >> 1) & 1, abort_flag)) { ok = false; if (lane == 0) atomicExch(status, 46); break; }
                tc_fence_after();
                const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN);
#pragma unroll 1
                for (int c = 32 * team; c < BN; c += 32 * TEAMS) {
                    uint32_t raw[32];
                    tmem_ld32(taddr + c, raw);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    const int n = tile * BN + c;
                    // this team's last read of the accumulator is done (one arrival a warp: those of its lanes take turns at the barrier)
                    auto release = [&]() {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_remote(in_first_cta(&acc_empty[buf]));
                    };
                    if (n >= N) {
                        if (c + 32 * TEAMS >= BN) release();
                        continue;
                    }
                    if (!TOP && c + 32 * TEAMS >= BN) release();
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(raw[j]);
                    if (n + 32 > N)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (n + j >= N) x[j] = -INFINITY;
                    float big[4] = {x[0], x[8], x[16], x[24]};
#pragma unroll
                    for (int j = 0; j < 32; ++j) big[j >> 3] = fmaxf(big[j >> 3], x[j]);
                    const float most = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
                    if (most > mine.m) {
                        const float moved = fmaxf(mine.m - most, LEAST), shrink = __expf(moved);
                        mine.w = shrink * (mine.w + moved * mine.s);
                        mine.s *= shrink;
                        mine.m = most;
                    }
                    const float base = mine.m == -INFINITY ? 0.f : mine.m;
                    const unsigned long long less = pair_of(-base, -base), log2e = pair_of(1.4426950408889634f, 1.4426950408889634f);
                    unsigned long long sa = 0ull, sb = 0ull, wa = 0ull, wb = 0ull;            // (pairs of zeros)
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const unsigned long long da = pair_add(pair_of(x[j], x[j + 1]), less), db = pair_add(pair_of(x[j + 2], x[j + 3]), less);
                        const unsigned long long ea = pair_ex2(pair_mul(da, log2e)), eb = pair_ex2(pair_mul(db, log2e));
                        sa = pair_add(sa, ea);
                        sb = pair_add(sb, eb);
                        wa = pair_fma(ea, da, wa);
                        wb = pair_fma(eb, db, wb);
                    }
                    float s0, s1, w0, w1;
                    pair_split(pair_add(sa, sb), s0, s1);
                    pair_split(pair_add(wa, wb), w0, w1);
                    float s_more = s0 + s1, w_more = w0 + w1;
                    if (w_more != w_more && s_more == s_more) {    // minus infinity among the logits: 0 times it is to be 0
                        w_more = 0.f;
#pragma unroll 1
                        for (int first = 0; first < 32; first += 8) {
#pragma unroll
                            for (int part = 0; part < 4; ++part)
                                if (first == 8 * part)
#pragma unroll
                                    for (int j = 8 * part; j < 8 * part + 8; ++j)
                                        w_more = fmaf(__expf(x[j] - base), fmaxf(x[j] - base, LEAST), w_more);
                        }
                    }
                    mine.s += s_more;
                    mine.w += w_more;
                    if ((unsigned)(target - n) < 32u)
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (target == n + j) out.given[m] = x[j];
                    if constexpr (TOP) {
                        // The eights in which some row of the warp has a number for its list, read once more: eight places in the program instead of 32,
                        // whose 20 KB of instructions were fetched anew for nearly every number.
                        unsigned parts = 0;
#pragma unroll
                        for (int part = 0; part < 4; ++part) parts |= __any_sync(0xffffffffu, big[part] >= limit) ? 1u << part : 0u;
#pragma unroll 1
                        for (; parts; parts &= parts - 1) {
                            const int first = 8 * (__ffs(parts) - 1);
                            uint32_t eight[8];
                            tmem_ld8(taddr + c + first, eight);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float v = __uint_as_float(eight[j]);
                                const int token = n + first + j;
                                if (v >= limit && (v > limit || token < limit_index) && token < N) {
                                    held[holds * ROW_THREADS] = ((unsigned long long)eight[j] << 32) | (uint32_t)token;
                                    ++holds;
                                }
                            }
                            if (__any_sync(0xffffffffu, holds > HELD - 8) && there) send(m);
                        }
                    }
                    if (TOP && c + 32 * TEAMS >= BN) release();
                }
            }
            if constexpr (TOP) {
                if (there) send(m);
            }
            if (ok && there) {
                float* to = out.sums + ((m * strips + unit % strips) * TEAMS + team) * 3;
                to[0] = mine.m;
                to[1] = mine.s;
                to[2] = mine.w;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    // (a CTA that gave up a wait may be in front of the other's use of its memory: both come here)
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * BN) : "memory");
    }
}

// One CTA a row. x / table: for a row whose list did not hold all.
__global__ void __launch_bounds__(NT)
join_kernel(const int* __restrict__ targets, int V, int strips, int top, Scratch in, Results out, const __nv_bfloat16* __restrict__ x, long long x_stride,
            const __nv_bfloat16* __restrict__ table, long long table_stride, int K, int* __restrict__ status) {
    __shared__ unsigned long long entry_s[CAPACITY], kept_s[MOST_TOP];
    __shared__ uint32_t group_s[GROUPS], limit_s, bound_s;
    __shared__ int count_s;
    __shared__ float logit_s[CHUNK];
    pdl_prologue();
    in.sums = pdl_fresh(in.sums);
    in.list = pdl_fresh(in.list);
    in.count = pdl_fresh(in.count);
    in.given = pdl_fresh(in.given);
    const long long r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const List list = {entry_s, kept_s, &count_s, &limit_s, group_s, &bound_s};
    if (top) {
        const int count = in.count[r];
        const bool whole = count >= top && count <= LIST;
        if (tid == 0) { count_s = whole ? count : 0; limit_s = 0; }
        if (whole) {
            for (int i = tid; i < count; i += NT) {
                const unsigned long long entry = in.list[r * LIST + i];
                entry_s[i] = entry_of(order_of(__uint_as_float((uint32_t)(entry >> 32))), (int)(uint32_t)entry);
            }
            __syncthreads();
            rank<NT>(list, top);
        } else {
            __syncthreads();
            for (int chunk = 0; chunk < V; chunk += CHUNK) {
                const int end = min(V, chunk + CHUNK);
                for (int token = chunk + warp; token < end; token += NT / 32) {
                    float sum = 0.f;
                    for (int k = lane; k < K; k += 32)
                        sum = fmaf(__bfloat162float(x[r * x_stride + k]), __bfloat162float(table[token * table_stride + k]), sum);
                    sum = warp_sum(sum);
                    if (lane == 0) logit_s[token - chunk] = sum;
                }
                __syncthreads();
                float v[PER], big = -INFINITY;
#pragma unroll
                for (int u = 0; u < PER; ++u) {
                    const int i = u * NT + tid;
                    v[u] = chunk + i < end ? logit_s[i] : -INFINITY;
                    big = fmaxf(big, v[u]);
                }
                consider<NT>(list, v, big, top, [&](int u) { const int i = chunk + u * NT + tid; return i < end ? i : -1; });
                __syncthreads();
            }
            rank<NT>(list, top);
        }
    }
    // the strips' sums, by the first warp
    Sums all = {-INFINITY, 0.f, 0.f};
    if (warp == 0) {
        for (int i = lane; i < TEAMS * strips; i += 32) {
            const float* one = in.sums + (r * TEAMS * strips + i) * 3;
            all = joined(all, Sums{one[0], one[1], one[2]});
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Sums other = {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o), __shfl_xor_sync(0xffffffffu, all.w, o)};
            all = joined(all, other);
        }
        const float log_s = logf(all.s), base = all.m == -INFINITY ? 0.f : all.m;
        if (lane == 0) {
            const int y = targets[r];
            float given = __uint_as_float(0x7fffffffu);
            if (y == -1) given = 0.f;
            else if (y >= 0 && y < V) given = (in.given[r] - base) - log_s;
            else if (status) atomicExch(status, 41);
            out.logprob[r] = given;
            out.entropy[r] = log_s - all.w / all.s;
        }
        if (lane < top) {
            const unsigned long long entry = entry_s[lane];
            out.top_logprob[r * top + lane] = (value_of(order_in(entry)) - base) - log_s;
            out.top_id[r * top + lane] = index_in(entry);
        }
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult result;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &result) == cudaSuccess &&
                       result == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
    }();
    return fn;
}
// rows x cols bfloat16, row pitch ld; boxes of 128 rows x 64 columns, 128-byte swizzle, zeros outside
static bool make_map(CUtensorMap* map, const void* base, long long rows, int cols, long long ld) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)BM}, elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// how a vocabulary is cut into strips: so that all pairs of CTAs end about together
static int strips_for(int tiles_m, int tiles_n, int pairs) {
    int best = 1;
    long long least = 1ll << 60;
    for (int s = 1; s <= tiles_n && s <= pairs; ++s) {
        const long long rounds = ((long long)tiles_m * s + pairs - 1) / pairs, time = rounds * ((tiles_n + s - 1) / s) * 64 + s;
        if (time < least) { least = time; best = s; }
    }
    return best;
}

}  // namespace headlp
}  // namespace ps

// The strips that ps_head_logprobs takes for these sizes (its `strips` argument; the scratch is sized by it); 0 where it does not take them.
PS_EXPORT int ps_head_logprobs_strips(int rows, int V) {
    using namespace ps::headlp;
    if (rows <= 0 || V <= 0) return 0;
    const int tiles_m = (rows + 2 * BM - 1) / (2 * BM), tiles_n = (V + BN - 1) / BN;
    return strips_for(tiles_m, tiles_n, 74);
}

// x [rows, K], table [V, K] bfloat16, row pitches multiples of 8, 16-byte aligned.  top 0: no sample.  Otherwise sample [rows, n] (pitch ld): the
// logits of tokens 0, every, 2 every, ..; list [rows, 2048], count, limit, limit_index [rows].  sums [rows, 4 * strips, 3], given [rows].
PS_EXPORT int ps_head_logprobs(const void* x, long long x_stride, const void* table, long long table_stride, int rows, int V, int K,
                               const int* targets, int top, const float* sample, long long ld, int n, int every, float* sums, float* given,
                               unsigned long long* list, int* count, float* limit, int* limit_index, int strips, float* logprob, float* entropy,
                               float* top_logprob, int* top_id, int* status, void* stream) {
    using namespace ps::headlp;
    if (rows <= 0) return PS_OK;
    if (!x || !table || !targets || !sums || !given || !logprob || !entropy || !status || V <= 0 || K <= 0 || top < 0 || top > V) return PS_ERR_BAD_ARGUMENT;
    if (top && (!sample || !list || !count || !limit || !limit_index || !top_logprob || !top_id || every <= 0 || n < top || n != (V + every - 1) / every ||
                ld < n))
        return PS_ERR_BAD_ARGUMENT;
    if (top > MOST_TOP || K % 8 || x_stride % 8 || table_stride % 8 || (((uintptr_t)x | (uintptr_t)table) & 15)) return PS_ERR_UNSUPPORTED;
    if (strips != ps_head_logprobs_strips(rows, V)) return PS_ERR_BAD_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const Scratch scratch = {sums, given, list, count, limit, limit_index};
    const ps::logprob::Results out = {logprob, entropy, top_logprob, top_id};
    if (top) {
        const int rc = ps::launch_pdl(sample_kernel, dim3(rows), dim3(NT), 0, s, sample, ld, n, every, top, scratch);
        if (rc) return rc;
    }
    CUtensorMap map_x, map_w;
    if (!make_map(&map_x, x, rows, K, x_stride) || !make_map(&map_w, table, V, K, table_stride)) return PS_ERR_LAUNCH;
    const int tiles_m = (rows + 2 * BM - 1) / (2 * BM), tiles_n = (V + BN - 1) / BN, pairs = tiles_m * strips < 74 ? tiles_m * strips : 74;
    auto kernel = top ? product_kernel<true> : product_kernel<false>;
    static size_t raised[2][ps::MAX_DEVICES] = {{0}, {0}};
    const size_t smem = top ? smem_bytes<true>() : smem_bytes<false>();
    if (!ps::ensure_dynamic_smem((const void*)kernel, smem, raised[top ? 1 : 0])) return PS_ERR_LAUNCH;
    int rc = ps::launch_pdl_clusters(kernel, dim3(2 * pairs), dim3(HEAD_THREADS), smem, s, dim3(2, 1, 1), map_x, map_w, targets, rows, V, K, strips,
                                     (tiles_n + strips - 1) / strips, scratch, status);
    if (rc) return rc;
    return ps::launch_pdl(join_kernel, dim3(rows), dim3(NT), 0, s, targets, V, strips, top, scratch, out, (const __nv_bfloat16*)x, x_stride,
                          (const __nv_bfloat16*)table, table_stride, K, status);
}
