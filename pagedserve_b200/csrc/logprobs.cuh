// Shared by the kernels that find log probabilities: sums of a row of logits as they come, and the list of its largest (logprobs.cu says how).
#pragma once

#include "common.cuh"

namespace ps {
namespace logprob {

constexpr int PER = 8, MOST_TOP = 32, RANK_AT = 128, GROUPS = 64;      // (a chunk: PER numbers of every thread of a CTA, NT of them)
constexpr int DIRECT = 32;                                       // threads of a chunk that may add what they have without a new bound
constexpr int THIN_FROM = 96;                                    // entries of a list from which the bound is applied to it, too
template <int NT> constexpr int capacity() { return MOST_TOP + RANK_AT + NT * PER; }
constexpr float LEAST = -1000.f;                                  // e^LEAST is 0, and LEAST times that too

// whole numbers in the order of the floats; 1: a NaN, behind everything; 0: nothing there
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 1u;
    const uint32_t bits = __float_as_uint(x + 0.0f);              // (-0 and 0 are equal)
    return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    if (order <= 1u) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
// order and index as one number: the larger one comes first
__device__ __forceinline__ unsigned long long entry_of(uint32_t order, int index) {
    return ((unsigned long long)order << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t order_in(unsigned long long entry) { return (uint32_t)(entry >> 32); }
__device__ __forceinline__ int index_in(unsigned long long entry) { return (int)~(uint32_t)entry; }

struct Sums {
    float m, s, w;
};
__device__ __forceinline__ float from_to(float m, float base) { return fmaxf(m - base, LEAST); }
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float base = r.m == -INFINITY ? 0.f : r.m, da = from_to(a.m, base), db = from_to(b.m, base), ea = __expf(da), eb = __expf(db);
    r.s = a.s * ea + b.s * eb;
    r.w = ea * (a.w + da * a.s) + eb * (b.w + db * b.s);
    return r;
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(const unsigned long long* local, int rank) {
    uint32_t remote;
    unsigned long long v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote) : "memory");
    return v;
}

struct Results {
    float* logprob;
    float* entropy;
    float* top_logprob;         // [rows, top]
    int* top_id;
};

// The list of a CTA: entries [0, count), of which the first `top` are ranked after rank().
struct List {
    unsigned long long* entry;  // [capacity]
    unsigned long long* kept;   // [MOST_TOP]
    int* count;
    uint32_t* limit;            // an entry joins if its order is beyond this one (0: the list has fewer than `top`)
    uint32_t* group;            // [GROUPS]
    uint32_t* bound;
};
// Sets *list.bound to a number's order that at least `top` of the numbers in hand reach, or to 0; `most`: the largest order of this thread's (0:
// it has none).  All threads; ends with the bound visible.
template <int NT>
__device__ __forceinline__ void find_bound(const List& list, uint32_t most, int top) {
    constexpr int LANES = NT / GROUPS;                            // threads of a group
    const int tid = threadIdx.x;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (tid % LANES == 0) list.group[tid / LANES] = most;
    __syncthreads();
    if (tid < GROUPS) {
        const uint32_t own = list.group[tid];
        int before = 0;
        for (int o = 0; o < GROUPS; ++o) before += list.group[o] > own || (list.group[o] == own && o < tid);
        if (before == top - 1) *list.bound = own;
    }
    __syncthreads();
}
// all threads; begins and ends with the list complete and visible
template <int NT>
__device__ __forceinline__ void rank(const List& list, int top) {
    int n = *list.count;
    if (n > THIN_FROM) {                                          // a long list: what is below the bound goes first
        constexpr int EACH = (capacity<NT>() + NT - 1) / NT;
        unsigned long long mine[EACH];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = i * NT + threadIdx.x;
            mine[i] = at < n ? list.entry[at] : 0ull;
            most = max(most, order_in(mine[i]));
        }
        find_bound<NT>(list, most, top);                          // (everyone has read its entries)
        if (threadIdx.x == 0) *list.count = 0;
        __syncthreads();
        const uint32_t from = max(*list.bound, 1u);
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (order_in(mine[i]) >= from) list.entry[atomicAdd(list.count, 1)] = mine[i];
        __syncthreads();
        n = *list.count;
    }
    for (int i = threadIdx.x; i < n; i += NT) {
        const unsigned long long mine = list.entry[i];
        int before = 0;
        for (int o = 0; o < n; ++o) before += list.entry[o] > mine;
        if (before < top) list.kept[before] = mine;
    }
    __syncthreads();
    if (threadIdx.x < top && (int)threadIdx.x < n) list.entry[threadIdx.x] = list.kept[threadIdx.x];
    if (threadIdx.x == 0) {
        *list.count = min(n, top);
        *list.limit = n >= top ? order_in(list.kept[top - 1]) : 0u;
    }
    __syncthreads();
}

// The numbers of a chunk, PER of each thread, to the list if they belong there; at(u): the index of the u-th of them, below 0 where there is none; `big`: the
// largest.  All threads.
template <int NT, typename At>
__device__ __forceinline__ void consider(const List& list, const float (&x)[PER], float big, int top, At at) {
    const uint32_t limit = *list.limit;
    const bool hit = limit <= 1u || order_of(big) > limit;        // (an open list takes everything)
    const int hits = __syncthreads_count(hit);
    if (hits == 0) return;
    uint32_t from = limit + 1;                                    // orders that join
    if (hits > DIRECT) {
        uint32_t most = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u)
            if (at(u) >= 0) most = max(most, order_of(x[u]));
        find_bound<NT>(list, most, top);
        from = max(from, max(*list.bound, 1u));
    }
    if (hit || hits > DIRECT) {
#pragma unroll
        for (int u = 0; u < PER; ++u)
            if (at(u) >= 0) {
                const uint32_t order = order_of(x[u]);
                if (order >= from) list.entry[atomicAdd(list.count, 1)] = entry_of(order, at(u));
            }
    }
    __syncthreads();
    if (hits > DIRECT || *list.count > top + RANK_AT) rank<NT>(list, top);
}

}  // namespace logprob
}  // namespace ps
