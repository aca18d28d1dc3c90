// What a row of logits says about given tokens: for row x and its token y, with m = max x, S = sum e^(x - m), W = sum e^(x - m) (x - m),
//   log probability  x_y - m - log S,      entropy  log S - W / S,      and the `top` largest log probabilities with their tokens,
// of equal logits the lower index first.  A token of -1 is none: its log probability is 0.  One outside the vocabulary sets *status and gets NaN.
// A NaN or +infinity among the logits makes a row's numbers NaN; -infinity is a token of probability 0.  NaN comes behind all others in the order.
//
// One pass over a row, which is all its traffic: a thread has 8 numbers of a chunk of 2,048, the next 8 on their way.  m, S and W are kept by
// thread, W moved to a new maximum m' by W' = e^(m - m') (W + (m - m') S).  Sums are float32, of about 200 numbers a thread and
// then of the threads by halving exchanges.
//
// The largest: 64 groups of 32 numbers each give their largest; the `top`-th of those is a bound that at least `top` numbers of the chunk
// reach, and hardly more than twice as many do.  These go to a list, which is ranked (each entry counts those in front of it).  From then
// on only numbers beyond the list's last join it, about top * (chunk size) / (numbers so far) a chunk, and the list is ranked again when it has grown by
// RANK_AT entries.  Rows on which more than 32 threads of a chunk find one (rising logits) go through the bound again, so that the list holds them:
// a chunk adds at most its 2,048 numbers.
//
// A row is one CTA, or the CTAs of a cluster that share its columns out (few rows).
#include "logprobs.cuh"

namespace ps {
namespace logprob {

template <bool TOP>
__global__ void __launch_bounds__(NT)
logprobs_kernel(const float* __restrict__ logits, long long ld, int V, const int* __restrict__ targets, int top, Results out,
                int* __restrict__ status) {
    __shared__ unsigned long long entry_s[TOP ? CAPACITY : 1], kept_s[TOP ? MOST_TOP : 1];
    __shared__ uint32_t group_s[TOP ? GROUPS : 1], limit_s, bound_s;
    __shared__ int count_s;
    __shared__ Sums warp_s[NT / 32];
    __shared__ float share_s[3];
    pdl_prologue();
    logits = pdl_fresh(logits);
    targets = pdl_fresh(targets);
    const long long r = blockIdx.x;
    const int share = blockIdx.z, shares = gridDim.z, tid = threadIdx.x;
    const float* row = logits + r * ld;
    const int per_share = ((V + shares - 1) / shares + CHUNK - 1) / CHUNK * CHUNK;
    const int begin = min(V, share * per_share), end = min(V, begin + per_share);
    const List list = {entry_s, kept_s, &count_s, &limit_s, group_s, &bound_s};
    if (TOP && tid == 0) { count_s = 0; limit_s = 0; }
    if (TOP) __syncthreads();

    Sums mine = {-INFINITY, 0.f, 0.f};
    float x[PER], next[PER];
    auto fetch = [&](int chunk, float (&v)[PER]) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int i = chunk + u * NT + tid;
            v[u] = i < end ? row[i] : -INFINITY;
        }
    };
    fetch(begin, next);
    for (int chunk = begin; chunk < end; chunk += CHUNK) {
#pragma unroll
        for (int u = 0; u < PER; ++u) x[u] = next[u];
        if (chunk + CHUNK < end) fetch(chunk + CHUNK, next);
        float big = x[0];
#pragma unroll
        for (int u = 1; u < PER; ++u) big = fmaxf(big, x[u]);
        const float m_new = fmaxf(mine.m, big), base = m_new == -INFINITY ? 0.f : m_new, moved = from_to(mine.m, base), shrink = __expf(moved);
        mine.w = shrink * (mine.w + moved * mine.s);
        mine.s *= shrink;
        mine.m = m_new;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const float d = x[u] - base, e = __expf(d);
            mine.s += e;                                          // (NaN where x is NaN or +infinity)
            mine.w = fmaf(e, fmaxf(d, LEAST), mine.w);
        }
        if (TOP) consider(list, x, chunk, end, big, top);
    }
    // the threads' sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums other = {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.w, o)};
        mine = joined(mine, other);
    }
    if ((tid & 31) == 0) warp_s[tid >> 5] = mine;
    __syncthreads();
    if (TOP) rank(list, top);
    Sums all = warp_s[0];
    for (int w = 1; w < NT / 32; ++w) all = joined(all, warp_s[w]);
    if (shares > 1) {
        if (tid == 0) { share_s[0] = all.m; share_s[1] = all.s; share_s[2] = all.w; }
        cluster_sync_all();
        if (share == 0) {
            for (int c = 1; c < shares; ++c) {
                const Sums other = {ld_cluster_f32(&share_s[0], c), ld_cluster_f32(&share_s[1], c), ld_cluster_f32(&share_s[2], c)};
                all = joined(all, other);
            }
            if (TOP) {
                // (the first share's entries are in place; the others' follow them)
                for (int i = tid; i < (shares - 1) * top; i += NT) {
                    const int c = 1 + i / top, k = i % top;
                    if (k < (int)ld_cluster_u32(&count_s, c)) list.entry[atomicAdd(&count_s, 1)] = ld_cluster_u64(&entry_s[k], c);
                }
                __syncthreads();
                rank(list, top);
            }
        }
    }
    if (share == 0) {
        const float log_s = logf(all.s), base = all.m == -INFINITY ? 0.f : all.m;
        if (tid == 0) {
            const int y = targets[r];
            float given = __uint_as_float(0x7fffffffu);
            if (y == -1) given = 0.f;
            else if (y >= 0 && y < V) given = (row[y] - base) - log_s;
            else if (status) atomicExch(status, 41);
            out.logprob[r] = given;
            out.entropy[r] = log_s - all.w / all.s;
        }
        if (TOP && tid < top) {
            const unsigned long long entry = list.entry[tid];
            out.top_logprob[r * top + tid] = (value_of(order_in(entry)) - base) - log_s;
            out.top_id[r * top + tid] = index_in(entry);
        }
    }
    if (shares > 1) cluster_sync_all();                            // the shares stay until they were read
}

}  // namespace logprob
}  // namespace ps

// logits: rows of V numbers, ld apart.  top: 0 to 32, at most V.
PS_EXPORT int ps_token_logprobs(const float* logits, long long ld, int rows, int V, const int* targets, int top, float* logprob, float* entropy,
                                float* top_logprob, int* top_id, int* status, void* stream) {
    using namespace ps::logprob;
    if (rows <= 0) return PS_OK;
    if (!logits || !targets || !logprob || !entropy || V <= 0 || ld < V || top < 0 || top > V) return PS_ERR_BAD_ARGUMENT;
    if (top > MOST_TOP) return PS_ERR_UNSUPPORTED;
    if (top && (!top_logprob || !top_id)) return PS_ERR_BAD_ARGUMENT;
    int shares = V > 2 * CHUNK ? (rows <= 148 ? 8 : rows <= 444 ? 4 : rows <= 888 ? 2 : 1) : 1;
    const Results out = {logprob, entropy, top_logprob, top_id};
    return ps::launch_pdl_cluster(top ? logprobs_kernel<true> : logprobs_kernel<false>, dim3(rows, 1, shares), dim3(NT), 0, (cudaStream_t)stream,
                                  shares, logits, ld, V, targets, top, out, status);
}
