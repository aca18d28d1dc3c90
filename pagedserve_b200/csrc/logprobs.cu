// What a row of logits says about given tokens: for row x and its token y, with m = max x, S = sum e^(x - m), W = sum e^(x - m) (x - m),
//   log probability  x_y - m - log S,      entropy  log S - W / S,      and the `top` largest log probabilities with their tokens,
// of equal logits the lower index first.  A token of -1 is none: its log probability is 0.  One outside the vocabulary sets *status and gets NaN.
// A NaN or +infinity among the logits makes a row's numbers NaN; -infinity is a token of probability 0.  NaN comes behind all others in the order.
//
// One pass over a row, which is all its traffic: a thread has 8 numbers of a chunk (2,048; 4,096 in CTAs of 512 threads), two pieces of 16 bytes, the next two on their way.  m, S and W are kept by
// thread, W moved to a new maximum m' by W' = e^(m - m') (W + (m - m') S).  Sums are float32, of about 200 numbers a thread and
// then of the threads by halving exchanges.
//
// The largest: 64 groups of a chunk's numbers (32 each; 64 in CTAs of 512 threads) give their largest; the `top`-th of those is a bound that at least `top` numbers of the first chunk
// reach, and hardly more than twice as many do.  These go to a list, which is ranked (each entry counts those in front of it).  From then
// on only numbers beyond the list's last join it, about top * (chunk size) / (numbers so far) a chunk, without a barrier; the list is looked at every four chunks and
// ranked when it has grown by RANK_AT entries (a look at every chunk cost 60 us of 164 with 2,047 rows and 5 alternatives).  Where more joined than it
// holds (rising logits), the four chunks are read once more, each behind a bound of its own, which adds at most a chunk's numbers.
//
// A row is one CTA, or the CTAs of a cluster that share its columns out (few rows).
//
// What bounds it, rows of 50,257: without alternatives the bytes (2,047 rows, 412 MB: 74 us, 5.6 TB/s); with them the list, its looks and rankings (5
// alternatives 121 us, 20 131, 32 145); 8 rows 10.3 us, one trip through a share's eighth of a row and the shares' join.
#include "logprobs.cuh"

namespace ps {
namespace logprob {

// What a kernel with a list has in shared memory (its dynamic part: with 1,024 threads more than the static part may be).
template <int NT>
struct ListMemory {
    unsigned long long entry[capacity<NT>()], kept[MOST_TOP];
    uint32_t group[GROUPS], limit, bound;
    int count, overflow;
};
constexpr int TOGETHER = 4;                                        // chunks between two looks at the list

template <int NT, bool TOP>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1)
logprobs_kernel(const float* __restrict__ logits, long long ld, int V, const int* __restrict__ targets, int top, Results out,
                int* __restrict__ status) {
    constexpr int CHUNK = NT * PER, CAPACITY = capacity<NT>();
    extern __shared__ __align__(16) unsigned char memory[];
    ListMemory<NT>& own = *reinterpret_cast<ListMemory<NT>*>(memory);
    __shared__ Sums warp_s[NT / 32];
    __shared__ float share_s[3];
    pdl_prologue();
    logits = pdl_fresh(logits);
    targets = pdl_fresh(targets);
    const long long r = blockIdx.x;
    const int share = blockIdx.z, shares = gridDim.z, tid = threadIdx.x;
    const float* row = logits + r * ld;
    // Pieces of 16 bytes: a piece begins `shift` numbers in front of an index that is a multiple of four.
    const int shift = (int)(((uintptr_t)row >> 2) & 3);
    const int per_share = ((V + shares - 1) / shares + 31) / 32 * 32;
    const int begin = min(V, share * per_share), end = min(V, begin + per_share);
    const List list = {own.entry, own.kept, &own.count, &own.limit, own.group, &own.bound};
    if (TOP && tid == 0) {
        own.count = own.overflow = 0;
        own.limit = 0;
    }
    if (TOP) __syncthreads();

    Sums mine = {-INFINITY, 0.f, 0.f};
    float x[PER], next[PER];
    auto index = [&](int chunk, int u) {                           // of a thread's u-th number, below 0: there is none
        const int i = chunk + (u >> 2) * (NT * 4) + tid * 4 + (u & 3) - shift;
        return i >= begin && i < end ? i : -1;
    };
    auto fetch = [&](int chunk, float (&v)[PER]) {
#pragma unroll
        for (int u = 0; u < PER; u += 4) {
            const int i = chunk + (u >> 2) * (NT * 4) + tid * 4 - shift;
            if (i >= begin && i + 3 < end) {
                const float4 four = *reinterpret_cast<const float4*>(row + i);
                v[u] = four.x; v[u + 1] = four.y; v[u + 2] = four.z; v[u + 3] = four.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[u + j] = i + j >= begin && i + j < end ? row[i + j] : -INFINITY;
            }
        }
    };
    auto largest = [&](const float (&v)[PER]) {
        float big = v[0];
#pragma unroll
        for (int u = 1; u < PER; ++u) big = fmaxf(big, v[u]);
        return big;
    };
    fetch(begin, next);
    int together = 0, settled = 0;                                 // chunks since the list was looked at, its entries then
    const int stop = end > begin ? end + shift : begin;
    for (int chunk = begin; chunk < stop; chunk += CHUNK) {
#pragma unroll
        for (int u = 0; u < PER; ++u) x[u] = next[u];
        if (chunk + CHUNK < stop) fetch(chunk + CHUNK, next);
        const float big = largest(x);
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
        if constexpr (TOP) {
            const uint32_t limit = own.limit;
            if (limit <= 1u) {                                    // (the same for all: it changes between barriers)
                consider<NT>(list, x, big, top, [&](int u) { return index(chunk, u); });
                __syncthreads();
                settled = own.count;
                __syncthreads();
                continue;
            }
            if (order_of(big) > limit) {
#pragma unroll
                for (int u = 0; u < PER; ++u) {
                    const uint32_t order = order_of(x[u]);
                    if (order > limit) {                          // (what is not there is minus infinity, which is beyond no limit)
                        const int place = atomicAdd(&own.count, 1);
                        if (place < CAPACITY) own.entry[place] = entry_of(order, index(chunk, u));
                        else own.overflow = 1;
                    }
                }
            }
            if (++together < TOGETHER && chunk + CHUNK < stop) continue;
            __syncthreads();
            const int count = own.count;
            const bool again = own.overflow != 0;
            __syncthreads();
            if (again) {                                          // rising logits: chunk by chunk, behind a bound of its own for each
                if (tid == 0) {
                    own.count = settled;
                    own.overflow = 0;
                }
                __syncthreads();
                for (int c = chunk - (together - 1) * CHUNK; c <= chunk; c += CHUNK) {
                    float v[PER];
                    fetch(c, v);
                    consider<NT>(list, v, largest(v), top, [&](int u) { return index(c, u); });
                    __syncthreads();
                }
                rank<NT>(list, top);
            } else if (count > top + RANK_AT) {
                rank<NT>(list, top);
            }
            settled = own.count;
            together = 0;
            __syncthreads();
        }
    }
    // the threads' sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums other = {__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.w, o)};
        mine = joined(mine, other);
    }
    if ((tid & 31) == 0) warp_s[tid >> 5] = mine;
    __syncthreads();
    if (TOP) rank<NT>(list, top);
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
                    if (k < (int)ld_cluster_u32(&own.count, c)) list.entry[atomicAdd(&own.count, 1)] = ld_cluster_u64(&own.entry[k], c);
                }
                __syncthreads();
                rank<NT>(list, top);
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

template <int NT, bool TOP>
int launch(const float* logits, long long ld, int rows, int V, const int* targets, int top, const Results& out, int* status, int shares, cudaStream_t s) {
    constexpr size_t SMEM = TOP ? sizeof(ListMemory<NT>) : 0;
    static size_t raised[MAX_DEVICES] = {0};
    if (!ensure_dynamic_smem((const void*)logprobs_kernel<NT, TOP>, SMEM, raised)) return PS_ERR_LAUNCH;
    return launch_pdl_cluster(logprobs_kernel<NT, TOP>, dim3(rows, 1, shares), dim3(NT), SMEM, s, shares, logits, ld, V, targets, top, out, status);
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
    const Results out = {logprob, entropy, top_logprob, top_id};
    // Few rows: eight CTAs of 512 threads for each (8 rows of 50,257, 5 alternatives: 10.2 us; with 256 threads 11.4, with 1,024 14.0).
    // Many: CTAs of 256 threads, enough of them that all SMs have as many as they hold, with the registers that ranking wants (2,047 rows, 5 alternatives:
    // four CTAs on an SM 124 us, six with 40 registers a thread 160).
    cudaStream_t s = (cudaStream_t)stream;
    const bool wide = rows <= 18 && V > 8192;
    const int shares = wide ? 8 : V > 4096 ? (rows <= 148 ? 8 : rows <= 444 ? 4 : rows <= 888 ? 2 : 1) : 1;
    if (wide) return top ? launch<512, true>(logits, ld, rows, V, targets, top, out, status, shares, s)
                         : launch<512, false>(logits, ld, rows, V, targets, top, out, status, shares, s);
    return top ? launch<256, true>(logits, ld, rows, V, targets, top, out, status, shares, s)
               : launch<256, false>(logits, ld, rows, V, targets, top, out, status, shares, s);
}
