// Log probabilities of given tokens with rank, entropy and top alternatives, and their gradient (see pssa_b200_token_logprobs_dev).
//
// Forward: one read of the row. Every thread keeps the running maximum, sum exp and sum exp * z of its vectors, counts the logits
// above the target's, and remembers the vector of its maximum; the threads' and then the CTAs' numbers are joined in a fixed order.
// One logit equal to the row's maximum stays out of the sums all the way, and ln sum exp z is log1p of the rest: a row that is sure
// of one id has small numbers, and they keep their digits (0.1 to 0.3 us of a small call, 2 to 8 % of many short rows).
// A few rows are split over the CTAs of a cluster, which meet in distributed shared memory: one launch and no workspace whatever
// the shape. Times are the kernel's in a graph of launches. 4096 x 131072 bf16: 207 us, 5.2 TB/s, at 84 instructions for 8 logits and
// 77 % of the issue slots; 4096 x 65536 fp32, half the instructions a byte: 173 us, 6.2 TB/s, HBM. One row of 16384: 9.2 us, of
// which the launch of the cluster, two dependent trips for the target's logit and the choice of 20 alternatives.
//
// Alternatives come from the same pass. The n-th best of the maxima of pairs of neighbouring threads (64, 128 or 512 of them) bounds
// the n-th best logit from below, and no logit above the bound lies outside the n pairs that reach it: only their shares, n / pairs
// of the row, are read again, and what is not below the bound is ranked, each against each: hardly more than n logits where n is
// well below the pairs, some n ln n where all pairs reach it, every logit where fewer pairs than n have one (8000 x 1000 bf16:
// 5 alternatives 38 us, 48 54, 64 1360). Keys are (value, lower id first) and so never equal: ties change nothing. Where more pass
// than there is room for (logits in an order made for it), the n are drawn one by one instead.
//
// Gradient: elementwise with the forward call's maximum and log sum, one read and one write: 4096 x 65536 bf16 in 159 us, 6.8 TB/s.
#include <cooperative_groups.h>

#include <type_traits>

#include "kernels.hpp"
#include "logit_row.cuh"

namespace pssa {
namespace {

namespace cg = cooperative_groups;
using Key = unsigned long long;

constexpr int kRoom = 1024;  // candidates of a CTA
constexpr int kMaxCtas = 8;  // of a cluster

struct RowPart {  // a CTA's numbers for its cluster
    float top, ref, sum, ent;
    unsigned above;
    bool apart;  // of one logit equal to `ref`: it is not in `sum`
};
// `sum` relative to `to` >= `ref`, where the logit of `ref` is 1 no longer
__device__ __forceinline__ void raise_to(RowPart& p, float to, float c) {
    if (p.apart && p.ref < to) p.sum += 1.0f, p.apart = false;
    rebase(p.ref, to, c, p.sum, p.ent);
    p.ref = to;
}

template <int THREADS>
struct LogprobShared {
    RowPart part, parts[kMaxCtas];
    float f[3][THREADS / 32];
    unsigned u[THREADS / 32];  // how many are above; the highest bit: one stays apart
    Key bound, wide[THREADS / 32];
    int candidates;
    Key pairs[THREADS / 2];
    Key best[PSSA_B200_MAX_TOP];  // descending; 0 behind the last
    Key found[kRoom];
};

template <int THREADS, typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* scratch, F op) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
    for (int m = THREADS / 64; m > 0; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// The part of a row that a CTA reads: vectors [v0, v1) of it, and the elements outside any vector: in front by the first CTA, behind by the last.
template <typename T>
struct Part {
    const T* x;
    const uint4* vec;
    int head, v0, v1, tail0, n;
    bool first, last;
    __device__ Part(const T* row, int n_, int rank, int ctas) : x(row), n(n_), first(rank == 0), last(rank == ctas - 1) {
        head = head_of(row, n);
        const int vecs = (n - head) / kVec<T>, each = (vecs + ctas - 1) / ctas;
        vec = reinterpret_cast<const uint4*>(row + head);
        v0 = min(rank * each, vecs), v1 = min(v0 + each, vecs);
        tail0 = head + vecs * kVec<T>;
    }
    // this thread's single element: its id, or -1
    __device__ int single() const {
        if (first && (int)threadIdx.x < head) return threadIdx.x;
        const int i = (int)threadIdx.x - kVec<T>;  // behind the heads' threads
        return last && i >= 0 && i < n - tail0 ? tail0 + i : -1;
    }
};

// The n best keys of the CTA's part into s.best. `own`: the thread's best key (0: it has none).
template <typename T, int THREADS>
__device__ void best_of_part(const Part<T>& part, Key own, int n, LogprobShared<THREADS>& s) {
    constexpr int kPairs = THREADS / 2;
    const int tid = threadIdx.x, single = part.single();
    // the n-th best of the pairs' maxima
    const Key mate = __shfl_xor_sync(0xffffffffu, own, 1);
    if ((tid & 1) == 0) s.pairs[tid >> 1] = own > mate ? own : mate;
    if (tid == 0) s.bound = 0, s.candidates = 0;
    if (tid < PSSA_B200_MAX_TOP) s.best[tid] = 0;
    __syncthreads();
    if (tid < kPairs) {
        const Key k = s.pairs[tid];
        int better = 0;
        for (int i = 0; i < kPairs; ++i) better += s.pairs[i] > k;
        if (k != 0 && better == n - 1) s.bound = k;  // stays 0 where fewer pairs have a logit: then all are candidates
    }
    __syncthreads();
    const Key bound = s.bound;
    auto offer = [&](float x, int id) {
        const Key k = key_of(x, id);
        if (k >= bound) {
            const int at = atomicAdd(&s.candidates, 1);
            if (at < kRoom) s.found[at] = k;
        }
    };
    if (single >= 0) offer(to_f32(part.x[single]), single);
    // the shares of the pairs that reach the bound, dealt out anew: item (pair, vector of it)
    const int steps = (part.v1 - part.v0 + THREADS - 1) / THREADS;
    const float floor = bound == 0 ? -INFINITY : key_value(bound);
    __shared__ short s_list[kPairs];
    __shared__ int s_pairs;
    if (tid == 0) s_pairs = 0;
    __syncthreads();
    if (tid < kPairs && s.pairs[tid] != 0 && s.pairs[tid] >= bound) s_list[atomicAdd(&s_pairs, 1)] = (short)tid;
    __syncthreads();
    const int items = s_pairs * steps * 2;
    for (int i = tid; i < items; i += THREADS) {
        const int step = (i >> 1) % steps, p = s_list[(i >> 1) / steps], v = part.v0 + step * THREADS + 2 * p + (i & 1);
        if (v >= part.v1) continue;
        float x[kVec<T>];
        unpack<T>(part.vec[v], x);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
            if (x[e] >= floor) offer(x[e], part.head + v * kVec<T> + e);
    }
    __syncthreads();
    const int c = s.candidates;
    if (c <= kRoom) {
        for (int i = tid; i < c; i += THREADS) {
            const Key k = s.found[i];
            int better = 0;
            for (int j = 0; j < c; ++j) better += s.found[j] > k;
            if (better < n) s.best[better] = k;
        }
    } else {  // one by one; a thread looks its share over again when it has lost its best
        for (int r = 0; r < n; ++r) {
            const Key best = block_reduce<THREADS>(own, s.wide, [](Key a, Key b) { return a > b ? a : b; });
            if (tid == 0) s.best[r] = best;
            if (own == best && own != 0) {
                own = 0;
                auto look = [&](float x, int id) {
                    const Key k = key_of(x, id);
                    if (k < best && k > own) own = k;
                };
                for (int v = part.v0 + tid; v < part.v1; v += THREADS) {
                    float x[kVec<T>];
                    unpack<T>(part.vec[v], x);
#pragma unroll
                    for (int e = 0; e < kVec<T>; ++e) look(x[e], part.head + v * kVec<T> + e);
                }
                if (single >= 0) look(to_f32(part.x[single]), single);
            }
        }
    }
    __syncthreads();
}

template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 10 : THREADS == 256 ? 5 : 1) token_logprobs_kernel(LogprobParams p, int ctas) {
    __shared__ LogprobShared<THREADS> s;
    pdl_wait();  // launched while the kernel before it ends: 2 us a call (it does not start the next one early: 256 rows took 9.4 for 7.9)
    constexpr int kWarps = THREADS / 32, N = kVec<T>, kAhead = 4;
    const size_t row = blockIdx.x / (unsigned)ctas;
    const int rank = blockIdx.x % (unsigned)ctas, tid = threadIdx.x, warp = tid >> 5;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    const int v = p.vocab;
    const Part<T> part(x, v, rank, ctas);
    const float inv_t = 1.0f / p.temperature, c = kLog2e / p.temperature;
    const uint32_t t = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = t < (uint32_t)v, none = t == PSSA_B200_NO_TOKEN;
    const float xt = has ? to_f32(x[t]) : INFINITY;

    SoftmaxSums<true, TOP, true> sums;
    unsigned above = 0;
    auto take = [&](uint4 raw, int at, auto first) {
        float f[N];
        unpack<T>(raw, f);
        const float m = vector_max<T>(raw, f);
        if (m > xt) {
#pragma unroll
            for (int i = 0; i < N; ++i) above += f[i] > xt;
        }
        sums.template add<decltype(first)::value>(f, m, at, c);
    };
    const int one = part.single();
    const float single = one >= 0 ? to_f32(x[one]) : -INFINITY;
    int at = part.v0 + tid;
    {
        uint4 raw[kAhead];
        float m = single;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (at + i * THREADS < part.v1) raw[i] = part.vec[at + i * THREADS];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (at + i * THREADS < part.v1) {
                float f[N];
                unpack<T>(raw[i], f);
                m = fmaxf(m, vector_max<T>(raw[i], f));
            }
        sums.start(warp_max(m), c);
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (at + i * THREADS < part.v1) take(raw[i], at + i * THREADS, std::true_type());
        at += kAhead * THREADS;
    }
    for (; at + (kAhead - 1) * THREADS < part.v1; at += kAhead * THREADS) {
        uint4 raw[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) raw[i] = part.vec[at + i * THREADS];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) take(raw[i], at + i * THREADS, std::false_type());
    }
    for (; at < part.v1; at += THREADS) take(part.vec[at], at, std::false_type());
    Key own = 0;  // the thread's best logit
    if (TOP) {
        if (const int w = sums.where >= 0 ? sums.where : part.v0 + tid; w < part.v1) {  // without one above -inf, the lowest of its ids
            float f[N];
            unpack<T>(part.vec[w], f);
            int e = 0;
#pragma unroll
            for (int i = N - 1; i >= 0; --i)
                if (f[i] == sums.top) e = i;
            own = key_of(sums.top, part.head + w * N + e);
        }
        if (one >= 0) {
            const Key k = key_of(single, one);
            own = k > own ? k : own;
        }
    }
    if (one >= 0) {
        sums.add1(single, c);
        above += single > xt;
    }
    // the CTA's numbers
    const float ref = block_reduce<THREADS>(sums.ref, s.f[0], [](float a, float b) { return fmaxf(a, b); });
    const float top = block_reduce<THREADS>(sums.top, s.f[0], [](float a, float b) { return fmaxf(a, b); });
    float ent = sums.entropy_total();
    const unsigned apart = __ballot_sync(0xffffffffu, sums.apart && sums.ref == ref);  // the first of the warp's stays apart
    const bool counts = sums.apart && (sums.ref < ref || (apart & ((1u << (tid & 31)) - 1)));
    float sum = sums.total() + (counts ? 1.0f : 0.0f);
    rebase(sums.ref, ref, c, sum, ent);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, m);
        ent += __shfl_xor_sync(0xffffffffu, ent, m);
        above += __shfl_xor_sync(0xffffffffu, above, m);
    }
    if ((tid & 31) == 0) s.f[1][warp] = sum, s.f[2][warp] = ent, s.u[warp] = above | (apart ? 0x80000000u : 0);
    __syncthreads();
    if (tid == 0) {
        sum = ent = 0.0f, above = 0;
        unsigned all = 0;
        for (int i = 0; i < kWarps; ++i) sum += s.f[1][i], ent += s.f[2][i], above += s.u[i] & 0x7fffffffu, all += s.u[i] >> 31;
        s.part = RowPart{top, ref, all > 1 ? sum + (float)(all - 1) : sum, ent, above, all > 0};
    }
    if (TOP) best_of_part<T, THREADS>(part, own, p.top_n, s);
    // the cluster's
    const cg::cluster_group cluster = cg::this_cluster();
    if (ctas > 1) {
        cluster.sync();
        if (rank == 0) {  // everything at once into this CTA's memory: one trip, not one for every step of the search below
            if (tid < ctas) s.parts[tid] = *cluster.map_shared_rank(&s.part, tid);
            if (TOP)
                for (int i = tid; i < p.top_n * ctas; i += THREADS) s.found[i] = cluster.map_shared_rank(s.best, i / p.top_n)[i % p.top_n];
        }
        cluster.barrier_arrive();
    }
    __syncthreads();
    if (rank == 0) {
        RowPart all = ctas > 1 ? s.parts[0] : s.part;
        for (int i = 1; i < ctas; ++i) {
            RowPart o = s.parts[i];
            const float to = fmaxf(all.ref, o.ref);
            raise_to(all, to, c);
            raise_to(o, to, c);
            all.top = fmaxf(all.top, o.top), all.sum += o.sum + (all.apart && o.apart ? 1.0f : 0.0f), all.ent += o.ent, all.above += o.above;
            all.apart |= o.apart;
        }
        const bool bad = all.sum != all.sum || all.top == INFINITY, empty = all.top == -INFINITY;
        if (!empty) raise_to(all, all.top, c);
        const float ls = empty ? 0.0f : all.apart ? log1pf(all.sum) : logf(all.sum);
        auto logp = [&](float a) { return bad ? kNan : empty ? -INFINITY : (a - all.top) * inv_t - ls; };
        if (tid == 0) {
            if (!has && !none) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
            if (p.logprob) p.logprob[row] = none ? 0.0f : has ? logp(xt) : kNan;
            if (p.rank) p.rank[row] = bad || !has ? 0 : all.above + 1;
            if (p.entropy) p.entropy[row] = bad ? kNan : empty ? 0.0f : ls - kLn2 * (all.ent / (all.apart ? 1.0f + all.sum : all.sum));
            if (p.stats) p.stats[2 * row] = bad ? kNan : all.top, p.stats[2 * row + 1] = bad ? kNan : ls;
        }
        if (TOP) {
            const int n = p.top_n;
            auto put = [&](int r, Key k) {
                p.top_ids[row * n + r] = k && !bad ? key_id(k) : PSSA_B200_NO_TOKEN;
                p.top_logprobs[row * n + r] = bad ? kNan : k ? logp(key_value(k)) : -INFINITY;
            };
            if (ctas == 1 || bad) {  // a row with a NaN may have fewer keys than places
                if (tid < n) put(tid, s.best[tid]);
            } else {  // a key's place is the number of better ones: its own list is in order, the others are searched
                for (int i = tid; i < n * ctas; i += THREADS) {
                    const int list = i / n, at_ = i - list * n;
                    const Key k = s.found[i];
                    if (k == 0) continue;
                    int place = at_;
                    for (int l = 0; l < ctas; ++l) {
                        if (l == list) continue;
                        const Key* o = s.found + l * n;
                        int lo = 0, hi = n;  // the first that is not better
                        while (lo < hi) {
                            const int mid = (lo + hi) >> 1;
                            if (o[mid] > k)
                                lo = mid + 1;
                            else
                                hi = mid;
                        }
                        place += lo;
                    }
                    if (place < n) put(place, k);
                }
                for (int r = min(v, n) + tid; r < n; r += THREADS) put(r, 0);  // fewer ids than places
            }
        }
    }
    if (ctas > 1) cluster.barrier_wait();  // no CTA leaves while its numbers are read
}

// d = p (A + B lp) + (at the target) g, lp = log2 p: one read, one write. A CTA takes `span` vectors of one row; rows that start at different
// distances from a 16-byte boundary in the two arrays go element by element.
constexpr int kGradThreads = 256, kGradAhead = 4;

template <typename T>
__global__ void __launch_bounds__(kGradThreads) token_logprobs_grad_kernel(LogprobGradParams p, unsigned spans) {
    pdl_wait();
    constexpr int N = kVec<T>;
    const size_t row = blockIdx.x / spans;
    const int span = blockIdx.x % spans, tid = threadIdx.x, v = p.vocab;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ld_grad;
    const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int head = together ? head_of(x, v) : v, vecs = (v - head) / N, tail0 = head + vecs * N;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    uint4* ov = reinterpret_cast<uint4*>(out + head);
    const int v0 = span * kGradThreads * kGradAhead + tid;
    uint4 raw[kGradAhead];
#pragma unroll
    for (int i = 0; i < kGradAhead; ++i)
        if (v0 + i * kGradThreads < vecs) raw[i] = xv[v0 + i * kGradThreads];

    const float inv_t = 1.0f / p.temperature, c = kLog2e / p.temperature;
    const uint32_t t = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = t < (uint32_t)v;
    const float w_lp = has && p.grad_logprob ? p.grad_logprob[row] : 0.0f, w_h = p.grad_entropy ? p.grad_entropy[row] : 0.0f;
    const float m = p.stats[2 * row], l2 = p.stats[2 * row + 1] * kLog2e, h = p.grad_entropy ? p.entropy[row] : 0.0f;
    const bool zero = (w_lp == 0.0f && w_h == 0.0f) || m == -INFINITY;
    const float g = w_lp * inv_t, a = -(g + w_h * inv_t * h), b = -w_h * inv_t * kLn2;
    if (span == 0 && tid == 0 && !has && t != PSSA_B200_NO_TOKEN) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    auto one = [&](float f) {
        const float lp = fmaf(f - m, c, -l2), pr = ex2(lp);
        // the lowest power that is not 0 is -149: below it the bracket only has to be finite. A NaN stays one through ex2.
        return pr * fmaf(b, fmaxf(lp, -200.0f), a);
    };
#pragma unroll
    for (int i = 0; i < kGradAhead; ++i) {
        const int at = v0 + i * kGradThreads;
        if (at >= vecs) break;
        float f[N];
        unpack<T>(raw[i], f);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = zero ? 0.0f : one(f[e]);
        const unsigned off = t - (unsigned)(head + at * N);
        if (off < (unsigned)N && !zero) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (off == (unsigned)e) f[e] += g;
        }
        ov[at] = pack<T>(f);
    }
    auto single = [&](int i) { out[i] = from_f32<T>(zero ? 0.0f : one(to_f32(x[i])) + ((unsigned)i == t ? g : 0.0f)); };
    if (!together) {
        const int i0 = span * kGradThreads * kGradAhead * N, n = min(kGradThreads * kGradAhead * N, v - i0);
        for (int i = tid; i < n; i += kGradThreads) single(i0 + i);
    } else if (span == 0) {
        if (tid < head) single(tid);
        if (tid < v - tail0) single(tail0 + tid);
    }
}

template <typename T, int THREADS, bool TOP>
cudaError_t launch_rows(pssa_b200_ctx* ctx, const LogprobParams& p, int ctas) {
    return launch_dependent_cluster(token_logprobs_kernel<T, THREADS, TOP>, dim3((unsigned)(p.rows * ctas)), dim3(THREADS), 0, ctx->stream, ctas, p, ctas);
}

}  // namespace

int32_t launch_token_logprobs(pssa_b200_ctx* ctx, const LogprobParams& p) {
    const size_t vecs = (size_t)p.vocab * dtype_size(p.dtype) / 16;
    // CTAs of a row: until the GPU has one to an SM, or a thread would have no vector left. A cluster costs 3 us (256 rows of 16384
    // with 5 alternatives: 8.1 us, 11.0 as pairs)
    int ctas = 1;
    while (ctas < kMaxCtas && p.rows * ctas < (size_t)ctx->sm_count && vecs / (ctas * 2) >= 256) ctas *= 2;
    const bool few = p.rows * ctas <= (size_t)ctx->sm_count && vecs / ctas >= 2048;  // more threads, where few CTAs have long parts
    // small CTAs where there are enough short rows: more rows on their way, and fewer threads to join for each (8000 x 1000 bf16 with 5
    // alternatives 71 -> 37 us, 4245 x 16384 fp16 with 20 66 -> 53). Their 64 pairs read n / 64 of a long row again for n
    // alternatives, nearly all of it for the most there may be (2048 x 16384 fp32 with 5, 20 and 64: 36, 45 and 129 us, with 256
    // threads 36, 40 and 52; 4245 x 16384 fp16 with 32, 48 and 64: 62, 78 and 178, with 256 threads 70, 78 and 87)
    const bool small = ctas == 1 && vecs <= 4096 && p.rows > (size_t)ctx->sm_count * 8 && p.top_n <= 48 && vecs * p.top_n <= 65536;
    if (p.rows * ctas > 0x7fffffffull) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 log probabilities: too many rows; refusing launch");
    const cudaError_t e = with_dtype(p.dtype, [&](auto t) {
        using T = decltype(t);
        if (small) return p.top_n ? launch_rows<T, 128, true>(ctx, p, ctas) : launch_rows<T, 128, false>(ctx, p, ctas);
        if (few) return p.top_n ? launch_rows<T, 1024, true>(ctx, p, ctas) : launch_rows<T, 1024, false>(ctx, p, ctas);
        return p.top_n ? launch_rows<T, 256, true>(ctx, p, ctas) : launch_rows<T, 256, false>(ctx, p, ctas);
    });
    if (e != cudaSuccess) return cuda_fail(ctx, e, "token_logprobs_kernel");
    return after_launch(ctx, "token_logprobs_kernel");
}

int32_t launch_token_logprobs_grad(pssa_b200_ctx* ctx, const LogprobGradParams& p) {
    const size_t per = (size_t)kGradThreads * kGradAhead * 16 / dtype_size(p.dtype), spans = (p.vocab + per - 1) / per;
    if (p.rows * spans > 0x7fffffffull) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 log probabilities' gradient: too many rows; refusing launch");
    const cudaError_t e = with_dtype(p.dtype, [&](auto t) {
        return launch_dependent(token_logprobs_grad_kernel<decltype(t)>, dim3((unsigned)(p.rows * spans)), dim3(kGradThreads), 0, ctx->stream, p,
                                (unsigned)spans);
    });
    if (e != cudaSuccess) return cuda_fail(ctx, e, "token_logprobs_grad_kernel");
    return after_launch(ctx, "token_logprobs_grad_kernel");
}

}  // namespace pssa
