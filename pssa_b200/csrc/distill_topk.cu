// Distillation from a teacher's best ids: divergence, a target's cross entropy and the gradient in one call (see
// pssa_b200_distill_topk_dev).
//
// A row of logits is read once and its gradient written once: a cluster of CTAs holds the row in shared memory between the pass
// that sums and the pass that writes. The listed ids are masked in shared memory, so that the pass sums the ids that are not listed
// by themselves: the mass of the rest is never the difference of two numbers near 1, and a student that is sure of the listed ids
// gets its gradient relative to the rest's own maximum. The listed ids, at most 256, are added one by one, and their gradient is
// written over the zeros that the pass left there. Every CTA of a cluster does the entries' arithmetic for itself, in the same order
// and so to the same bits.
//
// Times are the kernel's in a graph of launches. 2048 x 131072 bf16 with 64 entries: 303 us, 3.5 TB/s, losses alone 202; 2048 x 16384
// fp32 with a cross entropy at another temperature: 66 us, 4.1, losses alone 45. A CTA's steps come one after another (the ids, the row,
// the cluster's meeting, the write) and three CTAs to an SM cover for each other: the barrier is the largest stall, 55 % of the
// issue slots are taken. Smaller parts (396 us at 50 KB) repeat the entries' work more often, more threads (330 at 384, 364 at 512)
// the joining.
//
// Rows above 1.5 MiB do not fit a cluster's shared memory and take the second kernel: one CTA per row, a pass of single elements
// over global memory for each thing, the listed ids marked in a bitmap. 512 x 400003 fp32: 2.1 ms, 8 times what its bytes take.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "logit_row.cuh"
#include "tcgen05.cuh"

namespace pssa {
namespace {

namespace cg = cooperative_groups;
constexpr int kThreads = 256, kWarps = kThreads / 32;

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* scratch, F op) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int m = kWarps / 2; m > 0; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// The rest's term of the divergence. Where no id has it (all are listed, or masked) the student gives it nothing and the term is
// infinite, but for what the rounding of a full list leaves: an entry's fp32 log probability q is off by 2^-24 of |q| and of the log
// sum that it was made with, so their masses by at most 2^-24 (entropy + 10), below 2^-20 for 256 entries.
constexpr float kRounding = 0x1p-20f;
__device__ __forceinline__ float rest_term(float r, bool none_left, float log_rest) {
    if (!(r > 0.0f) || (none_left && r <= kRounding)) return 0.0f;
    return none_left ? INFINITY : r * (logf(r) - log_rest);
}

// a teacher's entry at its temperature; one that is +inf is no number like a NaN
__device__ __forceinline__ float teacher_entry(const DistillParams& p, size_t row, int i) {
    const float q = p.teacher[row * p.k + i] * (1.0f / p.teacher_temperature);
    return q < INFINITY ? q : kNan;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_topk_long_kernel(DistillParams p) {
    extern __shared__ unsigned s_bits[];
    __shared__ float s_f[kWarps], s_t[PSSA_B200_MAX_TEACHER];
    __shared__ double s_d[kWarps];
    __shared__ unsigned s_u[kWarps], s_id[PSSA_B200_MAX_TEACHER];
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    const int v = p.vocab, tid = threadIdx.x;
    const float inv_t = 1.0f / p.temperature;
    auto sum = [](auto a, auto b) { return a + b; };
    auto most = [](float a, float b) { return fmaxf(a, b); };
    float m = -INFINITY;
    unsigned bad = 0;
    for (int i = tid; i < (v + 31) / 32; i += kThreads) s_bits[i] = 0;
    for (int i = tid; i < v; i += kThreads) {
        const float a = to_f32(x[i]);
        bad |= !(a < INFINITY);
        m = fmaxf(m, a);
    }
    bad = block_reduce(bad, s_u, [](unsigned a, unsigned b) { return a | b; });
    m = block_reduce(m, s_f, most);
    const bool empty = m == -INFINITY;
    // the teacher's entries, one to a thread
    const uint32_t id = tid < p.k ? p.teacher_ids[row * p.k + tid] : PSSA_B200_NO_TOKEN;
    const bool entry = id < (uint32_t)v;
    bool wrong = !entry && id != PSSA_B200_NO_TOKEN;
    const float q = entry ? teacher_entry(p, row, tid) : -INFINITY;
    float t, log_t = q, r = 0.0f;
    if (p.rest) {
        t = entry ? expf(q) : 0.0f;
        r = fmaxf((float)(1.0 - block_reduce(entry ? exp((double)q) : 0.0, s_d, sum)), 0.0f);
        if (!__syncthreads_or(entry)) r = 0.0f;  // no entry: nothing to learn
    } else {
        const float mt = block_reduce(entry && q != q ? INFINITY : q, s_f, most);  // a NaN goes through the sum
        const float e = entry && mt > -INFINITY ? expf(q - mt) : 0.0f;
        const float st = block_reduce(e, s_f, sum);
        t = st != 0.0f ? e / st : 0.0f;
        log_t = q - mt - logf(st);
    }
    const float xe = entry ? to_f32(x[id]) : -INFINITY;
    if (tid < PSSA_B200_MAX_TEACHER) s_id[tid] = entry ? id : PSSA_B200_NO_TOKEN, s_t[tid] = t;
    __syncthreads();
    bool first = entry;
    if (entry) {
        atomicOr(&s_bits[id >> 5], 1u << (id & 31));
        for (int j = 0; j < tid; ++j) first = first && s_id[j] != id;
    }
    __syncthreads();
    float mu = -FLT_MAX;  // of the ids that are not listed: their sum is relative to their own maximum
    for (int i = tid; i < v; i += kThreads)
        if (!(s_bits[i >> 5] >> (i & 31) & 1)) mu = fmaxf(mu, to_f32(x[i]));
    mu = block_reduce(mu, s_f, most);
    float su = 0.0f, s1 = 0.0f;  // the ids that are not listed at T; all ids at 1
    for (int i = tid; i < v; i += kThreads) {
        const float a = to_f32(x[i]);
        if (!(s_bits[i >> 5] >> (i & 31) & 1)) su += expf((a - mu) * inv_t);
        s1 += expf(empty ? -INFINITY : a - m);
    }
    su = block_reduce(su, s_f, sum);
    s1 = block_reduce(s1, s_f, sum);
    const float z = empty ? -INFINITY : (xe - m) * inv_t, to_m = empty ? 0.0f : fmaxf(mu - m, -FLT_MAX);
    const float s = su * expf(to_m * inv_t) + block_reduce(first ? expf(z) : 0.0f, s_f, sum);
    const float ls = logf(s), log_rest = to_m * inv_t + logf(su) - ls, p_rest = expf(log_rest);
    float term = t > 0.0f || t != t ? t * (log_t - (empty ? -INFINITY : z - ls)) : 0.0f;
    float kl = block_reduce(term, s_f, sum);
    kl += rest_term(r, empty || su == 0.0f, log_rest);
    const float mass = block_reduce(t, s_f, sum) + r;
    const uint32_t tgt = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = tgt < (uint32_t)v, none = tgt == PSSA_B200_NO_TOKEN;
    wrong = wrong || (!has && !none && tid == 0);
    if (wrong) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    if (tid == 0) {
        if (p.kl) p.kl[row] = bad ? kNan : kl;
        if (p.ce) p.ce[row] = none ? 0.0f : bad || !has ? kNan : empty ? INFINITY : logf(s1) - (to_f32(x[tgt]) - m);
    }
    if (!p.grad) return;
    T* g = static_cast<T*>(p.grad) + row * p.ld_grad;
    const float w_kl = p.grad_kl ? p.grad_kl[row] : 0.0f, w_ce = p.grad_ce && has ? p.grad_ce[row] : 0.0f;
    const bool zero = (w_kl == 0.0f && w_ce == 0.0f) || (empty && !bad);
    const float g_kl = w_kl * inv_t;
    __syncthreads();  // the logits may be where the gradient goes: everything above has been read
    for (int i = tid; i < v; i += kThreads) {
        float d = 0.0f;
        if (!zero) {
            const float a = to_f32(x[i]);
            const bool listed = s_bits[i >> 5] >> (i & 31) & 1;
            if (w_kl != 0.0f) {  // a teacher that is no number does not enter without a weight
                if (listed)
                    d = g_kl * mass * (expf((a - m) * inv_t) / s);
                else
                    d = su > 0.0f ? g_kl * (expf((a - mu) * inv_t) / su * (p.rest ? mass * p_rest - r : mass * p_rest)) : 0.0f;
                if (listed)
                    for (int j = 0; j < p.k; ++j)
                        if (s_id[j] == (unsigned)i) d -= g_kl * s_t[j];
            }
            if (w_ce != 0.0f) d += w_ce * (expf(a - m) / s1 - (i == (int)tgt ? 1.0f : 0.0f));
            if (bad) d = kNan;
        }
        g[i] = from_f32<T>(d);
    }
}

// ROW_WARPS warps read the row and one the teacher's entries; the row comes in pieces, each with a barrier of its own
constexpr int kMostWarps = 8, kPieces = 4;
struct RestSums {  // of a CTA's unlisted ids: sums at the temperature, and at 1
    float top, ref, sum, sum1;
};
constexpr float kNotFirst = -1.0f;
struct Teacher {  // what one warp makes of a row's entries while the others read the row
    alignas(16) uint32_t id[PSSA_B200_MAX_TEACHER];  // PSSA_B200_NO_TOKEN: absent, and behind the last up to a multiple of 4
    float t[PSSA_B200_MAX_TEACHER], log_t[PSSA_B200_MAX_TEACHER], x[PSSA_B200_MAX_TEACHER];
    float t_at[PSSA_B200_MAX_TEACHER];   // the id's whole mass at its first entry, kNotFirst at others of it: the mass may be a NaN
    float x_max, rest, mass;             // of the listed logits; 1 - sum t, with DISTILL_REST; sum t + rest
    int bad, target;                     // a listed logit is no number; the target's entry or -1
};

// where the warp of the teacher and those of the row meet
template <int THREADS>
__device__ __forceinline__ void ids_ready() {
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// Run by one warp, the entries in steps of 32, behind its barrier with the others, who need the ids.
template <typename T, int THREADS>
__device__ void read_teacher(const DistillParams& p, size_t row, const T* x, uint32_t tgt, Teacher& s, bool report) {
    const int lane = threadIdx.x & 31, v = p.vocab;
    float q_max = -INFINITY, x_max = -INFINITY;
    bool wrong = false, bad = false, any = false;
    for (int i = lane; i < p.k; i += 32) {
        const uint32_t id = p.teacher_ids[row * p.k + i];
        const bool entry = id < (uint32_t)v;
        wrong |= !entry && id != PSSA_B200_NO_TOKEN, any |= entry;
        s.id[i] = entry ? id : PSSA_B200_NO_TOKEN;
    }
    if (lane < 3 && p.k + lane < PSSA_B200_MAX_TEACHER) s.id[p.k + lane] = PSSA_B200_NO_TOKEN;
    ids_ready<THREADS>();
    if (report && wrong) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    for (int i = lane; i < p.k; i += 32) {
        const uint32_t id = s.id[i];
        const bool entry = id != PSSA_B200_NO_TOKEN;
        const float q = entry ? teacher_entry(p, row, i) : -INFINITY, xe = entry ? to_f32(x[id]) : -INFINITY;
        bad |= xe != xe;
        s.x[i] = xe, s.log_t[i] = q;
        q_max = fmaxf(q_max, q != q ? INFINITY : q), x_max = fmaxf(x_max, xe);
    }
    float rest = 0.0f, mass = 0.0f;
    if (p.rest) {
        double sum = 0.0;  // of fp32 numbers: their difference from 1 is what is left
        for (int i = lane; i < p.k; i += 32) sum += s.t[i] = expf(s.log_t[i]);
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (__any_sync(0xffffffffu, any)) rest = fmaxf((float)(1.0 - sum), 0.0f);  // no entry: nothing to learn
    } else {
        q_max = warp_max(q_max);  // infinite with a NaN, which then goes through the sum
        float sum = 0.0f;
        for (int i = lane; i < p.k; i += 32) {
            const float e = q_max > -INFINITY ? expf(s.log_t[i] - q_max) : 0.0f;
            s.t[i] = e, sum += e;
        }
        sum = warp_sum(sum);
        const float log_sum = logf(sum);
        for (int i = lane; i < p.k; i += 32) s.t[i] = sum != 0.0f ? s.t[i] / sum : 0.0f, s.log_t[i] = s.log_t[i] - q_max - log_sum;
    }
    for (int i = lane; i < p.k; i += 32) mass += s.t[i];
    __syncwarp();
    // is an entry the first of its id, and what is the id's whole mass?
    int target = -1;
    for (int i = lane; i < p.k; i += 32) {
        const uint32_t id = s.id[i];
        bool first = id != PSSA_B200_NO_TOKEN;
        float t_at = 0.0f;
        for (int j = 0; j < p.k; j += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(s.id + j);
            if (o.x == id) first = first && j >= i, t_at += s.t[j];
            if (o.y == id) first = first && j + 1 >= i, t_at += s.t[j + 1];
            if (o.z == id) first = first && j + 2 >= i, t_at += s.t[j + 2];
            if (o.w == id) first = first && j + 3 >= i, t_at += s.t[j + 3];
        }
        s.t_at[i] = first ? t_at : kNotFirst;
        if (first && id == tgt) target = i;
    }
    x_max = warp_max(x_max), mass = warp_sum(mass) + rest, bad = __any_sync(0xffffffffu, bad), target = __reduce_max_sync(0xffffffffu, target);
    if (lane == 0) s.x_max = x_max, s.rest = rest, s.mass = mass, s.bad = bad, s.target = target;
}

// A CTA holds elements [rank * each, + each) of a row, at the distance from a 16-byte boundary that they have in global memory.
template <typename T, int ROW_WARPS>
__global__ void __launch_bounds__(32 * (ROW_WARPS + 1)) distill_topk_kernel(DistillParams p, int ctas, int each) {
    extern __shared__ __align__(128) unsigned char s_raw[];
    __shared__ Teacher s_teacher;
    __shared__ float s_top[ROW_WARPS], s_ref[ROW_WARPS], s_sum[ROW_WARPS], s_sum1[ROW_WARPS];
    __shared__ RestSums s_part;
    __shared__ __align__(8) uint64_t s_bar[kPieces];
    pdl_wait();
    constexpr int N = kVec<T>, kRowWarps = ROW_WARPS, kPartThreads = 32 * (ROW_WARPS + 1);
    const size_t row = blockIdx.x / (unsigned)ctas;
    const int rank = blockIdx.x % (unsigned)ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, v = p.vocab;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;

    // the part, on its way to shared memory: whole 16-byte pieces by one bulk copy, what lies around them by single loads
    const int e0 = min(rank * each, v), e1 = min(e0 + each, v), n = e1 - e0;
    const T* from = x + e0;
    const int off = (int)(reinterpret_cast<uintptr_t>(from) & 15) / (int)sizeof(T), head = off ? min(N - off, n) : 0;
    const int vecs = (n - head) / N, tail0 = head + vecs * N;
    T* held = reinterpret_cast<T*>(s_raw) + off;
    uint4* held_vec = reinterpret_cast<uint4*>(held + head);
    const int piece = (vecs + kPieces - 1) / kPieces;
    if (tid == 0) {
        for (int i = 0; i < kPieces; ++i) tc::mbar_init(&s_bar[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i * piece < vecs; ++i) {
            const int bytes = (min((i + 1) * piece, vecs) - i * piece) * 16;
            tc::mbar_expect_tx(&s_bar[i], bytes);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(held_vec + i * piece)),
                         "l"(from + head + (size_t)i * piece * N), "r"(bytes), "r"(tc::smem_u32(&s_bar[i]))
                         : "memory");
        }
    }
    if (tid < head) held[tid] = from[tid];
    if (tail0 + tid < n) held[tail0 + tid] = from[tail0 + tid];
    const float inv_t = 1.0f / p.temperature, c = kLog2e / p.temperature;
    const uint32_t tgt = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = tgt < (uint32_t)v, none = tgt == PSSA_B200_NO_TOKEN;
    const float w_kl = p.grad_kl ? p.grad_kl[row] : 0.0f, w_ce = p.grad_ce && has ? p.grad_ce[row] : 0.0f;
    float xt = -INFINITY;
    if (tid == 0 && rank == 0) {
        if (has) xt = to_f32(x[tgt]);
        if (!has && !none) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    }
    const bool two = p.targets && p.temperature != 1.0f;
    if (warp == kRowWarps) {
        read_teacher<T, kPartThreads>(p, row, x, has ? tgt : PSSA_B200_NO_TOKEN - 1, s_teacher, rank == 0);
    } else {
        ids_ready<kPartThreads>();  // and the barriers
        // the sums of the ids that are not listed; at temperature 1 they serve the cross entropy too. Each warp masks the listed ids of its own share.
        SoftmaxSums<false> rest, rest1;
        auto mask = [&](auto mine) {
            for (int i = lane; i < p.k; i += 32) {
                const uint32_t id = s_teacher.id[i];
                if (id >= (uint32_t)e0 && id < (uint32_t)e1 && mine((int)id - e0)) held[(int)id - e0] = from_f32<T>(-INFINITY);
            }
            __syncwarp();
        };
        auto sweep = [&](int lo, int hi, auto both) {
#pragma unroll 2
            for (int i = lo + lane; i < hi; i += 32) {
                const uint4 raw = held_vec[i];
                float f[N];
                unpack<T>(raw, f);
                const float m = vector_max<T>(raw, f);
                rest.add(f, m, 0, c);
                if (both) rest1.add(f, m, 0, kLog2e);
            }
        };
        for (int i = 0; i * piece < vecs; ++i) {
            if (!tc::mbar_wait(&s_bar[i], 0)) {
                if (lane == 0) atomicExch(p.status, PSSA_B200_ERR_TIMEOUT);
                tc::mbar_wait(&s_bar[i], 0);  // no CTA leaves with its copy on the way, if a wait can help it
                rest.sum = pair(kNan, kNan);  // the row's results are none, as of a row with a NaN
            }
            const int last = min((i + 1) * piece, vecs), share = (last - i * piece + kRowWarps - 1) / kRowWarps;
            const int lo = min(i * piece + warp * share, last), hi = min(lo + share, last);
            mask([&](int at) { return at >= head + lo * N && at < head + hi * N; });
            if (i == 0) {
                float f[N], m = -INFINITY;
                if (lo + lane < hi) {
                    unpack<T>(held_vec[lo + lane], f);
                    m = vector_max<T>(held_vec[lo + lane], f);
                }
                m = warp_max(m);
                rest.start(m, c), rest1.start(m, kLog2e);
            }
            if (two)
                sweep(lo, hi, std::true_type());
            else
                sweep(lo, hi, std::false_type());
        }
        if (warp == 0) {
            mask([&](int at) { return at < head || at >= tail0; });
            auto single = [&](int i) {
                const float f = to_f32(held[i]);
                rest.add1(f, c);
                if (two) rest1.add1(f, kLog2e);
            };
            if (tid < head) single(tid);
            if (tail0 + tid < n) single(tail0 + tid);
        }
        const float ref = warp_max(fmaxf(rest.ref, rest1.ref)), top = warp_max(rest.top);
        float sum = rest.total(), sum1 = rest1.total(), unused = 0.0f;
        rebase(rest.ref, ref, c, sum, unused);
        rebase(rest1.ref, ref, kLog2e, sum1, unused);
        sum = warp_sum(sum);
        if (two) sum1 = warp_sum(sum1);
        if (lane == 0) s_top[warp] = top, s_ref[warp] = ref, s_sum[warp] = sum, s_sum1[warp] = two ? sum1 : sum;
    }
    __syncthreads();
    // eight parts, one to a lane of each eight; every thread gets the same sums
    auto join = [&](RestSums a) {
        float to = a.ref, unused = 0.0f;
#pragma unroll
        for (int i = 4; i > 0; i >>= 1) {
            to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, i));
            a.top = fmaxf(a.top, __shfl_xor_sync(0xffffffffu, a.top, i));
        }
        rebase(a.ref, to, c, a.sum, unused);
        if (two) rebase(a.ref, to, kLog2e, a.sum1, unused);
        a.ref = to;
#pragma unroll
        for (int i = 4; i > 0; i >>= 1) {
            a.sum += __shfl_xor_sync(0xffffffffu, a.sum, i);
            if (two) a.sum1 += __shfl_xor_sync(0xffffffffu, a.sum1, i);
        }
        return a;
    };
    static_assert(kRowWarps <= kMostWarps, "a part to a lane of eight");
    const int eighth = lane & 7;
    const RestSums no_part{-INFINITY, -FLT_MAX, 0.0f, 0.0f};
    RestSums all = join(eighth < kRowWarps ? RestSums{s_top[eighth], s_ref[eighth], s_sum[eighth], s_sum1[eighth]} : no_part);
    const cg::cluster_group cluster = cg::this_cluster();
    if (ctas > 1) {
        if (tid == 0) s_part = all;
        cluster.sync();  // and every CTA has read the listed logits: from here on their places may be written
        all = join(eighth < ctas ? *cluster.map_shared_rank(&s_part, eighth) : no_part);
        cluster.barrier_arrive();
    }
    // with the listed ids: everything relative to the row's maximum m, the rest's sum to its own
    const float m = fmaxf(all.top, s_teacher.x_max), r = s_teacher.rest, mass = s_teacher.mass;
    const bool bad = s_teacher.bad || all.sum != all.sum || m == INFINITY, empty = m == -INFINITY;
    const float to_m = empty ? 0.0f : fmaxf(all.ref - m, -FLT_MAX);
    auto z_of = [&](float a) { return empty ? -INFINITY : (a - m) * inv_t; };
    float listed = 0.0f, listed1 = 0.0f;  // each warp for itself
    for (int i = lane; i < p.k; i += 32)
        if (s_teacher.t_at[i] != kNotFirst) {
            listed += expf(z_of(s_teacher.x[i]));
            if (two) listed1 += expf(empty ? -INFINITY : s_teacher.x[i] - m);
        }
    const float s = all.sum * ex2(to_m * c) + warp_sum(listed), ls = logf(s);
    const float s1 = two ? all.sum1 * ex2(to_m * kLog2e) + warp_sum(listed1) : s;
    const float log_rest = to_m * inv_t + logf(all.sum) - ls, p_rest = expf(log_rest);
    if (rank == 0 && warp == 0) {
        float kl = 0.0f;
        for (int i = lane; i < p.k; i += 32) {
            const float t = s_teacher.t[i];
            if (t > 0.0f || t != t) kl += t * (s_teacher.log_t[i] - (empty ? -INFINITY : z_of(s_teacher.x[i]) - ls));
        }
        kl = warp_sum(kl);
        kl += rest_term(r, empty || all.sum == 0.0f, log_rest);
        if (lane == 0) {
            if (p.kl) p.kl[row] = bad ? kNan : kl;
            if (p.ce) p.ce[row] = none ? 0.0f : bad || !has ? kNan : empty ? INFINITY : logf(s1) - (xt - m);
        }
    }
    if (p.grad) {
        const bool zero = (w_kl == 0.0f && w_ce == 0.0f) || (empty && !bad);
        const float g = w_kl * inv_t;
        // an unlisted id: its share of the rest, times a, and its probability at temperature 1
        const float a = w_kl != 0.0f && all.sum > 0.0f ? g * (p.rest ? mass * p_rest - r : mass * p_rest) / all.sum : 0.0f;
        const float a1 = w_ce * ex2(to_m * kLog2e) / s1, both = two ? a : a + a1;
        const float nref = -all.ref;
        T* out = static_cast<T*>(p.grad) + row * p.ld_grad + e0;
        const bool together = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(from)) & 15) == 0;
        auto write = [&](auto grad) {  // of a pair of logits
            auto grad1 = [&](T v) {
                float y, unused;
                split(grad(pair(to_f32(v), 0.0f)), y, unused);
                return from_f32<T>(y);
            };
            if (together) {
                uint4* out_vec = reinterpret_cast<uint4*>(out + head);
#pragma unroll 2
                for (int i = tid; i < vecs; i += kPartThreads) {
                    float f[N];
                    unpack<T>(held_vec[i], f);
#pragma unroll
                    for (int e = 0; e < N; e += 2) split(grad(pair(f[e], f[e + 1])), f[e], f[e + 1]);
                    out_vec[i] = pack<T>(f);
                }
                if (tid < head) out[tid] = grad1(held[tid]);
                if (tail0 + tid < n) out[tail0 + tid] = grad1(held[tail0 + tid]);
            } else {
                for (int i = tid; i < n; i += kPartThreads) out[i] = grad1(held[i]);
            }
        };
        auto powers = [&](F2 t) {
            float x0, x1;
            split(t, x0, x1);
            return pair(ex2(x0), ex2(x1));
        };
        const F2 nref2 = pair(nref, nref), c2 = pair(c, c), log2e2 = pair(kLog2e, kLog2e), both2 = pair(both, both), a12 = pair(a1, a1);
        if (zero || bad) {
            const float y = zero ? 0.0f : kNan;
            write([&](F2) { return pair(y, y); });
        } else {
            auto one = [&](F2 f) { return mul2(both2, powers(mul2(add2(f, nref2), c2))); };
            auto with_ce = [&](F2 f) { return fma2(a12, powers(mul2(add2(f, nref2), log2e2)), one(f)); };
            const bool ce2 = two && w_ce != 0.0f;
            if (ce2)
                write(with_ce);
            else
                write(one);
            const float xt_here = has && tgt >= (uint32_t)e0 && tgt < (uint32_t)e1 ? to_f32(held[tgt - e0]) : 0.0f;
            __syncthreads();  // the listed ids and the target go over what has been written
            for (int i = tid; i < p.k; i += kPartThreads) {
                const uint32_t id = s_teacher.id[i];
                const float t_at = s_teacher.t_at[i], xe = s_teacher.x[i];
                if (id < (uint32_t)e0 || id >= (uint32_t)e1 || t_at == kNotFirst) continue;
                float d = w_kl != 0.0f ? g * (mass * (expf(z_of(xe)) / s) - t_at) : 0.0f;
                if (w_ce != 0.0f) d += w_ce * (expf(xe - m) / s1 - (id == tgt ? 1.0f : 0.0f));
                out[id - e0] = from_f32<T>(d);
            }
            if (tid == 0 && w_ce != 0.0f && s_teacher.target < 0 && tgt >= (uint32_t)e0 && tgt < (uint32_t)e1) {
                float y, unused;
                split(ce2 ? with_ce(pair(xt_here, 0.0f)) : one(pair(xt_here, 0.0f)), y, unused);
                out[tgt - e0] = from_f32<T>(y - w_ce);
            }
        }
    }
    if (ctas > 1) cluster.barrier_wait();  // no CTA leaves while its sums are read
}

template <typename T, int ROW_WARPS>
int32_t launch_parts(pssa_b200_ctx* ctx, const DistillParams& p, int ctas) {
    // parts end on multiples of 16 bytes of the row, not of memory: rows may start anywhere
    const size_t each = ((p.vocab + ctas - 1) / ctas + kVec<T> - 1) / kVec<T> * kVec<T>, smem = (each + kVec<T>) * sizeof(T);
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        PSSA_CUDA(ctx, cudaFuncSetAttribute(distill_topk_kernel<T, ROW_WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        attr.done(ctx->device);
    }
    PSSA_CUDA(ctx, launch_dependent_cluster(distill_topk_kernel<T, ROW_WARPS>, dim3((unsigned)(p.rows * ctas)), dim3(32 * (ROW_WARPS + 1)), smem, ctx->stream,
                                            ctas, p, ctas, (int)each));
    return after_launch(ctx, "distill_topk_kernel");
}

}  // namespace

int32_t launch_distill_topk(pssa_b200_ctx* ctx, const DistillParams& p) {
    const size_t bytes = (size_t)p.vocab * dtype_size(p.dtype);
    if (bytes <= 8 * 192 * 1024) {
        // parts of at most 66 KB where eight of them hold the row, three CTAs to an SM; more parts where there are few rows
        int ctas = 1;
        while (ctas < 8 && (bytes > (size_t)ctas * 66 * 1024 || (p.rows * ctas < (size_t)ctx->sm_count * 2 && bytes / (ctas * 2) >= 4096))) ctas *= 2;
        if (p.rows * ctas > 0x7fffffffull) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 distillation: too many rows; refusing launch");
        // four row warps where there are enough short rows: more of them on their way (8039 x 5003 fp32 116 -> 75 us, 2000 x 16384 bf16
        // 50 -> 43; 2000 x 32768 72 -> 77)
        const bool small = ctas == 1 && bytes <= 32 * 1024 && p.rows > (size_t)ctx->sm_count * 8;
        return with_dtype(p.dtype, [&](auto t) {
            return small ? launch_parts<decltype(t), 4>(ctx, p, ctas) : launch_parts<decltype(t), kMostWarps>(ctx, p, ctas);
        });
    }
    const size_t smem = ((size_t)p.vocab + 31) / 32 * 4;
    if (smem > 200 * 1024)
        return fail(ctx, PSSA_B200_ERR_UNSUPPORTED, "B200 distillation: vocabulary %d exceeds one CTA's marks; refusing launch", p.vocab);
    return with_dtype(p.dtype, [&](auto t) -> int32_t {
        static PerDeviceOnce attr;
        if (attr.need(ctx->device)) {
            PSSA_CUDA(ctx, cudaFuncSetAttribute(distill_topk_long_kernel<decltype(t)>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
            attr.done(ctx->device);
        }
        distill_topk_long_kernel<decltype(t)><<<(unsigned)p.rows, kThreads, smem, ctx->stream>>>(p);
        return after_launch(ctx, "distill_topk_long_kernel");
    });
}

}  // namespace pssa
