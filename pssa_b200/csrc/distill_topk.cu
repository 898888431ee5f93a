// Distillation from a teacher's best ids: divergence, a target's cross entropy and the gradient in one call (see
// pssa_b200_distill_topk_dev). One CTA per row; the listed ids are marked in a bitmap, so that the mass of the ids that are not
// listed is summed by itself and never the difference of two numbers near 1.
#include "element.cuh"
#include "kernels.hpp"

namespace pssa {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr float kNan = __builtin_nanf("");

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

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_topk_kernel(DistillParams p) {
    extern __shared__ unsigned s_bits[];
    __shared__ float s_f[kWarps], s_x[PSSA_B200_MAX_TEACHER], s_t[PSSA_B200_MAX_TEACHER];
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
    const float q = entry ? p.teacher[row * p.k + tid] * (1.0f / p.teacher_temperature) : -INFINITY;
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
    s_id[tid] = entry ? id : PSSA_B200_NO_TOKEN;
    s_t[tid] = t;
    s_x[tid] = entry ? to_f32(x[id]) : -INFINITY;
    __syncthreads();
    bool first = entry;
    float t_at = 0.0f;
    if (entry) {
        atomicOr(&s_bits[id >> 5], 1u << (id & 31));
        for (int j = 0; j < p.k; ++j)
            if (s_id[j] == id) {
                first = first && j >= tid;
                t_at += s_t[j];
            }
    }
    __syncthreads();
    float su = 0.0f, s1 = 0.0f;  // the ids that are not listed at T; all ids at 1
    for (int i = tid; i < v; i += kThreads) {
        const float a = empty ? -INFINITY : to_f32(x[i]) - m;
        if (!(s_bits[i >> 5] >> (i & 31) & 1)) su += expf(a * inv_t);
        s1 += expf(a);
    }
    su = block_reduce(su, s_f, sum);
    s1 = block_reduce(s1, s_f, sum);
    const float z = empty ? -INFINITY : (s_x[tid] - m) * inv_t;
    const float s = su + block_reduce(first ? expf(z) : 0.0f, s_f, sum);
    const float ls = logf(s), log_rest = logf(su) - ls, p_rest = su / s;
    float term = t > 0.0f || t != t ? t * (log_t - (empty ? -INFINITY : z - ls)) : 0.0f;
    float kl = block_reduce(term, s_f, sum);
    if (r > 0.0f) kl += r * (logf(r) - (empty ? -INFINITY : log_rest));
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
            const float a = to_f32(x[i]) - m;
            const bool listed = s_bits[i >> 5] >> (i & 31) & 1;
            const float e = expf(a * inv_t);
            if (p.rest)
                d = listed ? g_kl * mass * (e / s) : su > 0.0f ? g_kl * (e / su * (mass * p_rest - r)) : 0.0f;
            else
                d = g_kl * mass * (e / s);
            if (listed)
                for (int j = 0; j < p.k; ++j)
                    if (s_id[j] == (unsigned)i) d -= g_kl * s_t[j];
            if (w_ce != 0.0f) d += w_ce * (expf(a) / s1 - (i == (int)tgt ? 1.0f : 0.0f));
            if (bad) d = kNan;
        }
        g[i] = from_f32<T>(d);
    }
}

}  // namespace

int32_t launch_distill_topk(pssa_b200_ctx* ctx, const DistillParams& p) {
    const size_t smem = ((size_t)p.vocab + 31) / 32 * 4;
    if (smem > 200 * 1024)
        return fail(ctx, PSSA_B200_ERR_UNSUPPORTED, "B200 distillation: vocabulary %d exceeds one CTA's marks; refusing launch", p.vocab);
    return with_dtype(p.dtype, [&](auto t) -> int32_t {
        static PerDeviceOnce attr;
        if (smem > 32 * 1024 && attr.need(ctx->device)) {
            PSSA_CUDA(ctx, cudaFuncSetAttribute(distill_topk_kernel<decltype(t)>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
            attr.done(ctx->device);
        }
        distill_topk_kernel<decltype(t)><<<(unsigned)p.rows, kThreads, smem, ctx->stream>>>(p);
        return after_launch(ctx, "distill_topk_kernel");
    });
}

}  // namespace pssa
