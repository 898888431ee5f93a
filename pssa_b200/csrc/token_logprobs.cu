// Log probabilities of given tokens with rank, entropy and top alternatives, and their gradient (see pssa_b200_token_logprobs_dev).
// One CTA per row, a pass over it for each thing that is asked.
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
    __syncthreads();  // scratch may still be read from the previous call
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int m = kWarps / 2; m > 0; m >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}

// ascending in (value, lower id first); -0 counts as +0
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
    int b = __float_as_int(x + 0.0f);
    b = b < 0 ? b ^ 0x7fffffff : b;
    return (unsigned long long)(unsigned)(b ^ 0x80000000) << 32 | (0xffffffffu - (unsigned)id);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(LogprobParams p) {
    __shared__ float s_f[kWarps];
    __shared__ unsigned s_u[kWarps];
    __shared__ unsigned long long s_k[kWarps];
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    const int v = p.vocab, tid = threadIdx.x;
    const float inv_t = 1.0f / p.temperature;
    auto sum = [](auto a, auto b) { return a + b; };
    float m = -INFINITY;
    unsigned bad = 0;
    for (int i = tid; i < v; i += kThreads) {
        const float a = to_f32(x[i]);
        bad |= !(a < INFINITY);
        m = fmaxf(m, a);
    }
    bad = block_reduce(bad, s_u, [](unsigned a, unsigned b) { return a | b; });
    m = block_reduce(m, s_f, [](float a, float b) { return fmaxf(a, b); });
    const uint32_t t = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = t < (uint32_t)v, none = t == PSSA_B200_NO_TOKEN;
    if (!has && !none && tid == 0) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    const bool empty = m == -INFINITY;
    const float xt = has ? to_f32(x[t]) : 0.0f;
    float s = 0.0f, e = 0.0f;
    unsigned above = 0;
    for (int i = tid; i < v; i += kThreads) {
        const float a = to_f32(x[i]), z = empty ? -INFINITY : (a - m) * inv_t, w = expf(z);
        s += w;
        if (w > 0.0f) e += w * z;
        above += has && a > xt;
    }
    s = block_reduce(s, s_f, sum);
    e = block_reduce(e, s_f, sum);
    above = block_reduce(above, s_u, sum);
    const float ls = empty ? 0.0f : logf(s);
    auto logp = [&](float a) { return bad ? kNan : empty ? -INFINITY : (a - m) * inv_t - ls; };
    if (tid == 0) {
        if (p.logprob) p.logprob[row] = none ? 0.0f : has ? logp(xt) : kNan;
        if (p.rank) p.rank[row] = bad || !has ? 0 : above + 1;
        if (p.entropy) p.entropy[row] = bad ? kNan : empty ? 0.0f : ls - e / s;
        if (p.stats) p.stats[2 * row] = bad ? kNan : m, p.stats[2 * row + 1] = bad ? kNan : ls;
    }
    unsigned long long last = ~0ull;
    for (int n = 0; n < p.top_n; ++n) {
        unsigned long long best = 0;
        for (int i = tid; i < v; i += kThreads) {
            const unsigned long long k = key_of(to_f32(x[i]), i);
            if (k < last && k > best) best = k;
        }
        best = block_reduce(best, s_k, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        last = best;
        if (tid == 0) {
            const unsigned id = 0xffffffffu - (unsigned)best;
            const bool there = n < v && !bad;
            p.top_ids[row * p.top_n + n] = there ? id : PSSA_B200_NO_TOKEN;
            p.top_logprobs[row * p.top_n + n] = bad ? kNan : there ? logp(to_f32(x[id])) : -INFINITY;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_grad_kernel(LogprobGradParams p) {
    const size_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    T* g = static_cast<T*>(p.grad) + row * p.ld_grad;
    const int v = p.vocab, tid = threadIdx.x;
    const float inv_t = 1.0f / p.temperature;
    const uint32_t t = p.targets ? p.targets[row] : PSSA_B200_NO_TOKEN;
    const bool has = t < (uint32_t)v;
    if (!has && t != PSSA_B200_NO_TOKEN && tid == 0) atomicExch(p.status, PSSA_B200_ERR_TOKEN);
    const float g_lp = has && p.grad_logprob ? p.grad_logprob[row] * inv_t : 0.0f;
    const float g_h = p.grad_entropy ? p.grad_entropy[row] * inv_t : 0.0f;
    const float m = p.stats[2 * row], ls = p.stats[2 * row + 1], h = p.grad_entropy ? p.entropy[row] : 0.0f;
    const bool zero = (g_lp == 0.0f && g_h == 0.0f) || m == -INFINITY;
    for (int i = tid; i < v; i += kThreads) {
        float d = 0.0f;
        if (!zero) {
            const float lp = (to_f32(x[i]) - m) * inv_t - ls, pr = expf(lp);
            d = g_lp * ((i == (int)t ? 1.0f : 0.0f) - pr);
            if (pr != 0.0f) d -= g_h * (pr * (lp + h));
        }
        g[i] = from_f32<T>(d);
    }
}

}  // namespace

int32_t launch_token_logprobs(pssa_b200_ctx* ctx, const LogprobParams& p) {
    with_dtype(p.dtype, [&](auto t) { token_logprobs_kernel<decltype(t)><<<(unsigned)p.rows, kThreads, 0, ctx->stream>>>(p); });
    return after_launch(ctx, "token_logprobs_kernel");
}

int32_t launch_token_logprobs_grad(pssa_b200_ctx* ctx, const LogprobGradParams& p) {
    with_dtype(p.dtype, [&](auto t) { token_logprobs_grad_kernel<decltype(t)><<<(unsigned)p.rows, kThreads, 0, ctx->stream>>>(p); });
    return after_launch(ctx, "token_logprobs_grad_kernel");
}

}  // namespace pssa
