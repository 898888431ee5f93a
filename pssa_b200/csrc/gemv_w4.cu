// Products of a few rows with a matrix in 4 bits, and quantisation to that form (see pssa_b200_gemv_w4_dev).
// One warp to a weight row, or to a group that is quantised.
#include "device_math.cuh"
#include "element.cuh"
#include "kernels.hpp"

namespace pssa {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) gemv_w4_kernel(GemvW4Params p) {
    const size_t n = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (n >= p.w.n) return;
    for (size_t r = 0; r < p.rows; ++r) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        float acc = 0.0f;
        for (size_t g = 0; g < p.w.groups; ++g) {
            const int zero = p.w.zeros ? p.w.zeros[n * p.w.groups + g] : 8;
            float part = 0.0f;
            for (size_t k = g * p.w.group + lane; k < min((g + 1) * p.w.group, p.w.k); k += 32) {
                const int c = p.w.codes[(n * p.w.k + k) >> 1] >> (k & 1) * 4 & 15;
                part = fmaf((float)(c - zero), to_f32(x[k]), part);
            }
            acc = fmaf(part, load_f32(p.w.scales, p.w.scale_dtype, n * p.w.groups + g), acc);
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
        if (lane == 0) {
            T* out = static_cast<T*>(p.out) + r * p.ldo + n;
            *out = from_f32<T>(apply_epilogue(p.epilogue, acc, p.alpha, p.epilogue == EPI_ADD_OUT ? to_f32(*out) : 0.0f));
        }
    }
}

__device__ __forceinline__ void store_scale(void* scales, int dtype, size_t i, float v) {
    if (dtype == PSSA_B200_F32)
        static_cast<float*>(scales)[i] = v;
    else if (dtype == PSSA_B200_BF16)
        static_cast<__nv_bfloat16*>(scales)[i] = from_f32<__nv_bfloat16>(v);
    else
        static_cast<__half*>(scales)[i] = from_f32<__half>(v);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) w4_quantize_kernel(W4Params p, const T* __restrict__ w) {
    const size_t at = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (at >= p.n * p.groups) return;
    const size_t n = at / p.groups, g = at % p.groups, k0 = g * p.group, k1 = min(k0 + p.group, p.k);
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
    for (size_t k = k0 + lane; k < k1; k += 32) {
        const float a = to_f32(w[n * p.k + k]);
        bad |= !isfinite(a);
        lo = fminf(lo, a), hi = fmaxf(hi, a);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    bad = __any_sync(0xffffffffu, bad);
    float step = p.zeros ? __fdiv_rn(__fsub_rn(hi, lo), 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    step = fminf(step, p.scale_dtype == PSSA_B200_F32 ? 3.402823466e38f : p.scale_dtype == PSSA_B200_BF16 ? 3.3895314e38f : 65504.0f);
    if (bad) step = __builtin_nanf("");
    if (lane == 0) store_scale(p.scales, p.scale_dtype, at, step);
    if (p.scale_dtype == PSSA_B200_BF16) step = to_f32(from_f32<__nv_bfloat16>(step));
    if (p.scale_dtype == PSSA_B200_F16) step = to_f32(from_f32<__half>(step));
    const bool live = step > 0.0f;
    const float zero = !p.zeros ? 8.0f : live ? fminf(fmaxf(rintf(__fdiv_rn(-lo, step)), 0.0f), 15.0f) : 0.0f;
    if (lane == 0 && p.zeros) p.zeros[at] = (uint8_t)zero;
    for (size_t k = k0 + 2 * lane; k < k1; k += 64) {
        unsigned byte = 0;
        for (int j = 0; j < 2; ++j) {
            const float a = to_f32(w[n * p.k + k + j]);
            const float c = live ? fminf(fmaxf(rintf(__fdiv_rn(a, step)) + zero, 0.0f), 15.0f) : zero;
            byte |= (unsigned)c << 4 * j;
        }
        p.codes[(n * p.k + k) >> 1] = (uint8_t)byte;
    }
}

}  // namespace

int32_t launch_w4_quantize(pssa_b200_ctx* ctx, const W4Params& w, const void* src, int dtype) {
    const size_t blocks = (w.n * w.groups * 32 + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 4-bit weights: too many groups; refusing launch");
    with_dtype(dtype, [&](auto t) {
        w4_quantize_kernel<<<(unsigned)blocks, kThreads, 0, ctx->stream>>>(w, static_cast<const decltype(t)*>(src));
    });
    return after_launch(ctx, "w4_quantize_kernel");
}

int32_t launch_gemv_w4(pssa_b200_ctx* ctx, const GemvW4Params& p) {
    const size_t blocks = (p.w.n * 32 + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 4-bit product: too many weight rows; refusing launch");
    with_dtype(p.dtype, [&](auto t) { gemv_w4_kernel<decltype(t)><<<(unsigned)blocks, kThreads, 0, ctx->stream>>>(p); });
    return after_launch(ctx, "gemv_w4_kernel");
}

}  // namespace pssa
