// A pass over a row of logits (or a part of one): 16-byte loads, the running maximum, sum and entropy sum of a softmax in registers, and the
// cut of a row that starts anywhere into single elements and whole vectors.
#pragma once
#include <cfloat>
#include <type_traits>

#include "element.cuh"

namespace pssa {

constexpr float kNan = __builtin_nanf("");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T>
constexpr int kVec = 16 / sizeof(T);  // elements of a vector

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 numbers in one instruction
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(F2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

template <typename T>
__device__ __forceinline__ void unpack(uint4 v, float (&x)[kVec<T>]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&x)[kVec<T>]) {
    uint32_t u[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(x[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// elements in front of the first 16-byte boundary of a row (at most all of it)
template <typename T>
__device__ __forceinline__ int head_of(const T* x, int n) {
    return min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), n);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// the largest of a vector's elements; a NaN only where there is nothing else
template <typename T>
__device__ __forceinline__ float vector_max(uint4 v, const float (&x)[kVec<T>]) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {  // two at a time, as they lie
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
        const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    } else {
        return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    }
}

// Running softmax sums of the logits that a thread has met, relative to `ref`, and their maximum. `ref` starts as the largest of a
// warp's first logits and is raised only when a logit is 4 or more above it in powers of two: some lane of a warp meets a new maximum
// of its own at nearly every vector, and following each took 237 us for 4096 x 131072 bf16, now 212. Sums stay below 2^4 a logit and
// lose nothing. `ref` is never below the lowest finite number: a row of that value alone is a distribution like any other, a row of
// -inf is none. A difference is formed before it is scaled, so that logits far from zero lose nothing. A NaN or +inf makes `sum` a
// NaN, or `top` infinite.
// APART: the logit that `ref` was taken from stays out of the sums, where it would be 1 (`apart`). Of a row that is sure of one id the
// sum is then what that id leaves, and ln(1 + sum) is right to its last bits however small it is: with the 1 in it, a row whose
// entropy is 0.004 lost 4e-5 of it.
template <bool ENTROPY, bool WHERE = false, bool APART = false>
struct SoftmaxSums {
    float top = -INFINITY, ref = -FLT_MAX, lim = -FLT_MAX;
    F2 sum = {0}, ent = {0};  // sum 2^t, sum 2^t t with t = (x - ref) c; 64 bits of 0 are a pair of zeros
    int where = -1;           // WHERE: the first vector that holds `top`
    bool apart = false;

    __device__ __forceinline__ void start(float m, float c) {
        if (m > ref) ref = m, lim = m + 4.0f / c;
    }
    __device__ __forceinline__ void raise(float m, float c) {
        if (APART && apart) sum = add2(sum, pair(1.0f, 0.0f));
        const float d = fmaxf((ref - m) * c, -1e4f), f = ex2(d);
        const F2 f2 = pair(f, f);
        if (ENTROPY) ent = mul2(f2, fma2(pair(d, d), sum, ent));
        sum = mul2(f2, sum);
        start(m, c);
    }
    // N elements whose largest is m. FIRST: they are among those that the warp started from, of which none is above `ref`. With APART, x
    // comes back without the one that stays out.
    template <bool FIRST = false, int N>
    __device__ __forceinline__ void add(float (&x)[N], float m, int at, float c) {
        if (WHERE) where = m > top ? at : where;
        top = fmaxf(top, m);
        if (FIRST ? APART && m == ref && !apart : m > lim) {
            if (!FIRST) raise(m, c);
            if (APART) {
                apart = true;
                bool out = false;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (x[i] == m && !out) x[i] = -INFINITY, out = true;
            }
        }
        const F2 nref = pair(-ref, -ref), c2 = pair(c, c);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const F2 t = mul2(add2(pair(x[i], x[i + 1]), nref), c2);
            float a, b;
            split(t, a, b);
            const F2 w = pair(ex2(a), ex2(b));
            sum = add2(sum, w);
            if (ENTROPY) ent = fma2(w, pair(fmaxf(a, -200.0f), fmaxf(b, -200.0f)), ent);  // 2^-200 is 0: 0 times -inf would not be
        }
    }
    __device__ __forceinline__ void add1(float x, float c) {
        top = fmaxf(top, x);
        if (x > lim) {
            raise(x, c);
            apart = false;
        }
        if (APART && x == ref && !apart) {
            apart = true;
            return;
        }
        const float t = (x - ref) * c, w = ex2(t);
        sum = add2(sum, pair(w, 0.0f));
        if (ENTROPY) ent = fma2(pair(w, 0.0f), pair(fmaxf(t, -200.0f), 0.0f), ent);
    }
    __device__ __forceinline__ float total() const {
        float a, b;
        split(sum, a, b);
        return a + b;
    }
    __device__ __forceinline__ float entropy_total() const {
        float a, b;
        split(ent, a, b);
        return a + b;
    }
};

// sums relative to `from`, as sums relative to `to` >= from
__device__ __forceinline__ void rebase(float from, float to, float c, float& sum, float& ent) {
    const float d = fmaxf((from - to) * c, -1e4f), f = ex2(d);
    ent = f * fmaf(d, sum, ent);
    sum *= f;
}

// ascending in (value, lower id first); -0 counts as +0; 0 is no key
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
    int b = __float_as_int(x + 0.0f);
    b = b < 0 ? b ^ 0x7fffffff : b;
    return (unsigned long long)(unsigned)(b ^ 0x80000000) << 32 | (0xffffffffu - (unsigned)id);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const int b = (int)(unsigned)(k >> 32) ^ 0x80000000;
    return __int_as_float(b < 0 ? b ^ 0x7fffffff : b);
}
__device__ __forceinline__ unsigned key_id(unsigned long long k) { return 0xffffffffu - (unsigned)k; }

}  // namespace pssa
