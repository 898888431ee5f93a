// Products of a few rows with a matrix in 4 bits, and quantisation to that form (see pssa_b200_gemv_w4_dev).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "device_math.cuh"
#include "element.cuh"
#include "kernels.hpp"
#include "logit_row.cuh"

namespace pssa {
namespace {

constexpr int kThreads = 256;

// ---- product
//
// out[r, n] = sum over groups of scale * sum over the group's columns of (code - zero) * x. Code minus zero is a small whole
// number, exact in bf16 and fp16, so the inner sums go through mma.m16n8k16 with 16 weight rows as A, the inputs' rows as the 8
// columns of B and fp32 accumulators, and only a group's sum meets the scale. An fp32 input is three columns, its bits cut into
// three bf16 numbers that add up to it.
//
// A chunk is 128 columns. Lane (g, t) of a warp (g = lane / 4, t = lane % 4) loads 16 bytes, 32 codes, of rows g and g + 8, so that
// a row's chunk is 64 bytes in a row. Which columns the four lanes of a row multiply at a time is free as long as A and B agree,
// but all of one product have to be of one group: as they lie for groups of 128 and more, after one exchange between lanes two
// apart for 64, after a 4 x 4 transposition for 32. `run_placed` says which run of 8 columns is where. A word's 8 codes become 4
// registers of two columns 4 apart, by a mask and the bits of 128 (fp16: 1024) that put a code into a mantissa; x is staged with
// its runs in that order.
//
// What it spends: one row of 32768 x 8192 takes 40 us, 3.4 TB/s, of which 38 stay when all loads hit the same chunk. It issues in 55 %
// of its slots: the conversion of the codes is most of the instructions, but the 16 warps of an SM also wait, with one chunk each
// on its way, and 256 CTAs over 148 SMs leave 40 SMs half empty. 48 rows of 16384 x 4096 take 43 us: staging 11, joining and storing
// 11, products and conversions the rest, one after another, with no pipe above 28 %. Codes through a
// ring of bulk copies (73 us: a barrier and a trip for the scales per piece) and one tile of rows a warp with three chunks on
// their way (58 us: the work per chunk beside the conversion, twice as often) were slower.
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 128;

struct W4Split {
    int chunks;      // of 128 columns
    int ctas;        // of a cluster, which splits the columns
    int per_cta;     // chunks of a CTA
    int stage;       // chunks whose inputs are in shared memory at a time
    int k_warps;     // warps of a CTA that share weight rows and split the columns
    int slice;       // input rows of a CTA
    int row_lots_log;  // of staging, see there
    unsigned group_inverse;  // of a group's chunks: 2^32 over them, rounded up; 0 for one
    int vec;         // x starts and steps on 16 bytes
};

template <typename T>
struct Mma {  // fp32 inputs: three bf16 pieces
    static constexpr int pieces = 3;
    static constexpr uint32_t magic = 0x43004300u;
};
template <>
struct Mma<__nv_bfloat16> {
    static constexpr int pieces = 1;
    static constexpr uint32_t magic = 0x43004300u;
};
template <>
struct Mma<__half> {
    static constexpr int pieces = 1;
    static constexpr uint32_t magic = 0x64006400u;
};

template <typename T>
__device__ __forceinline__ uint32_t minus2(uint32_t a, uint32_t b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// c (+)= a b; FIRST: without what c holds
template <typename T, bool FIRST>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float c0 = FIRST ? 0.0f : c[0], c1 = FIRST ? 0.0f : c[1], c2 = FIRST ? 0.0f : c[2], c3 = FIRST ? 0.0f : c[3];
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// the run of a chunk, of 8 columns, that ends up in a word of lane t
template <int MODE>
__device__ __forceinline__ int run_placed(int word, int t) {
    if (MODE == 0) return 4 * t + word;
    if (MODE == 2) return 4 * word + t;
    return (word & 1) + 8 * (word >> 1) + 4 * (t & 1) + 2 * (t >> 1);
}

__device__ __forceinline__ void swap_words(uint32_t& lo, uint32_t& hi, bool upper, int mask) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? lo : hi, mask);
    if (upper)
        lo = got;
    else
        hi = got;
}
template <int MODE>
__device__ __forceinline__ void by_group(int t, uint4& w) {
    if (MODE == 0) return;
    if (MODE == 2) {
        swap_words(w.x, w.y, t & 1, 1);
        swap_words(w.z, w.w, t & 1, 1);
    }
    swap_words(w.x, w.z, t & 2, 2);
    swap_words(w.y, w.w, t & 2, 2);
}

__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// 8 inputs of one run as 16-bit numbers in the order of the codes' registers: columns (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ uint4 interleave(uint4 v) {
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

// 8 inputs, as they lie
template <typename T>
struct Run {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* x, bool in, int vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
        if (!in) return;
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(x)[i];
        } else if constexpr (sizeof(T) == 4) {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(x);
            v[0] = make_uint4(u[0], u[1], u[2], u[3]), v[1] = make_uint4(u[4], u[5], u[6], u[7]);
        } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
            v[0] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
        }
    }
    // into place `at` in the order of the codes' registers, and for fp32 the two after it in steps of `step`
    __device__ __forceinline__ void store(uint4* at, int step) const {
        if constexpr (sizeof(T) == 4) {
            uint32_t u[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
            for (int piece = 0; piece < 3; ++piece) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = __byte_perm(u[j], u[j + 4], 0x7632);  // the upper halves: cut, not rounded
                at[piece * step] = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(__uint_as_float(u[j]) - __uint_as_float(u[j] & 0xffff0000u));
            }
        } else {
            *at = interleave(v[0]);
        }
    }
};

__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t mask, uint32_t bits) {  // (w & mask) | bits
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
// a word's codes of rows g and g + 8, less their zeros, as the A operands of two products: columns (0, 4), (1, 5) and (2, 6), (3, 7)
template <typename T>
__device__ __forceinline__ void numbers(uint32_t low, uint32_t high, uint32_t zero_low, uint32_t zero_high, uint32_t (&a)[2][4]) {
    constexpr uint32_t kMagic = Mma<T>::magic;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        a[j >> 1][2 * (j & 1)] = minus2<T>(masked(low >> 4 * j, 0x000f000fu, kMagic), zero_low);
        a[j >> 1][2 * (j & 1) + 1] = minus2<T>(masked(high >> 4 * j, 0x000f000fu, kMagic), zero_high);
    }
}

constexpr int ctas_per_sm(int nt) { return nt <= 2 ? 2 : 1; }
constexpr int kMaxCols = 48;  // of B at a time

// MODE 0: groups of 128 and more, 1: of 64, 2: of 32.
// A CTA: kWarps / k_warps warps side by side over weight rows, each with MT times 16 of them, times k_warps over the columns'
// chunks; NT times 8 columns of B. A warp has the codes of its next chunk on their way while it multiplies one. The CTAs of a
// cluster split the columns further and each joins the sums of a part of the rows. Sums are joined in a fixed order.
template <typename T, int NT, int MT, int MODE>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) gemv_w4_kernel(GemvW4Params p, W4Split sp) {
    extern __shared__ uint4 s_x[];
    pdl_wait();
    constexpr int P = Mma<T>::pieces;
    constexpr uint32_t kMagic = Mma<T>::magic;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = warp % sp.k_warps, wm = warp / sp.k_warps, m_warps = kWarps / sp.k_warps;
    const int cta_rows = m_warps * MT * 16, rank = blockIdx.x % (unsigned)sp.ctas;
    const size_t n0 = (size_t)(blockIdx.x / (unsigned)sp.ctas) * cta_rows, r0 = (size_t)blockIdx.y * sp.slice;
    const int in_rows = (int)min((size_t)sp.slice, p.rows - r0), cols = in_rows * P;
    const int c0 = min(rank * sp.per_cta, sp.chunks), c1 = min(c0 + sp.per_cta, sp.chunks);
    const size_t row_bytes = p.w.k >> 1;
    const int k = (int)p.w.k;

    // This lane's weight rows are g + 8 m of the warp's; those behind the last row are not fetched, multiply what was there before
    // and are not stored. It fetches the scales and zeros of the t-th of them, for its quad. Inputs behind the last column are
    // staged as 0: any codes serve there.
    const size_t n_lane = n0 + (size_t)wm * MT * 16 + g;
    const int left = n_lane < p.w.n ? (int)min(p.w.n - n_lane, (size_t)MT * 16) : 0;
    const uint8_t* codes = p.w.codes + (left ? n_lane : 0) * row_bytes;
    const size_t next_row = 8 * row_bytes;
    const int last_word = (int)row_bytes - 16;
    constexpr int kGroups = MODE == 0 ? 1 : 2 * MODE;  // of a chunk
    const bool scaled = t < 2 * MT && 8 * t < left;
    const size_t scale0 = scaled ? (n_lane + 8 * t) * p.w.groups : 0;
    const int groups = scaled ? (int)p.w.groups : 0;
    const bool wide = p.w.scale_dtype == PSSA_B200_F32, halves = p.w.scale_dtype == PSSA_B200_F16;
    const int scale_shift = wide ? 0 : 16;
    struct Fetched {
        uint4 w[2 * MT];
        uint32_t scale[kGroups], zero[kGroups];  // as they lie
    };
    auto fetch = [&](int chunk, Fetched& f) {
        const uint8_t* at = codes + min(chunk * (kChunk / 2) + 16 * t, last_word);
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m, at += next_row)
            if (8 * m < left) f.w[m] = load_codes(at);
        const int group0 = MODE != 0 ? chunk * kGroups : sp.group_inverse ? (int)__umulhi((unsigned)chunk, sp.group_inverse) : chunk;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            const bool there = group0 + q < groups;
            const size_t i = scale0 + group0 + q;
            f.scale[q] = 0, f.zero[q] = 8;
            if (there && wide) f.scale[q] = static_cast<const uint32_t*>(p.w.scales)[i];
            if (there && !wide) f.scale[q] = static_cast<const uint16_t*>(p.w.scales)[i];
            if (there && p.w.zeros) f.zero[q] = p.w.zeros[i];
        }
    };
    float acc[MT][NT][4] = {};
    Fetched now{}, next{};
    if (c0 + wk < c1) fetch(c0 + wk, now);
    int col_at[NT];  // this lane's place among a word's columns of B; the last column in place of those behind it, which are not stored
#pragma unroll
    for (int j = 0; j < NT; ++j) col_at[j] = min(j * 8 + g, cols - 1) * 4 + t;

    const T* x = static_cast<const T*>(p.x) + r0 * p.ldx;
    // 16 threads to a chunk's runs of one row; the others take other rows, or chunks where there are few rows. Lanes next to each
    // other store to different banks.
    const int run_at = threadIdx.x & 3, run_word = threadIdx.x >> 3 & 3, lot = (threadIdx.x >> 5) * 2 + (threadIdx.x >> 2 & 1);
    const int run = run_placed<MODE>(run_word, run_at), row_lots = 1 << sp.row_lots_log, chunk_lots = kThreads / 16 >> sp.row_lots_log;
    auto stage = [&](int first) {
        const int last = min(first + sp.stage, c1);
        for (int r = lot & (row_lots - 1); r < in_rows; r += row_lots) {
            const T* from = x + (size_t)r * p.ldx + 8 * run;
            uint4* at = s_x + (run_word * cols + r * P) * 4 + run_at;
#pragma unroll 4
            for (int c = first + (lot >> sp.row_lots_log); c < last; c += chunk_lots) {
                Run<T> v;
                v.load(from + c * kChunk, c * kChunk + 8 * run < k, sp.vec);
                v.store(at + (c - first) * 16 * cols, 4);
            }
        }
    };
    // with many columns of B a chunk at a time: its inputs are on their way while the one before is multiplied
    constexpr int kRuns = (kMaxCols / P * 16 + kThreads - 1) / kThreads;
    Run<T> coming[kRuns];
    auto load_chunk = [&](int c) {
#pragma unroll
        for (int u = 0; u < kRuns; ++u)
            if (lot + 16 * u < in_rows) coming[u].load(x + (size_t)(lot + 16 * u) * p.ldx + c * kChunk + 8 * run, c * kChunk + 8 * run < k, sp.vec);
    };
    auto store_chunk = [&](uint4* to) {
#pragma unroll
        for (int u = 0; u < kRuns; ++u)
            if (lot + 16 * u < in_rows) coming[u].store(to + (run_word * cols + (lot + 16 * u) * P) * 4 + run_at, 4);
    };
    auto work = [&](Fetched& f, const uint4* xs) {
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) by_group<MODE>(t, f.w[m]);
        float part[MT][NT][4], own[kGroups];
        uint32_t zero[2 * MT];
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            // fp32 and bf16 scales by a shift, fp16 ones converted: a choice of two numbers, not of two ways
            const float shifted = __uint_as_float(f.scale[q] << scale_shift), half = __half2float(__ushort_as_half((unsigned short)f.scale[q]));
            own[q] = halves ? half : shifted;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            constexpr int kWords = 4 / kGroups;  // of a group
            const int q = i / kWords;
            if (i % kWords == 0) {
#pragma unroll
                for (int m = 0; m < 2 * MT; ++m) zero[m] = kMagic | __shfl_sync(0xffffffffu, f.zero[q], (lane & 28) + m) * 0x00010001u;
            }
            uint4 v[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) v[j] = xs[i * cols * 4 + col_at[j]];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                auto word = [&](const uint4& w) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; };
                uint32_t a[2][4];
                numbers<T>(word(f.w[2 * m]), word(f.w[2 * m + 1]), zero[2 * m], zero[2 * m + 1], a);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (i % kWords == 0)
                        mma16816<T, true>(part[m][j], a[0], v[j].x, v[j].y);
                    else
                        mma16816<T, false>(part[m][j], a[0], v[j].x, v[j].y);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) mma16816<T, false>(part[m][j], a[1], v[j].z, v[j].w);
                if ((i + 1) % kWords == 0) {  // a group's sums, or a chunk's of a longer group, meet their scale
                    const float low = __shfl_sync(0xffffffffu, own[q], (lane & 28) + 2 * m), high = __shfl_sync(0xffffffffu, own[q], (lane & 28) + 2 * m + 1);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[m][j][e] = fmaf(part[m][j][e], e < 2 ? low : high, acc[m][j][e]);
                }
            }
        }
    };
    if constexpr (NT >= 3) {
        if (c0 < c1) {
            load_chunk(c0);
            store_chunk(s_x);
            if (c0 + 1 < c1) load_chunk(c0 + 1);
        }
        __syncthreads();
#pragma unroll 2
        for (int c = c0; c < c1; ++c) {
            if (c + 1 < c1) fetch(c + 1, next);
            work(now, s_x + (c - c0 & 1) * 16 * cols);
            if (c + 1 < c1) store_chunk(s_x + (c + 1 - c0 & 1) * 16 * cols);
            if (c + 2 < c1) load_chunk(c + 2);
            now = next;
            __syncthreads();
        }
    } else {
        for (int first = c0; first < c1; first += sp.stage) {
            if (first != c0) __syncthreads();
            stage(first);
            __syncthreads();
            const int last = min(first + sp.stage, c1);
#pragma unroll 2
            for (int chunk = first + wk; chunk < last; chunk += sp.k_warps) {
                if (chunk + sp.k_warps < c1) fetch(chunk + sp.k_warps, next);
                work(now, s_x + (chunk - first) * 16 * cols);
                now = next;
            }
        }
    }
    // the warps' sums side by side in shared memory, [k_warps][cta_rows][pitch]
    __syncthreads();
    float* red = reinterpret_cast<float*>(s_x);
    const int pitch = cols | 1, tile = cta_rows * pitch;  // odd: neighbouring rows in different banks
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = (wm * MT + m) * 16 + (e >> 1) * 8 + g, col = j * 8 + 2 * t + (e & 1);
                if (col < cols) red[wk * tile + row * pitch + col] = acc[m][j][e];
            }
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    if (sp.ctas > 1)
        cluster.sync();
    else
        __syncthreads();
    // each CTA of a cluster joins and stores a part of the rows: neighbouring threads neighbouring rows of weights
    const int each = cta_rows / sp.ctas, row = rank * each + threadIdx.x % each;
    const size_t n = n0 + row;
    if (n < p.w.n) {
        T* out = static_cast<T*>(p.out) + r0 * p.ldo + n;
#pragma unroll 2
        for (int r = threadIdx.x / each; r < in_rows; r += kThreads / each) {
            float v = 0.0f;
#pragma unroll
            for (int piece = 0; piece < P; ++piece) {
                const int at = row * pitch + r * P + piece;
                float sum = 0.0f;
                for (int c = 0; c < sp.ctas; ++c) {
                    const float* from = sp.ctas > 1 ? cluster.map_shared_rank(red, c) : red;
                    if constexpr (NT >= 3) {
                        sum += from[at];
                    } else {
                        float u[kWarps];
#pragma unroll
                        for (int w = 0; w < kWarps; ++w) u[w] = w < sp.k_warps ? from[w * tile + at] : 0.0f;
                        sum += ((u[0] + u[1]) + (u[2] + u[3])) + ((u[4] + u[5]) + (u[6] + u[7]));
                    }
                }
                v += sum;
            }
            T* o = out + (size_t)r * p.ldo;
            *o = from_f32<T>(apply_epilogue(p.epilogue, v, p.alpha, p.epilogue == EPI_ADD_OUT ? to_f32(*o) : 0.0f));
        }
    }
    if (sp.ctas > 1) cluster.sync();  // no CTA leaves while its sums are read
}

__device__ __forceinline__ void store_scale(void* scales, int dtype, size_t i, float v) {
    if (dtype == PSSA_B200_F32)
        static_cast<float*>(scales)[i] = v;
    else if (dtype == PSSA_B200_BF16)
        static_cast<__nv_bfloat16*>(scales)[i] = from_f32<__nv_bfloat16>(v);
    else
        static_cast<__half*>(scales)[i] = from_f32<__half>(v);
}

// Scale and zero of one group from its lanes' smallest and largest weight; the order of every fp32 operation is the definition's.
struct GroupForm {
    float step, inv;
    int zero;
    bool live, exact;  // exact: 1 / step is no normal number, or quotients are too large for the short way (a scale cut to its type)
};
template <int LANES>
__device__ __forceinline__ GroupForm group_form(const W4Params& p, size_t at, float lo, float hi, bool bad, bool store) {
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, m) != 0;
    }
    float step = p.zeros ? __fdiv_rn(__fsub_rn(hi, lo), 15.0f) : __fdiv_rn(fmaxf(hi, -lo), 7.0f);
    step = fminf(step, p.scale_dtype == PSSA_B200_F32 ? 3.402823466e38f : p.scale_dtype == PSSA_B200_BF16 ? 3.3895314e38f : 65504.0f);
    if (bad) step = __builtin_nanf("");
    if (store) store_scale(p.scales, p.scale_dtype, at, step);
    if (p.scale_dtype == PSSA_B200_BF16) step = to_f32(from_f32<__nv_bfloat16>(step));
    if (p.scale_dtype == PSSA_B200_F16) step = to_f32(from_f32<__half>(step));
    GroupForm f;
    f.step = step, f.live = step > 0.0f;
    f.zero = !p.zeros ? 8 : f.live ? (int)fminf(fmaxf(rintf(__fdiv_rn(-lo, step)), 0.0f), 15.0f) : 0;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f.inv) : "f"(step));
    f.exact = !(f.inv >= FLT_MIN && f.inv <= FLT_MAX && fmaxf(hi, -lo) * f.inv < 64.0f);
    if (store && p.zeros) p.zeros[at] = (uint8_t)f.zero;
    return f;
}
// clamp(rint(a / step) + zero, 0, 15)
__device__ __noinline__ unsigned exact_code(float a, float step, int zero) {
    return (unsigned)fminf(fmaxf(rintf(__fdiv_rn(a, step)) + (float)zero, 0.0f), 15.0f);
}
// The same for 8 weights, as one word. The product with 1 / step is within 3e-6 of the quotient where that is below 16, so that
// both round to the same whole number unless it lies within 1e-5 of the middle of two; there, and where 1 / step is no normal
// number, the division decides, out of line. Adding 1.5 * 2^23 rounds to a whole number and leaves it in the low bits: a
// conversion for each weight would be bound by the units that convert (167 us for 16384 x 8192 bf16, now 129).
__device__ __forceinline__ unsigned codes_of(const GroupForm& f, const float* x) {
    if (!f.live) return 0x11111111u * (unsigned)f.zero;
    constexpr float kRound = 12582912.0f;
    float middle = f.exact ? 1.0f : 0.0f;
    unsigned word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = x[j] * f.inv, r = v + kRound;
        middle = fmaxf(middle, fabsf(v - (r - kRound)));
        const int q = __float_as_int(r) - (__float_as_int(kRound) - f.zero);
        word |= (unsigned)min(max(q, 0), 15) << 4 * j;
    }
    if (!(middle < 0.49999f)) {
        word = 0;
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            float a = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) a = i == j ? x[i] : a;
            word |= exact_code(a, f.step, f.zero) << 4 * j;
        }
    }
    return word;
}

// Groups of LANES * 32 columns, 32 / LANES of them to a warp: one read of the weights, in units of 8 columns that neighbouring
// lanes hold in turn. What a group costs besides its weights, two divisions first of all, is shared by 32 of them (16384 x 8192
// bf16 with zeros: 129 us, 2.6 TB/s; 141 with 16 to a lane). Bound by the instructions of the codes. w starts on 16 bytes.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) w4_quantize_groups_kernel(W4Params p, const T* __restrict__ w) {
    pdl_wait();
    constexpr int kUnits = 4, kWords = sizeof(T) / 2;  // units of a lane; 16-byte words of a unit
    const size_t total = p.n * p.groups, at = ((size_t)blockIdx.x * kThreads + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES;
    const size_t n = total >> 32 ? at / p.groups : (unsigned)at / (unsigned)p.groups, k0 = (at - n * p.groups) * p.group, row = n * p.k;
    const int left = at < total ? (int)min(p.group, p.k - k0) : 0;  // columns of the group
    uint4 raw[kUnits][kWords];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int k = (u * LANES + lane) * 8;
#pragma unroll
        for (int j = 0; j < kWords; ++j) raw[u][j] = k < left ? reinterpret_cast<const uint4*>(w + row + k0 + k)[j] : make_uint4(0, 0, 0, 0);
    }
    auto unit = [&](int u, float (&x)[8]) {
        if constexpr (sizeof(T) == 4) {
            unpack<T>(raw[u][0], *reinterpret_cast<float(*)[4]>(x));
            unpack<T>(raw[u][1], *reinterpret_cast<float(*)[4]>(x + 4));
        } else {
            unpack<T>(raw[u][0], x);
        }
    };
    float lo = 0.0f, hi = 0.0f;
    bool bad = false;
    if constexpr (sizeof(T) == 4) {
        float none = 0.0f;  // a NaN once a weight is none or infinite
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            float x[8];
            unit(u, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]), none = fmaf(x[j], 0.0f, none);
        }
        bad = none != none;
    } else {  // two at a time, as they lie; a NaN stays one
        using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
        const T2* h = reinterpret_cast<const T2*>(raw);
        T2 a = h[0], b = h[0];
#pragma unroll
        for (int j = 1; j < kUnits * 4; ++j) a = __hmin2_nan(a, h[j]), b = __hmax2_nan(b, h[j]);
        lo = fminf(to_f32(a.x), to_f32(a.y)), hi = fmaxf(to_f32(b.x), to_f32(b.y));
        const float none = fmaf(to_f32(a.x), 0.0f, fmaf(to_f32(a.y), 0.0f, fmaf(to_f32(b.x), 0.0f, to_f32(b.y) * 0.0f)));
        bad = none != none, lo = fminf(lo, 0.0f), hi = fmaxf(hi, 0.0f);
    }
    const GroupForm f = group_form<LANES>(p, at, lo, hi, bad, lane == 0 && left > 0);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int k = (u * LANES + lane) * 8;
        float x[8];
        unit(u, x);
        if (k < left) *reinterpret_cast<unsigned*>(p.codes + (row + k0 + k >> 1)) = codes_of(f, x);
    }
}

// Groups of any length, one to a warp, read twice; and weights that start anywhere.
template <typename T>
__global__ void __launch_bounds__(kThreads) w4_quantize_kernel(W4Params p, const T* __restrict__ w) {
    pdl_wait();
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
    const GroupForm f = group_form<32>(p, at, lo, hi, bad, lane == 0);
    for (size_t k = k0 + 2 * lane; k < k1; k += 64) {
        const unsigned even = f.live ? exact_code(to_f32(w[n * p.k + k]), f.step, f.zero) : (unsigned)f.zero;
        const unsigned odd = f.live ? exact_code(to_f32(w[n * p.k + k + 1]), f.step, f.zero) : (unsigned)f.zero;
        p.codes[(n * p.k + k) >> 1] = (uint8_t)(even | odd << 4);
    }
}

}  // namespace

int32_t launch_w4_quantize(pssa_b200_ctx* ctx, const W4Params& w, const void* src, int dtype) {
    // lanes of a group share a warp evenly
    const bool together = w.group <= 512 && (w.group & (w.group - 1)) == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const size_t lanes = together ? w.group / 32 : 32, per = kThreads / lanes, blocks = (w.n * w.groups + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 4-bit weights: too many groups; refusing launch");
    const cudaError_t e = with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const T* x = static_cast<const T*>(src);
        auto launch = [&](void (*kernel)(W4Params, const T*)) { return launch_dependent(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, ctx->stream, w, x); };
        if (!together) return launch(w4_quantize_kernel<T>);
        switch (lanes) {
            case 1: return launch(w4_quantize_groups_kernel<T, 1>);
            case 2: return launch(w4_quantize_groups_kernel<T, 2>);
            case 4: return launch(w4_quantize_groups_kernel<T, 4>);
            case 8: return launch(w4_quantize_groups_kernel<T, 8>);
            default: return launch(w4_quantize_groups_kernel<T, 16>);
        }
    });
    if (e != cudaSuccess) return cuda_fail(ctx, e, "w4_quantize_kernel");
    return after_launch(ctx, together ? "w4_quantize_groups_kernel" : "w4_quantize_kernel");
}

namespace {
template <typename T, int NT, int MT, int MODE>
int32_t launch_tiles(pssa_b200_ctx* ctx, const GemvW4Params& p, int slice) {
    constexpr int P = Mma<T>::pieces;
    W4Split sp{};
    sp.chunks = (int)((p.w.k + kChunk - 1) / kChunk);
    // chunk * inverse >> 32 is chunk / group chunks while chunk * (group chunks) < 2^32
    const size_t group_chunks = p.w.group / kChunk;
    sp.group_inverse = group_chunks > 1 ? (unsigned)(((1ull << 32) + group_chunks - 1) / group_chunks) : 0;
    if (sp.chunks > 65535) return fail(ctx, PSSA_B200_ERR_UNSUPPORTED, "B200 4-bit product: width %zu above 8388480; refusing launch", p.w.k);
    sp.vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.ldx * sizeof(T) % 16 == 0;
    sp.slice = slice;
    while (1 << sp.row_lots_log < slice && sp.row_lots_log < 4) ++sp.row_lots_log;
    // Warps take columns rather than rows while the GPU has room for the CTAs, two to an SM (head of 16384 x 768, 1 row: 6.8, 6.2,
    // 5.7 and 7.5 us with 1, 2, 4 and 8 of them to a row). With many columns of B they share the staged inputs instead (48 rows of
    // 16384 x 4096: 47, 57, 81 and 124 us).
    sp.k_warps = 1;
    while (NT <= 2 && sp.k_warps < kWarps && sp.k_warps < sp.chunks && (p.w.n * sp.k_warps * 2 + kWarps * MT * 16 - 1) / (kWarps * MT * 16) <= (size_t)ctx->sm_count * 2)
        sp.k_warps *= 2;
    const int cta_rows = kWarps / sp.k_warps * MT * 16;
    const size_t tiles = (p.w.n + cta_rows - 1) / cta_rows, slices = (p.rows + slice - 1) / slice;
    if (tiles > 0x7fffffff / 8 || slices > 65535) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 4-bit product: too many rows; refusing launch");
    int ctas = 1;
    while (ctas < 8 && tiles * slices * ctas * 2 <= (size_t)ctx->sm_count * ctas_per_sm(NT) && ctas * 2 * sp.k_warps <= sp.chunks) ctas *= 2;
    sp.ctas = ctas, sp.per_cta = (sp.chunks + ctas - 1) / ctas;
    const size_t chunk_bytes = (size_t)256 * slice * P, room = 96 * 1024;  // two CTAs to an SM
    sp.stage = NT >= 3 ? 2 : (int)std::min<size_t>(sp.per_cta, std::max<size_t>(sp.k_warps, room / chunk_bytes / sp.k_warps * sp.k_warps));
    const size_t smem = std::max(chunk_bytes * sp.stage, (size_t)kWarps * MT * 16 * (slice * P | 1) * 4);
    static PerDeviceOnce attr;
    if (attr.need(ctx->device)) {
        PSSA_CUDA(ctx, cudaFuncSetAttribute(gemv_w4_kernel<T, NT, MT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        attr.done(ctx->device);
    }
    PSSA_CUDA(ctx, launch_dependent_cluster(gemv_w4_kernel<T, NT, MT, MODE>, dim3((unsigned)(tiles * ctas), (unsigned)slices), dim3(kThreads), smem, ctx->stream,
                                            ctas, p, sp));
    return after_launch(ctx, "gemv_w4_kernel");
}
}  // namespace

int32_t launch_gemv_w4(pssa_b200_ctx* ctx, const GemvW4Params& p) {
    return with_dtype(p.dtype, [&](auto t) -> int32_t {
        using T = decltype(t);
        constexpr size_t P = Mma<T>::pieces;
        // up to 48 columns of B at a time, the rows spread evenly over as many times as that takes
        const size_t most = std::min(p.rows, kMaxCols / P), slices = (p.rows + most - 1) / most, slice = (p.rows + slices - 1) / slices, cols = slice * P;
        auto by_group = [&](auto mode) {
            constexpr int M = decltype(mode)::value;
            if (cols <= 8) return launch_tiles<T, 1, 2, M>(ctx, p, (int)slice);
            if (cols <= 16) return launch_tiles<T, 2, 2, M>(ctx, p, (int)slice);
            if (cols <= 24) return launch_tiles<T, 3, 2, M>(ctx, p, (int)slice);
            if (cols <= 32) return launch_tiles<T, 4, 2, M>(ctx, p, (int)slice);
            return launch_tiles<T, 6, 2, M>(ctx, p, (int)slice);
        };
        if (p.w.group == 32) return by_group(std::integral_constant<int, 2>());
        if (p.w.group == 64) return by_group(std::integral_constant<int, 1>());
        return by_group(std::integral_constant<int, 0>());
    });
}

}  // namespace pssa
