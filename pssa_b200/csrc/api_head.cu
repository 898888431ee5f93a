// extern "C" entry points of the operators on a head's weights and logits: products with 4-bit weights, log probabilities, distillation.
#include <cmath>
#include <initializer_list>

#include "bounds.hpp"
#include "element.cuh"
#include "kernels.hpp"

using namespace pssa;

namespace {

// These calls leave the caller's current device as it was.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
        error = before_ == device ? cudaSuccess : cudaSetDevice(device);
        moved_ = before_ >= 0 && before_ != device;
    }
    ~OnDevice() {
        if (moved_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    cudaError_t error;

  private:
    int before_ = -1;
    bool moved_ = false;
};

int32_t invalid(pssa_b200_ctx* ctx, const char* what, const char* why) {
    return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: %s; refusing launch", what, why);
}

bool known_dtype(int32_t dtype) { return dtype >= PSSA_B200_F32 && dtype <= PSSA_B200_F16; }
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// arrays of u32 or fp32, each of which may be absent
bool words(std::initializer_list<const void*> arrays) {
    for (const void* p : arrays)
        if (!aligned(p, 4)) return false;
    return true;
}

// [rows, cols] elements with a row pitch, in bytes
struct Pitched {
    uintptr_t start;
    size_t bytes, width, pitch;  // from the first element to behind the last; of a row; from row to row
};
int32_t pitched(pssa_b200_ctx* ctx, const char* what, const char* array, size_t rows, size_t cols, size_t ld, int32_t dtype, const void* p, Pitched* out) {
    if (ld < cols) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: pitch %zu of %s is smaller than its width %zu; refusing launch", what, ld, array, cols);
    int32_t rc;
    size_t n;
    if ((rc = f32_elems(ctx, what, {rows, ld}, &n))) return rc;
    const size_t size = dtype_size(dtype);
    if (!aligned(p, size)) return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: %s is not aligned to its element; refusing launch", what, array);
    *out = Pitched{reinterpret_cast<uintptr_t>(p), ((rows - 1) * ld + cols) * size, cols * size, ld * size};
    return PSSA_B200_OK;
}

// whether two arrays share an element: not where the rows of one lie between those of the other, at the same pitch
bool overlap(const Pitched& a, const Pitched& b) {
    if (a.start >= b.start + b.bytes || b.start >= a.start + a.bytes) return false;
    if (a.pitch != b.pitch) return true;
    const size_t off = b.start >= a.start ? (b.start - a.start) % a.pitch : a.pitch - 1 - (a.start - b.start - 1) % a.pitch;  // of b's rows in a's
    return off < a.width || off + b.width > a.pitch;
}

// rows of logits and the temperature they are read at
int32_t logits_shape(pssa_b200_ctx* ctx, const char* what, const void* logits, int32_t dtype, size_t rows, size_t vocab, size_t ld, float temperature,
                     Pitched* extent) {
    if (!logits) return invalid(ctx, what, "null logits");
    if (!known_dtype(dtype)) return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: unknown element type %d; refusing launch", what, dtype);
    if (rows == 0 || vocab == 0 || rows > 0x7fffffff || vocab > 0x7fffffff)
        return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: row count and vocabulary must be in 1..2^31-1; refusing launch", what);
    // 1 / T, and the same for powers of two, have to be numbers
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(1.4427f / temperature))
        return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: temperature %g is not a positive finite number; refusing launch", what, (double)temperature);
    return pitched(ctx, what, "the logits", rows, vocab, ld, dtype, logits, extent);
}

// a gradient may lie in the logits' own place, or clear of them
int32_t gradient_place(pssa_b200_ctx* ctx, const char* what, const Pitched& logits, void* grad, size_t ld_grad, size_t rows, size_t vocab, int32_t dtype) {
    Pitched g;
    const int32_t rc = pitched(ctx, what, "the gradient", rows, vocab, ld_grad, dtype, grad, &g);
    if (rc) return rc;
    if (g.start == logits.start ? rows > 1 && g.pitch != logits.pitch : overlap(logits, g))
        return invalid(ctx, what, "the gradient overlaps the logits without lying in their place");
    return PSSA_B200_OK;
}

int32_t w4_shape(pssa_b200_ctx* ctx, const char* what, size_t n, size_t k, size_t group, const void* codes, const void* scales, int32_t scale_dtype) {
    if (!codes || !scales) return invalid(ctx, what, "null codes or scales");
    if (!known_dtype(scale_dtype)) return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: unknown scale type %d; refusing launch", what, scale_dtype);
    if (n == 0 || k == 0 || n > 0x7fffffff || k > 0x7fffffff)
        return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: dimensions must be in 1..2^31-1; refusing launch", what);
    if (k % 32 != 0) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: width %zu is not a multiple of 32; refusing launch", what, k);
    if (!(group == 32 || group == 64 || (group != 0 && group % 128 == 0 && group < k + 128)))
        return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: group %zu is not 32, 64 or a multiple of 128 of the width; refusing launch", what, group);
    if (!aligned(codes, 16)) return invalid(ctx, what, "codes do not start on a 16-byte boundary");
    if (!aligned(scales, dtype_size(scale_dtype))) return invalid(ctx, what, "scales are not aligned to their type");
    size_t e;
    return f32_elems(ctx, what, {n, k}, &e);
}

W4Params w4_params(const void* codes, const void* scales, int32_t scale_dtype, const uint8_t* zeros, size_t n, size_t k, size_t group) {
    W4Params w{};
    w.codes = static_cast<uint8_t*>(const_cast<void*>(codes)), w.scales = const_cast<void*>(scales), w.zeros = const_cast<uint8_t*>(zeros);
    w.scale_dtype = scale_dtype, w.n = n, w.k = k, w.group = group, w.groups = (k + group - 1) / group;
    return w;
}

}  // namespace

extern "C" {

int32_t pssa_b200_w4_quantize_dev(pssa_b200_ctx* ctx, const void* w, int32_t dtype, size_t n, size_t k, size_t group, uint8_t* codes, void* scales,
                                  int32_t scale_dtype, uint8_t* zeros) {
    if (!ctx) return fail(nullptr, PSSA_B200_ERR_INVALID_ARGUMENT, "null context");
    const char* what = "4-bit weights";
    int32_t rc = w4_shape(ctx, what, n, k, group, codes, scales, scale_dtype);
    if (rc) return rc;
    if (!w) return invalid(ctx, what, "null weights");
    if (!known_dtype(dtype)) return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: unknown element type %d; refusing launch", what, dtype);
    if (!aligned(w, dtype_size(dtype))) return invalid(ctx, what, "weights are not aligned to their element");
    const OnDevice on(ctx->device);
    PSSA_CUDA(ctx, on.error);
    return launch_w4_quantize(ctx, w4_params(codes, scales, scale_dtype, zeros, n, k, group), w, dtype);
}

int32_t pssa_b200_gemv_w4_dev(pssa_b200_ctx* ctx, const void* x, int32_t dtype, size_t rows, size_t ldx, const uint8_t* codes, const void* scales,
                              int32_t scale_dtype, const uint8_t* zeros, size_t n, size_t k, size_t group, void* out, size_t ldo, int32_t epilogue,
                              float alpha) {
    if (!ctx) return fail(nullptr, PSSA_B200_ERR_INVALID_ARGUMENT, "null context");
    const char* what = "4-bit product";
    int32_t rc = w4_shape(ctx, what, n, k, group, codes, scales, scale_dtype);
    if (rc) return rc;
    if (!x || !out) return invalid(ctx, what, "null buffer");
    if (!known_dtype(dtype)) return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: unknown element type %d; refusing launch", what, dtype);
    if (rows == 0 || rows > 0x7fffffff) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: row count must be in 1..2^31-1; refusing launch", what);
    if (epilogue < PSSA_B200_EPI_NONE || epilogue > PSSA_B200_EPI_ADD_OUT)
        return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: unknown epilogue %d; refusing launch", what, epilogue);
    Pitched from, to;
    if ((rc = pitched(ctx, what, "x", rows, k, ldx, dtype, x, &from))) return rc;
    if ((rc = pitched(ctx, what, "out", rows, n, ldo, dtype, out, &to))) return rc;
    if (overlap(from, to)) return invalid(ctx, what, "x and out overlap");
    const OnDevice on(ctx->device);
    PSSA_CUDA(ctx, on.error);
    GemvW4Params p{};
    p.w = w4_params(codes, scales, scale_dtype, zeros, n, k, group);
    p.x = x, p.out = out, p.dtype = dtype, p.epilogue = epilogue, p.rows = rows, p.ldx = ldx, p.ldo = ldo, p.alpha = alpha;
    return launch_gemv_w4(ctx, p);
}

int32_t pssa_b200_token_logprobs_dev(pssa_b200_ctx* ctx, const void* logits, int32_t dtype, size_t rows, size_t vocab, size_t ld, float temperature,
                                     const uint32_t* targets, float* logprob, uint32_t* rank, float* entropy, float* stats, size_t top_n,
                                     uint32_t* top_ids, float* top_logprobs) {
    if (!ctx) return fail(nullptr, PSSA_B200_ERR_INVALID_ARGUMENT, "null context");
    const char* what = "log probabilities";
    Pitched extent;
    const int32_t rc = logits_shape(ctx, what, logits, dtype, rows, vocab, ld, temperature, &extent);
    if (rc) return rc;
    if (top_n > PSSA_B200_MAX_TOP)
        return fail(ctx, PSSA_B200_ERR_UNSUPPORTED, "B200 %s: %zu alternatives are more than %d; refusing launch", what, top_n, PSSA_B200_MAX_TOP);
    if ((top_n != 0) != (top_ids != nullptr) || (top_n != 0) != (top_logprobs != nullptr))
        return invalid(ctx, what, "alternatives need top_n, top_ids and top_logprobs, all or none");
    if ((logprob || rank) && !targets) return invalid(ctx, what, "log probability and rank need targets");
    if (!logprob && !rank && !entropy && !stats && top_n == 0) return invalid(ctx, what, "no output is asked for");
    if (!words({targets, logprob, rank, entropy, stats, top_ids, top_logprobs})) return invalid(ctx, what, "an array is not aligned to its elements");
    const OnDevice on(ctx->device);
    PSSA_CUDA(ctx, on.error);
    LogprobParams p{};
    p.logits = logits, p.dtype = dtype, p.rows = rows, p.ld = ld, p.vocab = (int)vocab, p.temperature = temperature;
    p.targets = logprob || rank ? targets : nullptr, p.logprob = logprob, p.rank = rank, p.entropy = entropy, p.stats = stats;
    p.top_n = (int)top_n, p.top_ids = top_ids, p.top_logprobs = top_logprobs, p.status = ctx->status_dev;
    return launch_token_logprobs(ctx, p);
}

int32_t pssa_b200_token_logprobs_grad_dev(pssa_b200_ctx* ctx, const void* logits, int32_t dtype, size_t rows, size_t vocab, size_t ld, float temperature,
                                          const uint32_t* targets, const float* stats, const float* entropy, const float* grad_logprob,
                                          const float* grad_entropy, void* grad_logits, size_t ld_grad) {
    if (!ctx) return fail(nullptr, PSSA_B200_ERR_INVALID_ARGUMENT, "null context");
    const char* what = "log probabilities' gradient";
    Pitched extent;
    int32_t rc = logits_shape(ctx, what, logits, dtype, rows, vocab, ld, temperature, &extent);
    if (rc) return rc;
    if (!grad_logits || !stats) return invalid(ctx, what, "null gradient or stats");
    if (grad_logprob && !targets) return invalid(ctx, what, "a weight of the log probability needs targets");
    if (grad_entropy && !entropy) return invalid(ctx, what, "a weight of the entropy needs the entropy");
    if (!words({targets, stats, entropy, grad_logprob, grad_entropy})) return invalid(ctx, what, "an array is not aligned to its elements");
    if ((rc = gradient_place(ctx, what, extent, grad_logits, ld_grad, rows, vocab, dtype))) return rc;
    const OnDevice on(ctx->device);
    PSSA_CUDA(ctx, on.error);
    LogprobGradParams p{};
    p.logits = logits, p.dtype = dtype, p.rows = rows, p.ld = ld, p.ld_grad = ld_grad, p.vocab = (int)vocab, p.temperature = temperature;
    p.targets = grad_logprob ? targets : nullptr, p.stats = stats, p.entropy = entropy, p.grad_logprob = grad_logprob;
    p.grad_entropy = grad_entropy, p.grad = grad_logits, p.status = ctx->status_dev;
    return launch_token_logprobs_grad(ctx, p);
}

int32_t pssa_b200_distill_topk_dev(pssa_b200_ctx* ctx, const void* logits, int32_t dtype, size_t rows, size_t vocab, size_t ld, float temperature,
                                   const uint32_t* teacher_ids, const float* teacher, size_t k, float teacher_temperature, const uint32_t* targets,
                                   uint32_t flags, float* kl, float* ce, const float* grad_kl, const float* grad_ce, void* grad_logits,
                                   size_t ld_grad) {
    if (!ctx) return fail(nullptr, PSSA_B200_ERR_INVALID_ARGUMENT, "null context");
    const char* what = "distillation";
    Pitched extent;
    int32_t rc = logits_shape(ctx, what, logits, dtype, rows, vocab, ld, temperature, &extent);
    if (rc) return rc;
    if (!teacher_ids || !teacher) return invalid(ctx, what, "null teacher");
    if (k == 0) return fail(ctx, PSSA_B200_ERR_SHAPE, "B200 %s: a teacher has at least one entry for a row; refusing launch", what);
    if (k > PSSA_B200_MAX_TEACHER)
        return fail(ctx, PSSA_B200_ERR_UNSUPPORTED, "B200 %s: %zu entries for a row are more than %d; refusing launch", what, k, PSSA_B200_MAX_TEACHER);
    if (flags & ~PSSA_B200_DISTILL_REST) return invalid(ctx, what, "unknown flags");
    if (!(teacher_temperature > 0.0f) || !std::isfinite(teacher_temperature) || !std::isfinite(1.0f / teacher_temperature))
        return fail(ctx, PSSA_B200_ERR_INVALID_ARGUMENT, "B200 %s: teacher temperature %g is not a positive finite number; refusing launch", what,
                    (double)teacher_temperature);
    if ((flags & PSSA_B200_DISTILL_REST) && teacher_temperature != 1.0f)
        return invalid(ctx, what, "with the mass of the other ids the teacher's entries are log probabilities, of temperature 1");
    if ((ce || grad_ce) && !targets) return invalid(ctx, what, "the cross entropy needs targets");
    if (grad_logits && !grad_kl && !grad_ce) return invalid(ctx, what, "a gradient needs the weight of a loss");
    if (!grad_logits && (grad_kl || grad_ce)) return invalid(ctx, what, "weights of losses without a gradient");
    if (!kl && !ce && !grad_logits) return invalid(ctx, what, "no output is asked for");
    if (!words({teacher_ids, teacher, targets, kl, ce, grad_kl, grad_ce})) return invalid(ctx, what, "an array is not aligned to its elements");
    if (grad_logits && (rc = gradient_place(ctx, what, extent, grad_logits, ld_grad, rows, vocab, dtype))) return rc;
    const OnDevice on(ctx->device);
    PSSA_CUDA(ctx, on.error);
    DistillParams p{};
    p.logits = logits, p.dtype = dtype, p.rows = rows, p.ld = ld, p.ld_grad = ld_grad, p.vocab = (int)vocab, p.k = (int)k;
    p.rest = (flags & PSSA_B200_DISTILL_REST) != 0, p.temperature = temperature, p.teacher_temperature = teacher_temperature;
    p.teacher_ids = teacher_ids, p.targets = ce || grad_ce ? targets : nullptr, p.teacher = teacher, p.grad_kl = grad_kl, p.grad_ce = grad_ce;
    p.kl = kl, p.ce = ce, p.grad = grad_logits, p.status = ctx->status_dev;
    return launch_distill_topk(ctx, p);
}

}  // extern "C"
