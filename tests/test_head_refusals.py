"""What the operators on a head's weights and logits refuse, on the CPU: every check runs before the device is touched, so a call
that is let through ends with status 3 here (no device) and launches nothing."""
import os
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
CUDA = pathlib.Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
pytestmark = pytest.mark.skipif(not (CUDA / "include" / "cuda_runtime.h").exists(), reason="no CUDA headers")

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstdint>
#include <string>
#include "context.hpp"
int bad = 0;
pssa_b200_ctx ctx;
void expect(int32_t got, int32_t want, int line) {
    // a refused call says so; one that is let through fails for want of a device
    const bool said = want == 3 || want == -1 || ctx.error.find("refusing launch") != std::string::npos;
    if ((want >= 0 && got != want) || !said) ++bad, std::printf("line %d: status %d, expected %d: %s\n", line, got, want, ctx.error.c_str());
    ctx.error.clear();
}
#define EXPECT(want, call) expect(call, want, __LINE__)
template <typename T = float> T* at(uintptr_t p) { return reinterpret_cast<T*>(p); }
enum { OK = 3, ARG = 1, SHAPE = 2, UNSUPPORTED = 6 };
struct L {  // a call of token_logprobs that is in order
    uintptr_t x = 0x100000000; int dtype = 0; size_t rows = 4, vocab = 1000, ld = 1000; float t = 1; uintptr_t tgt = 0x1000, lp = 0x2000, rank = 0x3000;
    uintptr_t h = 0x4000, st = 0x5000; size_t n = 5; uintptr_t ids = 0x6000, top = 0x7000;
    int32_t go() { return pssa_b200_token_logprobs_dev(&ctx, at(x), dtype, rows, vocab, ld, t, at<uint32_t>(tgt), at(lp), at<uint32_t>(rank), at(h), at(st), n,
                                                       at<uint32_t>(ids), at(top)); }
};
struct G {
    uintptr_t x = 0x100000000; int dtype = 0; size_t rows = 4, vocab = 1000, ld = 1000; float t = 1; uintptr_t tgt = 0x1000, st = 0x5000, h = 0x4000;
    uintptr_t glp = 0x8000, gh = 0x9000, g = 0x200000000; size_t ldg = 1000;
    int32_t go() { return pssa_b200_token_logprobs_grad_dev(&ctx, at(x), dtype, rows, vocab, ld, t, at<uint32_t>(tgt), at(st), at(h), at(glp), at(gh), at(g), ldg); }
};
struct D {
    uintptr_t x = 0x100000000; int dtype = 0; size_t rows = 4, vocab = 1000, ld = 1000; float t = 1; uintptr_t ids = 0x1000, te = 0x2000; size_t k = 8; float tt = 1;
    uintptr_t tgt = 0x3000; uint32_t flags = 0; uintptr_t kl = 0x4000, ce = 0x5000, gk = 0x6000, gc = 0x7000, g = 0x200000000; size_t ldg = 1000;
    int32_t go() { return pssa_b200_distill_topk_dev(&ctx, at(x), dtype, rows, vocab, ld, t, at<uint32_t>(ids), at(te), k, tt, at<uint32_t>(tgt), flags, at(kl), at(ce),
                                                     at(gk), at(gc), at(g), ldg); }
};
struct W {
    uintptr_t w = 0x100000000; int dtype = 0; size_t n = 64, k = 256, group = 64; uintptr_t codes = 0x200000000, sc = 0x3000; int sd = 0; uintptr_t z = 0x5000;
    int32_t go() { return pssa_b200_w4_quantize_dev(&ctx, at(w), dtype, n, k, group, at<uint8_t>(codes), at(sc), sd, at<uint8_t>(z)); }
};
struct V {
    uintptr_t x = 0x100000000; int dtype = 0; size_t rows = 2, ldx = 256; uintptr_t codes = 0x200000000, sc = 0x3000; int sd = 0; uintptr_t z = 0x5000;
    size_t n = 64, k = 256, group = 64; uintptr_t out = 0x300000000; size_t ldo = 64; int epi = 0;
    int32_t go() { return pssa_b200_gemv_w4_dev(&ctx, at(x), dtype, rows, ldx, at<uint8_t>(codes), at(sc), sd, at<uint8_t>(z), n, k, group, at(out), ldo, epi, 1.0f); }
};
template <typename C, typename F> int32_t with(F f) { C c; f(c); return c.go(); }
#define CALL(C, want, change) EXPECT(want, with<C>([](C& c) { change; }))
int main() {
    const float inf = INFINITY, nan = NAN;
    (void)inf, (void)nan;
    // logits, in all three calls
#define LOGITS(C) \
    CALL(C, OK, ;); CALL(C, ARG, c.x = 0); CALL(C, ARG, c.dtype = 3); CALL(C, ARG, c.dtype = -1); CALL(C, SHAPE, c.rows = 0); CALL(C, SHAPE, c.vocab = 0); \
    CALL(C, SHAPE, c.ld = 999); CALL(C, SHAPE, c.rows = (size_t)1 << 31); CALL(C, SHAPE, (c.vocab = (size_t)1 << 31, c.ld = c.vocab)); \
    CALL(C, SHAPE, c.ld = (size_t)1 << 61); CALL(C, ARG, c.t = 0); CALL(C, ARG, c.t = -1); CALL(C, ARG, c.t = NAN); CALL(C, ARG, c.t = INFINITY); \
    CALL(C, ARG, c.t = 1e-39f); CALL(C, OK, c.t = 1e-30f); CALL(C, ARG, c.x += 2); CALL(C, ARG, (c.dtype = 1, c.x += 1)); CALL(C, OK, (c.dtype = 2, c.x += 2)); \
    CALL(C, OK, (c.vocab = 1, c.ld = 1, c.rows = 1));
    LOGITS(L) LOGITS(G) LOGITS(D)
    CALL(L, UNSUPPORTED, c.n = 65); CALL(L, OK, c.n = 64); CALL(L, ARG, c.n = 0); CALL(L, ARG, c.ids = 0); CALL(L, ARG, c.top = 0);
    CALL(L, OK, (c.n = 0, c.ids = 0, c.top = 0)); CALL(L, ARG, c.tgt = 0); CALL(L, OK, (c.tgt = 0, c.lp = 0, c.rank = 0));
    CALL(L, ARG, (c.n = 0, c.ids = 0, c.top = 0, c.lp = 0, c.rank = 0, c.h = 0, c.st = 0)); CALL(L, OK, (c.n = 0, c.ids = 0, c.top = 0, c.lp = 0, c.h = 0, c.st = 0));
    CALL(G, ARG, c.g = 0); CALL(G, ARG, c.st = 0); CALL(G, ARG, c.tgt = 0); CALL(G, ARG, c.h = 0); CALL(G, OK, (c.h = 0, c.gh = 0)); CALL(G, OK, (c.tgt = 0, c.glp = 0));
    CALL(G, OK, c.g = c.x); CALL(G, ARG, c.g = c.x + 4); CALL(G, ARG, (c.g = c.x, c.ldg = 1001)); CALL(G, OK, (c.g = c.x, c.ldg = 1001, c.rows = 1));
    CALL(G, ARG, c.g = c.x + 15996); CALL(G, OK, c.g = c.x + 16000); CALL(G, ARG, c.g = c.x - 4); CALL(G, SHAPE, c.ldg = 999); CALL(G, ARG, c.g += 1);
    CALL(D, ARG, c.ids = 0); CALL(D, ARG, c.te = 0); CALL(D, SHAPE, c.k = 0); CALL(D, UNSUPPORTED, c.k = 257); CALL(D, OK, c.k = 256); CALL(D, ARG, c.flags = 2);
    CALL(D, OK, c.flags = 1); CALL(D, ARG, (c.flags = 1, c.tt = 2)); CALL(D, ARG, c.tt = 0); CALL(D, ARG, c.tt = NAN); CALL(D, ARG, c.tgt = 0);
    CALL(D, OK, (c.tgt = 0, c.ce = 0, c.gc = 0)); CALL(D, ARG, (c.gk = 0, c.gc = 0)); CALL(D, ARG, c.g = 0); CALL(D, OK, (c.g = 0, c.gk = 0, c.gc = 0));
    CALL(D, ARG, (c.g = 0, c.gk = 0, c.gc = 0, c.kl = 0, c.ce = 0)); CALL(D, OK, c.g = c.x); CALL(D, ARG, c.g = c.x + 8); CALL(D, SHAPE, c.ldg = 12);
#define WEIGHTS(C) \
    CALL(C, OK, ;); CALL(C, ARG, c.codes = 0); CALL(C, ARG, c.sc = 0); CALL(C, ARG, c.sd = 3); CALL(C, SHAPE, c.n = 0); CALL(C, SHAPE, c.k = 0); \
    CALL(C, SHAPE, c.group = 0); CALL(C, SHAPE, c.group = 16); CALL(C, SHAPE, c.group = 96); CALL(C, SHAPE, c.group = 384); CALL(C, OK, c.group = 256); \
    CALL(C, OK, c.group = 128); CALL(C, OK, c.group = 32); CALL(C, ARG, c.codes += 8); CALL(C, ARG, c.sc += 2); CALL(C, OK, (c.sd = 1, c.sc += 2)); \
    CALL(C, ARG, c.dtype = 3); CALL(C, OK, c.z = 0); CALL(C, OK, (c.k = 160, c.group = 256)); CALL(C, SHAPE, (c.k = 160, c.group = 384));
    WEIGHTS(W) WEIGHTS(V)
    CALL(W, SHAPE, c.k = 240); CALL(W, ARG, c.w = 0); CALL(W, ARG, c.w += 2); CALL(W, SHAPE, c.n = (size_t)1 << 31);
    CALL(V, SHAPE, (c.k = 240)); CALL(V, ARG, c.x = 0); CALL(V, ARG, c.out = 0); CALL(V, SHAPE, c.rows = 0); CALL(V, SHAPE, c.ldx = 255); CALL(V, SHAPE, c.ldo = 63);
    CALL(V, ARG, c.epi = 6); CALL(V, ARG, c.epi = -1); CALL(V, ARG, c.out = c.x + 2044); CALL(V, OK, c.out = c.x + 2048); CALL(V, ARG, c.x += 1);
    CALL(V, SHAPE, c.rows = (size_t)1 << 31);
    // no context
    if (pssa_b200_w4_quantize_dev(nullptr, at(1), 0, 1, 32, 32, at<uint8_t>(16), at(4), 0, nullptr) != 1) ++bad;
    if (pssa_b200_model_score_logprobs(nullptr, 0, nullptr, nullptr, 1, 1.0f, nullptr, nullptr, nullptr, 0, nullptr, nullptr) != 1) ++bad;
    return bad;
}
"""


def test_bad_calls_are_refused_before_the_device_is_touched(tmp_path):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: a call that is in order would run")
    from pssa_b200 import build
    lib = build.build()
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    made = subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "pssa_b200" / "csrc"), "-I", str(CUDA / "include"), str(src), "-o", str(exe), str(lib),
                           f"-Wl,-rpath,{lib.parent}"], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout + ran.stderr


def test_the_python_methods_check_element_types():
    """Types are taken from the tensors; those of a raw pointer have to be named."""
    import torch

    from pssa_b200 import _native as N
    from pssa_b200.dispatch import _dtype
    assert _dtype(torch.zeros(1, dtype=torch.bfloat16), None, "x") == N.BF16
    assert _dtype(1234, "float16", "x") == N.F16 and _dtype(torch.zeros(1), "float32", "x") == N.F32
    for x, given in ((torch.zeros(1, dtype=torch.float64), None), (1234, None), (torch.zeros(1), "bfloat16"), (1234, "int8")):
        with pytest.raises(TypeError):
            _dtype(x, given, "x")
