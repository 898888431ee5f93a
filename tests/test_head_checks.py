"""More of what the operators on a head's weights and logits refuse, on the CPU: checked before the device is touched."""
import subprocess

import pytest

from test_head_refusals import CUDA, PROGRAM, ROOT

pytestmark = pytest.mark.skipif(not (CUDA / "include" / "cuda_runtime.h").exists(), reason="no CUDA headers")


def run_checks(tmp_path, lines):
    """The program of test_head_refusals with other calls."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: a call that is in order would run")
    from pssa_b200 import build
    lib = build.build()
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM[:PROGRAM.index("int main()")] + "int main() {\n" + lines + "\nreturn bad;\n}\n")
    made = subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "pssa_b200" / "csrc"), "-I", str(CUDA / "include"), str(src), "-o", str(exe), str(lib),
                           f"-Wl,-rpath,{lib.parent}"], capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout + ran.stderr


def test_arrays_of_words_start_on_words(tmp_path):
    """A misaligned one would be a fault of the device."""
    run_checks(tmp_path, "".join(f"CALL({call}, ARG, c.{array} += {by});\n" for call, arrays in
                                 (("L", ("tgt", "lp", "rank", "h", "st", "ids", "top")), ("G", ("tgt", "st", "h", "glp", "gh")),
                                  ("D", ("ids", "te", "tgt", "kl", "ce", "gk", "gc"))) for array in arrays for by in (1, 2, 3)) +
               "CALL(W, OK, c.z += 1); CALL(V, OK, c.z += 3); CALL(L, OK, c.tgt += 4); CALL(D, OK, c.te += 4);")



def test_rows_may_lie_between_each_other(tmp_path):
    """Two arrays with the same pitch in bytes whose rows alternate share no element; anything less is refused."""
    run_checks(tmp_path, "".join(f"""
CALL({c}, OK, (c.ld = 2000, c.ldg = 2000, c.g = c.x + 4000)); CALL({c}, OK, (c.ld = 2000, c.ldg = 2000, c.g = c.x - 4000));
CALL({c}, ARG, (c.ld = 2000, c.ldg = 2000, c.g = c.x + 3996)); CALL({c}, ARG, (c.ld = 2000, c.ldg = 2000, c.g = c.x + 4004));
CALL({c}, OK, (c.ld = 2001, c.ldg = 2001, c.g = c.x + 4004)); CALL({c}, OK, (c.ld = 2001, c.ldg = 2001, c.g = c.x + 8004 + 4000));
CALL({c}, ARG, (c.ld = 1999, c.ldg = 1999, c.g = c.x + 4000)); CALL({c}, ARG, (c.ld = 2000, c.ldg = 2001, c.g = c.x + 4000));
CALL({c}, OK, (c.dtype = 1, c.ld = 2000, c.ldg = 2000, c.g = c.x + 2000));
""" for c in "GD") + """
CALL(V, OK, (c.ldx = 320, c.ldo = 320, c.out = c.x + 1024)); CALL(V, ARG, (c.ldx = 320, c.ldo = 320, c.out = c.x + 1020));
CALL(V, ARG, (c.ldx = 320, c.ldo = 320, c.out = c.x + 1028)); CALL(V, ARG, (c.ldx = 319, c.ldo = 319, c.out = c.x + 1024));
CALL(V, OK, (c.ldx = 320, c.ldo = 320, c.out = c.x - 256)); CALL(V, ARG, (c.ldx = 320, c.ldo = 64, c.out = c.x + 1024));
""")


class Array:
    """What the methods look at of a tensor."""

    def __init__(self, dtype="float32", device=0, dense=True, last=1):
        import torch
        self.dtype, self._device, self._dense, self._last = getattr(torch, dtype), device, dense, last

    def data_ptr(self):
        return 64

    def get_device(self):
        return self._device

    def is_contiguous(self):
        return self._dense

    def stride(self, dim):
        return self._last


def calls_of(gpu):
    """Each method with arrays that are in order, and which of them are ids, numbers in fp32, bytes or rows with a pitch."""
    f, i, b = Array, lambda: Array("int32"), lambda: Array("uint8")
    rows = lambda: Array(dense=False)  # noqa: E731
    return [
        (lambda a: gpu.token_logprobs_dev(a.pop("logits"), 4, 10, a.pop("targets"), top_n=3, **a),
         dict(logits=rows(), targets=i(), logprob=f(), rank=i(), entropy=f(), stats=f(), top_ids=Array("uint32"), top_logprobs=f())),
        (lambda a: gpu.token_logprobs_grad_dev(a.pop("logits"), 4, 10, a.pop("targets"), a.pop("stats"), a.pop("grad_logits"), **a),
         dict(logits=rows(), targets=i(), stats=f(), grad_logits=rows(), grad_logprob=f(), entropy=f(), grad_entropy=f())),
        (lambda a: gpu.distill_topk_dev(a.pop("logits"), 4, 10, a.pop("teacher_ids"), a.pop("teacher"), 3, **a),
         dict(logits=rows(), teacher_ids=i(), teacher=f(), kl=f(), grad_kl=f(), targets=i(), ce=f(), grad_ce=f(), grad_logits=rows())),
        (lambda a: gpu.w4_quantize_dev(a.pop("w"), 4, 64, 32, a.pop("codes"), a.pop("scales"), a.pop("zeros")),
         dict(w=Array("bfloat16"), codes=b(), scales=f(), zeros=b())),
        (lambda a: gpu.gemv_w4_dev(a.pop("x"), 2, a.pop("codes"), a.pop("scales"), a.pop("zeros"), 4, 64, 32, a.pop("out")),
         dict(x=rows(), codes=b(), scales=Array("float16"), zeros=b(), out=rows())),
    ]


def test_the_python_methods_check_every_array():
    """int64 ids, as argmax and multinomial give them, would be read as pairs of words, fp64 or bf16 numbers as others; arrays of the
    host or of another device would be a fault, strided ones other elements."""
    import numpy as np
    from pssa_b200 import dispatch as D
    gpu = D.B200Dispatch.__new__(D.B200Dispatch)
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or 0

    gpu._lib, gpu._h, gpu.device = Lib(), None, 0
    ids = {"targets", "rank", "top_ids", "teacher_ids"}
    for n, (call, good) in enumerate(calls_of(gpu)):
        call(dict(good))
        raw = dict(good)
        for name in raw:
            if not (name in ("logits", "x", "w", "scales", "out", "grad_logits")):
                raw[name] = 64  # an address is taken as it is
        call(raw)
        assert len(seen) == 2 * n + 2
        for name, a in good.items():
            typed = name in ("logits", "x", "w", "scales", "out", "grad_logits")
            wrong = [Array("float64"), Array("int64"), Array("int16"), np.zeros(4, np.float32)]
            if name in ids:
                wrong.append(Array("float32"))
            elif not typed:
                wrong.append(Array("bfloat16"))
            kind = str(a.dtype)[6:]
            wrong += [Array(kind, device=-1), Array(kind, device=1), Array(kind, dense=False, last=2)]
            if name not in ("logits", "x", "out", "grad_logits"):
                wrong.append(Array(kind, dense=False))
            for w in wrong:
                with pytest.raises(TypeError, match=name):
                    call(dict(good, **{name: w}))
    assert len(seen) == 10
