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
