"""The orthogonalisation's kernels compiled for the CPU under the sanitizers
(tests/cpp/step_orthogonalize_emulation_test.cc): every index is bounds-checked,
and loads into LDS land as late as the kernels' own waits allow."""
import os

import pytest

from test_kernels_on_cpu import BUILD, ROOT, SANITIZERS, SHIM, _clang, _run

SOURCE = os.path.join(ROOT, "tensorflow-allreduce_amd", "csrc", "step_orthogonalize.hip")
CPP = os.path.join(ROOT, "tests", "cpp")


@pytest.mark.parametrize("sanitizer, arguments", [("asan", []), ("tsan", ["brief"])])
def test_kernels_under_sanitizers(sanitizer, arguments):
    clang = _clang()
    if clang is None:
        pytest.skip("no clang++ (the kernels use clang vector extensions)")
    os.makedirs(BUILD, exist_ok=True)
    flags = ["-std=c++17", "-O0", "-g1", "-mf16c", "-fno-omit-frame-pointer", "-pthread", "-Wno-pass-failed", "-I", SHIM, "-I", CPP,
             "-I", os.path.join(ROOT, "include")] + SANITIZERS[sanitizer]
    obj = os.path.join(BUILD, "step_orthogonalize_cpu_%s.o" % sanitizer)
    exe = os.path.join(BUILD, "step_orthogonalize_emulation_test_" + sanitizer)
    _run([clang, "-x", "c++"] + flags + ["-I", os.path.dirname(SOURCE), "-include", "step_matrix_shim.h", "-c", "-o", obj, SOURCE])
    _run([clang] + flags + ["-o", exe, os.path.join(CPP, "step_orthogonalize_emulation_test.cc"), obj])
    env = dict(os.environ, TSAN_OPTIONS="halt_on_error=1:report_signal_unsafe=0")
    out = _run([exe] + arguments, timeout=900, env=env)
    assert "step orthogonalize emulation: ok" in out, out[-4000:]
