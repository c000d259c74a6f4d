"""Checks of the step operators that need no GPU: the C ABI against its
binding, refusals, the embedding kernels compiled for the CPU under the
sanitizers (tests/cpp/step_emulation_test.cc), and a scan of the assembly for
selects on a stale condition code (see test_kernels_on_cpu.py)."""
import ctypes
import os
import re
import shutil

import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi
from test_kernels_on_cpu import BUILD, HIP_FLAGS, ROOT, SANITIZERS, SHIM, _clang, _run, kernels_in_scratch, stale_selects

CSRC = os.path.join(ROOT, "tensorflow-allreduce_amd", "csrc")
EMBEDDING = os.path.join(CSRC, "step_embedding.hip")
ORTHOGONALIZE = os.path.join(CSRC, "step_orthogonalize.hip")
HEADERS = [os.path.join(ROOT, "include", "step_abi.h"), os.path.join(CSRC, "step_common.h")]


def test_binding_covers_the_header():
    text = open(HEADERS[0]).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = sorted(set(re.findall(r"\b(step_\w+)\s*\(", text)))
    assert sorted(step_abi.EXPORTS) == declared
    lib = step_abi.lib()
    assert lib.step_abi_version() == 1
    for status in range(6):
        assert lib.step_status_string(status)


def test_pieces_are_half_the_square_root_and_at_least_64():
    lib = step_abi.lib()
    for tokens, piece in ((0, 64), (1, 64), (16384, 64), (16385, 128), (65536, 128), (1 << 20, 512)):
        assert lib.step_embedding_piece(tokens) == piece


def test_workspace_of_sizes_that_do_not_fit_is_zero():
    lib = step_abi.lib()
    assert lib.step_embedding_gradient_workspace(1 << 31, 8, 4) == 0
    assert lib.step_sum_slices_workspace(8, 1 << 31, 4) == 0
    assert lib.step_embedding_gradient_workspace(0, 0, 0) > 0


@pytest.mark.parametrize("call, words", [
    (lambda: mpi.embedding([1, 2], torch.zeros(3, 3)), "torch.Tensor"),
    (lambda: mpi.embedding(torch.zeros(2), torch.zeros(3, 3)), "ids has type"),
    (lambda: mpi.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 3)), "GPU kernels only"),
    (lambda: mpi.embedding_gradient(torch.zeros(2, 3, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 5), "grad has type"),
    (lambda: mpi.embedding_gradient(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), 5), "GPU kernels only"),
    (lambda: mpi.orthogonalize(torch.zeros(3, 3)), "GPU kernels only"),
    (lambda: mpi.orthogonalize(torch.zeros(3, 3, dtype=torch.float64)), "update has type"),
    (lambda: mpi.Muon([torch.nn.Parameter(torch.zeros(3))]), "it takes matrices"),
    (lambda: mpi.Muon([torch.nn.Parameter(torch.zeros(3, 3))], adjust="x"), "adjust is"),
    (lambda: mpi.Muon([torch.nn.Parameter(torch.zeros(3, 3))], coefficients=(1, 2)), "coefficients are"),
    (lambda: mpi.sum_slices(torch.zeros(2, 3)), "IndexedSlices"),
    (lambda: mpi.sum_slices(mpi.IndexedSlices(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64), (5, 3))), "GPU kernels only"),
])
def test_refusals_before_any_gpu_work(call, words):
    with pytest.raises(mpi.InvalidArgumentError, match=re.escape(words)):
        call()


def _emulation(sanitizer):
    clang = _clang()
    if clang is None:
        pytest.skip("no clang++ (the kernels use clang vector extensions)")
    os.makedirs(BUILD, exist_ok=True)
    shim = os.path.join(ROOT, "tests", "cpp", "step_wave_shim.h")
    test = os.path.join(ROOT, "tests", "cpp", "step_emulation_test.cc")
    flags = ["-std=c++17", "-O1", "-g", "-mf16c", "-fno-omit-frame-pointer", "-pthread", "-I", SHIM,
             "-I", os.path.join(ROOT, "include")] + SANITIZERS[sanitizer]
    obj = os.path.join(BUILD, "step_embedding_cpu_%s.o" % sanitizer)
    exe = os.path.join(BUILD, "step_emulation_test_" + sanitizer)
    _run([clang, "-x", "c++"] + flags + ["-I", CSRC, "-include", shim, "-c", "-o", obj, EMBEDDING])
    _run([clang] + flags + ["-o", exe, test, obj])
    return exe


@pytest.mark.parametrize("sanitizer, arguments", [("asan", []), ("tsan", ["brief"])])
def test_embedding_kernels_under_sanitizers_on_the_cpu(sanitizer, arguments):
    env = dict(os.environ, TSAN_OPTIONS="halt_on_error=1:report_signal_unsafe=0")
    out = _run([_emulation(sanitizer)] + arguments, timeout=900, env=env)
    assert "step emulation: ok" in out, out[-4000:]


def _assembly(source):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    os.makedirs(BUILD, exist_ok=True)
    asm = os.path.join(BUILD, os.path.basename(source).replace(".hip", "_gfx950.s"))
    sources = [source, os.path.abspath(__file__)] + HEADERS
    if not os.path.exists(asm) or os.path.getmtime(asm) < max(os.path.getmtime(f) for f in sources):
        _run([hipcc] + HIP_FLAGS + ["-I", os.path.join(ROOT, "include"), "-S", "--cuda-device-only", "-o", asm, source])
    return open(asm).read()


def test_embedding_refuses_what_no_launch_holds():
    """A launch has less than 2^32 lanes; the pointers are never followed."""
    lib = step_abi.lib()
    p, big = 4096, 1 << 62

    def lookup(tokens, width):
        return lib.step_embedding_lookup(p, 1, tokens, p, 3, 100, width, width, 1.0, p, None)

    def gradient(tokens, rows, width):
        return lib.step_embedding_gradient(p, 1, tokens, p, 3, rows, width, width, 1.0, p, p, big, None)

    def slices(tokens, width):
        return lib.step_sum_slices(p, 1, tokens, p, 3, 100, width, width, 1.0, p, p, p, p, big, None)

    limit = 5
    assert lookup(1 << 26, 2048) == lookup((1 << 31) - 1, 512) == limit
    assert gradient(1 << 27, 100, 2048) == gradient(1 << 26, 100, 4096) == gradient(100, 1 << 30, 1) == limit
    assert slices(1 << 27, 2048) == slices(1 << 26, 4096) == limit


def test_orthogonalize_refuses_on_the_host():
    """The C entry points' own checks, with pointers that are never followed."""
    lib = step_abi.lib()
    M = step_abi.Matrix
    one = M(4096, 4096, 4096, 100, 200, 3, 0.1)
    size = lib.step_orthogonalize_workspace(one, 1, 0)
    assert size > 3 * 128 * 256 * 2 * 4 and lib.step_orthogonalize_workspace(one, 1, 1) > size
    abc = (ctypes.c_float * 15)()

    def call(m=one, length=1, dtype=0, out=0, steps=5, table=abc, ws=4096, bytes=size):
        return lib.step_orthogonalize(m, length, dtype, out, 0, steps, table, 0.0, ws, bytes, None)

    assert call(dtype=1) == call(out=2) == 1
    assert call(steps=0) == call(steps=65) == call(table=None) == call(ws=None) == call(ws=4097) == call(bytes=size - 1) == 2
    assert call(m=None) == 2
    assert call(m=M(None, None, 4096, 100, 200, 3, 0)) == call(m=M(4096, None, None, 100, 200, 3, 0)) == 2
    assert call(m=M(4096, None, 4096, (1 << 20) + 1, 1, 1, 0)) == call(m=M(4096, None, 4096, 1 << 20, 1 << 20, 1, 0)) == 5
    assert lib.step_muon(M(4096, None, 4096, 100, 200, 3, 0), 1, 0, 0, 5, abc, 0.0, 0.9, 1, 1.0, 4096, size, None) == 2
    for empty in (M(None, None, None, 0, 700, 3, 0), M(None, None, None, 700, 0, 3, 0), M(None, None, None, 700, 700, 0, 0)):
        assert lib.step_orthogonalize_workspace(empty, 1, 0) == 0 and call(m=empty, ws=None, bytes=0) == 0
    # the workspace of a long list is that of its largest round, not of the whole list
    many = (M * 500)(*[M(4096, 4096, 4096, 4096, 4096, 1, 0.1) for _ in range(500)])
    assert lib.step_orthogonalize_workspace(many, 500, 0) < 6 << 30
    assert lib.step_orthogonalize_workspace(M(4096, None, 4096, 65, 65, 10 ** 7, 0), 1, 0) < 4 << 30
    # small ones need none
    assert lib.step_orthogonalize_workspace(M(4096, None, 4096, 64, 256, 10 ** 7, 0), 1, 1) == 0


def test_orthogonalize_assembly():
    text = _assembly(ORTHOGONALIZE)
    found = stale_selects(text)
    assert not found, "scalar selects on a stale condition code: %r" % (found[:5],)
    kernels = kernels_in_scratch(text, ("norm_kernel", "first_kernel", "product_kernel", "small_kernel"))
    assert kernels["seen"] >= 37 and not kernels["scratch"], kernels


def test_embedding_assembly():
    text = _assembly(EMBEDDING)
    found = stale_selects(text)
    assert not found, "scalar selects on a stale condition code: %r" % (found[:5],)
    kernels = kernels_in_scratch(text, ("lookup_kernel", "sort_one_kernel", "scatter_kernel", "sum_kernel", "join_kernel"))
    assert kernels["seen"] >= 17 and not kernels["scratch"], kernels


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_slices_on_the_cpu_are_applied_as_ever(dtype):
    """apply_gradients with slices that are not on the GPU, or of a type that sum_slices does not take."""
    w = torch.zeros(5, 3, dtype=dtype, requires_grad=True)
    slices = mpi.IndexedSlices(torch.ones(4, 3, dtype=dtype), torch.tensor([1, 4, 1, 0]), (5, 3))
    mpi.DistributedOptimizer(torch.optim.SGD([w], lr=1.0)).apply_gradients([(slices, w)])
    assert w[:, 0].tolist() == [-1.0, -2.0, 0.0, 0.0, -1.0] and w.grad.is_coalesced()
