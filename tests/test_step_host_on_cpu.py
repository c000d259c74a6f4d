"""Host side of the step operators, without a GPU: what a list of matrices asks
for, and what the Python entry points do before any kernel is launched."""
import ctypes
import types

import pytest
import torch
from torch.autograd import forward_ad

import mpi_collectives as mpi
from mpi_collectives import step_abi, step_ops


def matrices(*shapes):
    return (step_abi.Matrix * len(shapes))(*[step_abi.Matrix(4096, 4096, 4096, r, c, 1, 0.1) for r, c in shapes])


def test_small_matrices_need_no_workspace_among_larger_ones():
    """Unless all are precise: then they ride along with the larger ones' products."""
    lib = step_abi.lib()
    mixed, large = matrices((64, 256), (300, 200), (20, 30)), matrices((300, 200))
    assert lib.step_orthogonalize_workspace(mixed, 3, 0) == lib.step_orthogonalize_workspace(large, 1, 0) > 0
    assert lib.step_orthogonalize_workspace(mixed, 3, 1) > lib.step_orthogonalize_workspace(large, 1, 1) > 0
    for precise in (0, 1):
        assert lib.step_orthogonalize_workspace(matrices((64, 256), (20, 30)), 2, precise) == 0


@pytest.fixture
def plain(monkeypatch):
    """The kernels of the lookup and its gradient as plain torch operations on the CPU, invisible to autograd."""
    def lookup(ids, weight, scale):
        inside = ((ids >= 0) & (ids < weight.shape[0])).unsqueeze(-1)
        out = torch.where(inside, scale * weight.detach()[ids.clamp(0, weight.shape[0] - 1)], 0.0)
        return torch.from_numpy(out.numpy().copy())

    def gradient(grad, ids, rows, scale):
        inside = (ids >= 0) & (ids < rows)
        out = torch.zeros(rows, grad.shape[-1], dtype=grad.dtype).index_add(0, ids[inside], scale * grad.detach()[inside])
        return torch.from_numpy(out.numpy().copy())

    monkeypatch.setattr(step_ops, "_lookup", lambda *a: torch.no_grad()(lookup)(*a))
    monkeypatch.setattr(step_ops, "_gradient", lambda *a: torch.no_grad()(gradient)(*a))
    monkeypatch.setattr(step_ops, "_check_tensor", lambda *a: None)


IDS = torch.tensor([[2, 0, -1], [2, 5, 1]])


def test_forward_mode(plain):
    """Both operators are linear: the tangent of the result is the operator on the tangent."""
    weight, tangent = torch.randn(4, 3), torch.randn(4, 3)
    grad, grad_tangent = torch.randn(2, 3, 3), torch.randn(2, 3, 3)
    with forward_ad.dual_level():
        for needed in (False, True):
            w = forward_ad.make_dual(weight.clone().requires_grad_(needed), tangent)
            primal, moved = forward_ad.unpack_dual(mpi.embedding(IDS, w, scale=2.0))
            assert torch.equal(primal, mpi.embedding(IDS, weight, scale=2.0))
            assert torch.equal(moved, mpi.embedding(IDS, tangent, scale=2.0))
            g = forward_ad.make_dual(grad.clone().requires_grad_(needed), grad_tangent)
            primal, moved = forward_ad.unpack_dual(mpi.embedding_gradient(g, IDS, 4, scale=2.0))
            assert torch.equal(primal, mpi.embedding_gradient(grad, IDS, 4, scale=2.0))
            assert torch.equal(moved, mpi.embedding_gradient(grad_tangent, IDS, 4, scale=2.0))
        with torch.no_grad():
            moved = forward_ad.unpack_dual(mpi.embedding(IDS, forward_ad.make_dual(weight, tangent))).tangent
            assert torch.equal(moved, mpi.embedding(IDS, tangent))
        assert forward_ad.unpack_dual(mpi.embedding(IDS, weight)).tangent is None
        zero = torch._efficientzerotensor(4, 3)
        assert not forward_ad.unpack_dual(mpi.embedding(IDS, forward_ad.make_dual(weight, zero))).tangent.any()


@pytest.mark.parametrize("sparse", [False, True])
def test_forward_over_backward(plain, sparse):
    """A Hessian times a vector: the gradient of sum((2 W[ids])^3) is 24 n W^2 where n tokens have a row, its tangent 48 n W t."""
    weight, tangent = torch.randn(4, 3, dtype=torch.float64), torch.randn(4, 3, dtype=torch.float64)
    with forward_ad.dual_level():
        w = weight.clone().requires_grad_(True)
        out = mpi.embedding(IDS, forward_ad.make_dual(w, tangent), scale=2.0, sparse=sparse)
        first, = torch.autograd.grad(out.pow(3).sum(), w)
        primal, moved = forward_ad.unpack_dual(first)
    count = torch.tensor([1.0, 1.0, 2.0, 0.0], dtype=torch.float64).unsqueeze(1)
    assert torch.allclose(primal, 24 * count * weight ** 2) and torch.allclose(moved, 48 * count * weight * tangent)


def test_backward_over_forward(plain):
    """The tangent of the result is differentiable with respect to the table's tangent."""
    weight, tangent = torch.randn(4, 3), torch.randn(4, 3, requires_grad=True)
    with forward_ad.dual_level():
        moved = forward_ad.unpack_dual(mpi.embedding(IDS, forward_ad.make_dual(weight, tangent), scale=2.0)).tangent
    moved.sum().backward()
    assert tangent.grad[:, 0].tolist() == [2.0, 2.0, 4.0, 0.0]


def _muon(weight):
    opt = mpi.Muon([torch.nn.Parameter(weight)])
    opt.step()
    return weight


@pytest.mark.parametrize("call", [
    lambda x: mpi.embedding(IDS, x), lambda x: mpi.embedding(IDS, x.clone().requires_grad_(True)),
    lambda x: mpi.embedding_gradient(x, torch.tensor([1, 0, 2, 2]), 5), lambda x: mpi.orthogonalize(x),
    lambda x: mpi.sum_slices(mpi.IndexedSlices(x, torch.tensor([1, 0, 2, 2]), (4, 3))).values, _muon])
def test_what_records_a_trace_is_refused(plain, call):
    """A trace would hold the empty result and not the launch that fills it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 3)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(mpi.InvalidArgumentError, match="does not hold"):
            make_fx(call, tracing_mode=mode)(x)
    with pytest.raises(mpi.InvalidArgumentError, match="does not hold"):
        torch.jit.trace(call, x)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(mpi.InvalidArgumentError, match="does not hold"):
        call(x)


def test_other_modes_of_torch_are_none_of_a_trace(plain):
    """Counting flops, say."""
    from torch.utils.flop_counter import FlopCounterMode
    weight = torch.randn(4, 3)
    with FlopCounterMode(display=False):
        out = mpi.embedding(IDS, weight)
    assert torch.equal(out, mpi.embedding(IDS, weight))


def _slices(rows, row, dense_rows, dtype=torch.float32):
    """Stand-ins for tensors on the GPU that nothing reads."""
    meta = lambda shape, kind: types.SimpleNamespace(  # noqa: E731
        is_cuda=True, dtype=kind, shape=torch.Size(shape), dim=lambda: len(shape), element_size=lambda: kind.itemsize)
    return mpi.IndexedSlices(meta((rows, row), dtype), meta((rows,), torch.int64), (dense_rows, row))


@pytest.mark.parametrize("rows, row, dense_rows, dtype, fits", [
    (5, 3, 7, torch.float32, True), (5, 3, 7, torch.float64, False),
    (5, 3, (1 << 31) - 1, torch.float32, True), (5, 3, 1 << 31, torch.float32, False), (5, 3, 1 << 40, torch.float32, False),
    ((1 << 31) - 1, 1, 9, torch.bfloat16, True), (1 << 31, 1, 9, torch.bfloat16, False),
    (2, 67107840, 9, torch.float32, True), (2, 67107841, 9, torch.float32, False),
    (1 << 24, 1024, 9, torch.float32, True), (1 << 27, 1024, 9, torch.float32, False), (1 << 28, 2048, 9, torch.bfloat16, False)])
def test_slices_beyond_the_kernels_sizes_go_to_torch(rows, row, dense_rows, dtype, fits):
    """apply_gradients asks can_sum_slices first; what it lets through, the entry point takes."""
    slices = _slices(rows, row, dense_rows, dtype)
    assert step_ops.can_sum_slices(slices) == fits
    if fits:
        code = {torch.float32: 0, torch.bfloat16: 3}[dtype]
        status = step_abi.lib().step_sum_slices(4096, 2, rows, 4096, code, dense_rows, row, row, 1.0, 4096, 4096,
                                                ctypes.c_void_p(4096), None, 0, None)
        assert status == 2          # only the workspace is missing: the sizes passed
    slices.dense_shape = None
    assert not step_ops.can_sum_slices(slices)


# Batches of matrices and the sides of the tiles their products take (X X^T, A A, B X and the last B X), chosen so that
# every kernel there is runs, with tiles that the matrix's edge cuts, in more than one step.
TILES = {
    ((1, 300, 500), False): (64, 64, 64, 64),
    ((7, 1040, 1220), False): (128, 128, 128, 128),
    ((1, 2731, 1000), False): (64, 64, 128, 128),
    ((3, 1900, 2500), False): (128, 128, 256, 256),
    ((3, 2220, 2230), False): (192, 192, 256, 256),
    ((3, 2440, 2460), False): (256, 256, 128, 128),
    ((1, 300, 500), True): (64, 64, 64, 64),
    ((1, 1000, 2731), True): (64, 64, 128, 128),
    ((3, 2220, 2400), True): (128, 128, 128, 128),
    ((9, 1040, 1220), True): (128, 128, 128, 128),
}


@pytest.mark.parametrize("shape, precise", TILES)
def test_sides_of_tiles(shape, precise):
    lib, (count, rows, cols) = step_abi.lib(), shape
    one = step_abi.Matrix(4096, None, 4096, rows, cols, count, 0.0)
    assert tuple(lib.step_orthogonalize_side(one, 1, precise, k) for k in range(4)) == TILES[shape, precise]
    assert lib.step_orthogonalize_side(one, 1, precise, 4) == 0


def test_every_tile_there_is_has_a_test():
    for precise, kernels in ((False, [{64, 128, 192, 256}, {64, 128, 192, 256}, {64, 128, 256}, {64, 128, 256}]), (True, [{64, 128}] * 4)):
        for k, sides in enumerate(kernels):
            assert {t[k] for (_, p), t in TILES.items() if p == precise} == sides


def test_sides_of_nothing():
    lib = step_abi.lib()
    for m in (matrices((64, 256)), matrices((0, 500)), matrices()):
        assert [lib.step_orthogonalize_side(m, len(m), 0, k) for k in range(4)] == [0] * 4


def test_views_that_stand_for_the_negative_of_their_memory(plain):
    """The imaginary part of a conjugate is one: the kernels read memory, so it has to be made to hold the values."""
    z = torch.randn(4, 1, dtype=torch.complex64)
    weight = z.conj().imag
    assert weight.is_neg()
    assert torch.equal(mpi.embedding(IDS, weight), mpi.embedding(IDS, -z.imag))
    leaf = z.conj().imag.resolve_neg().clone().requires_grad_(True)
    grad = torch.randn(2, 3, 1, dtype=torch.complex64)
    mpi.embedding(IDS, leaf).backward(grad.conj().imag)
    assert torch.equal(leaf.grad, mpi.embedding_gradient(-grad.imag, IDS, 4))
    assert torch.equal(mpi.embedding_gradient(grad.conj().imag, IDS, 4), leaf.grad)
