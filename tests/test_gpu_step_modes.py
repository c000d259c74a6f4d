"""GPU tests of the step operators under the ways torch calls them: forward-mode
differentiation, torch.compile."""
import pytest
import torch
from torch.autograd import forward_ad

import mpi_collectives as mpi
from mpi_collectives import step_abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def values(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_tangents(dtype):
    """Both operators are linear: the tangent is the operator on the tangent, bit for bit, whatever its strides."""
    ids = torch.randint(-1, 40, (3, 50), generator=torch.Generator().manual_seed(1)).cuda()
    weight, grad = values(2, 40, 72, dtype=dtype), values(3, 3, 50, 72, dtype=dtype)
    weight_tangent, grad_tangent = values(4, 72, 40, dtype=dtype).t(), values(5, 3, 72, 50, dtype=dtype).transpose(1, 2)
    with forward_ad.dual_level():
        for needed in (False, True):
            w = forward_ad.make_dual(weight.clone().requires_grad_(needed), weight_tangent)
            primal, moved = forward_ad.unpack_dual(mpi.embedding(ids, w, scale=3.0))
            assert torch.equal(primal, mpi.embedding(ids, weight, scale=3.0))
            assert torch.equal(moved, mpi.embedding(ids, weight_tangent, scale=3.0))
            g = forward_ad.make_dual(grad.clone().requires_grad_(needed), grad_tangent)
            primal, moved = forward_ad.unpack_dual(mpi.embedding_gradient(g, ids, 40, scale=3.0))
            assert torch.equal(primal, mpi.embedding_gradient(grad, ids, 40, scale=3.0))
            assert torch.equal(moved, mpi.embedding_gradient(grad_tangent, ids, 40, scale=3.0))


def test_tangent_against_differences():
    """Small powers of two: the difference quotient is exact."""
    ids = torch.tensor([[2, 0, 2], [-1, 1, 2]]).cuda()
    weight = torch.tensor([[1.0, 0.5], [2.0, -1.0], [0.25, 4.0]]).cuda()
    tangent = torch.tensor([[2.0, 1.0], [0.0, -4.0], [0.5, 8.0]]).cuda()
    with forward_ad.dual_level():
        moved = forward_ad.unpack_dual(mpi.embedding(ids, forward_ad.make_dual(weight, tangent), scale=2.0)).tangent
    quotient = (mpi.embedding(ids, weight + 0.25 * tangent, scale=2.0) - mpi.embedding(ids, weight, scale=2.0)) / 0.25
    assert torch.equal(moved, quotient)


@pytest.mark.parametrize("sparse", [False, True])
def test_forward_over_backward(sparse):
    """The gradient of sum(W[ids]^2) is 2 n W where n tokens have a row, its tangent 2 n t."""
    ids = torch.tensor([2, 0, -1, 2]).cuda()
    weight, tangent = values(6, 4, 24), values(7, 4, 24)
    count = torch.tensor([[1.0], [0.0], [2.0], [0.0]]).cuda()
    with forward_ad.dual_level():
        w = weight.clone().requires_grad_(True)
        out = mpi.embedding(ids, forward_ad.make_dual(w, tangent), sparse=sparse)
        primal, moved = forward_ad.unpack_dual(torch.autograd.grad(out.square().sum(), w)[0])
    assert torch.equal(primal, 2 * count * weight) and torch.equal(moved, 2 * count * tangent)


def test_compiled_around():
    """torch.compile breaks its graph around the operators and runs them as they are."""
    import torch._dynamo
    torch._dynamo.reset()
    ids = torch.tensor([[0, 2, -1, 2], [1, 1, 0, 3]]).cuda()
    weight, update = values(8, 4, 24), values(9, 70, 90)

    def step(ids, weight, update):
        return (mpi.embedding(ids, weight * 2, scale=3.0) + 1).square().sum(), mpi.orthogonalize(update + 1) * 2

    results = []
    for f in (step, torch.compile(step, backend="eager")):
        for _ in range(2):
            leaf = weight.clone().requires_grad_(True)
            loss, out = f(ids, leaf, update)
            loss.backward()
            results.append((loss.detach(), out, leaf.grad))
    torch._dynamo.reset()
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


def test_views_that_stand_for_the_negative_of_their_memory():
    """The imaginary part of a conjugate, of one column: its memory holds the other sign at any stride the kernels take."""
    z = torch.complex(values(10, 30, 1), values(11, 30, 1))
    ids = torch.randint(-1, 30, (50,), generator=torch.Generator().manual_seed(12)).cuda()
    view, plain = z.conj().imag, -z.imag
    assert view.is_neg()
    assert torch.equal(mpi.embedding(ids, view), mpi.embedding(ids, plain))
    index = torch.arange(30).remainder(7).cuda()
    assert torch.equal(mpi.embedding_gradient(view, index, 7), mpi.embedding_gradient(plain, index, 7))
    got, want = (mpi.sum_slices(mpi.IndexedSlices(v, index, (7, 1))) for v in (view, plain))
    assert torch.equal(got.values, want.values)
    assert torch.equal(mpi.orthogonalize(view), mpi.orthogonalize(plain))
    leaf = values(13, 7, 1).requires_grad_(True)
    mpi.embedding(index, leaf).backward(view)
    assert torch.equal(leaf.grad, mpi.embedding_gradient(plain, index, 7))
    one, other = (torch.nn.Parameter(values(14, 30, 1)) for _ in range(2))
    one.grad, other.grad = view, plain
    mpi.Muon([one]).step(), mpi.Muon([other]).step()
    assert torch.equal(one, other)
    weight = torch.nn.Parameter(view)
    weight.grad = torch.ones(30, 1).cuda()
    with pytest.raises(mpi.InvalidArgumentError, match="negative"):
        mpi.Muon([weight]).step()
