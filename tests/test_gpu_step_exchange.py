"""GPU tests of the step operators' gradients through DistributedOptimizer:
sparse and dense ones in one optimizer, with and without the fusion buffer."""
import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def values(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def exchange(ranks, opts, weights, fill):
    """One step of every rank: fill(r) makes its gradients; they are exchanged and applied."""
    with mpi.Session(size=ranks) as session:
        pairs = []
        for r in range(ranks):
            with session.as_rank(r):
                opts[r].zero_grad(set_to_none=True)
                fill(r)
                pairs.append(opts[r].compute_gradients())
        session.run()
        for r in range(ranks):
            with session.as_rank(r):
                opts[r].apply_gradients(pairs[r])


@pytest.mark.parametrize("fusion", [False, True])
@pytest.mark.parametrize("ranks", [1, 3])
@pytest.mark.parametrize("with_dense", [True, False])
def test_sparse_and_dense_gradients_in_one_optimizer(ranks, fusion, with_dense):
    """The average of every rank's gradients, a sum of at most `tokens` rows and `ranks` ranks, each addition off by U of
    what has been added up, the division, the learning rate and the update by U each."""
    rows, width, tokens, lr = 40, 24, 64, 0.5
    table, matrix = values(1, rows, width), values(2, width, 10)
    weights = [[table.clone().requires_grad_(True)] + ([matrix.clone().requires_grad_(True)] if with_dense else []) for _ in range(ranks)]
    opts = [mpi.DistributedOptimizer(torch.optim.SGD(w, lr=lr), fusion=fusion) for w in weights]
    ids = [torch.randint(-1, rows, (tokens,), generator=torch.Generator().manual_seed(10 + r)).cuda() for r in range(ranks)]
    grads, dense = [values(20 + r, tokens, width) for r in range(ranks)], [values(30 + r, width, 10) for r in range(ranks)]

    def fill(r):
        mpi.embedding(ids[r], weights[r][0], sparse=True).backward(grads[r])
        if with_dense:
            (weights[r][1] * dense[r]).sum().backward()

    exchange(ranks, opts, weights, fill)
    total, size = torch.zeros(rows, width, dtype=torch.float64).cuda(), torch.zeros(rows, width, dtype=torch.float64).cuda()
    for i, g in zip(ids, grads):
        total.index_add_(0, i[i >= 0], g[i >= 0].double())
        size.index_add_(0, i[i >= 0], g[i >= 0].double().abs())
    want = table.double() - lr * total / ranks
    bound = lr / ranks * (tokens + ranks + 3) * U * size + 2 * U * want.abs()
    for w in weights:
        assert bool(((w[0].detach().double() - want).abs() <= bound).all())
        assert w[0].grad.is_sparse and w[0].grad.is_coalesced()
        if with_dense:
            mean, most = sum(d.double() for d in dense) / ranks, sum(d.double().abs() for d in dense) / ranks
            assert bool(((w[1].detach().double() - (matrix.double() - lr * mean)).abs() <= lr * (ranks + 3) * U * most + 2 * U * w[1].detach().double().abs()).all())
    for w in weights[1:]:
        assert all(torch.equal(a, b) for a, b in zip(w, weights[0]))


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("fusion", [False, True])
@pytest.mark.parametrize("ranks", [1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_gradients_are_exchanged_in_32(dtype, ranks, fusion):
    """Each rank's own gradient is rounded to the type once (half a step h of each), the average once, its product with the
    learning rate and the new weight once each by the optimizer; float32 additions besides. What is below float16's smallest
    normal number is rounded to a multiple of 2^-24. The replicas are the same bit for bit."""
    rows, width, tokens, lr, h = 40, 24, 64, 0.5, HALF_STEP[dtype]
    table, matrix, third = values(1, rows, width, dtype=dtype), values(2, width, 10, dtype=dtype), values(3, 7)
    weights = [[t.clone().requires_grad_(True) for t in (table, matrix, third)] for _ in range(ranks)]
    opts = [mpi.DistributedOptimizer(torch.optim.SGD(w, lr=lr), fusion=fusion) for w in weights]
    ids = [torch.randint(-1, rows, (tokens,), generator=torch.Generator().manual_seed(10 + r)).cuda() for r in range(ranks)]
    grads = [values(20 + r, tokens, width, dtype=dtype) for r in range(ranks)]
    dense, small = [values(30 + r, width, 10, dtype=dtype) for r in range(ranks)], [values(40 + r, 7) for r in range(ranks)]

    def fill(r):
        mpi.embedding(ids[r], weights[r][0], sparse=True).backward(grads[r])
        weights[r][1].grad = dense[r].clone()
        weights[r][2].grad = small[r].clone()                     # a float32 one beside them

    for step in range(2):
        before = [[w.detach().clone() for w in ws] for ws in weights]
        exchange(ranks, opts, weights, fill)
        local = []
        for i, g in zip(ids, grads):
            local.append(torch.zeros(rows, width, dtype=torch.float64).cuda().index_add_(0, i[i >= 0], g[i >= 0].double()))
        size = sum(torch.zeros(rows, width, dtype=torch.float64).cuda().index_add_(0, i[i >= 0], g[i >= 0].double().abs()) for i, g in zip(ids, grads))
        for k, (locals_, sizes) in enumerate(((local, size), ([d.double() for d in dense], sum(d.double().abs() for d in dense)))):
            mean = sum(locals_) / ranks
            want = before[0][k].double() - lr * mean
            slack = lr / ranks * (tokens + ranks + 3) * U * sizes
            bound = 1.01 * (lr * h * (sum(x.abs() for x in locals_) / ranks + 2 * mean.abs()) + h * want.abs() + slack) + 4 * 2.0 ** -25
            for w in weights:
                assert w[k].grad.dtype == dtype
                assert bool(((w[k].detach().double() - want).abs() <= bound).all())
        mean = sum(s.double() for s in small) / ranks
        assert bool(((weights[0][2].detach().double() - (before[0][2].double() - lr * mean)).abs() <= 1e-6).all())
        for w in weights[1:]:
            assert all(torch.equal(a, b) for a, b in zip(w, weights[0]))


@pytest.mark.parametrize("fusion", [False, True])
def test_muon_in_bfloat16_through_the_exchange(fusion):
    """The same step as Muon alone on the average rounded once, bit for bit."""
    ranks, shapes = 3, [(70, 90), (64, 64), (130, 40)]
    make = lambda: [torch.nn.Parameter(values(k, *s, dtype=torch.bfloat16)) for k, s in enumerate(shapes)]  # noqa: E731
    weights, mirror = [make() for _ in range(ranks)], make()
    opts = [mpi.DistributedOptimizer(mpi.Muon(w, weight_decay=0.1), fusion=fusion) for w in weights]
    alone = mpi.Muon(mirror, weight_decay=0.1)
    for step in range(2):
        grads = [[values(100 * step + 10 * r + k, *s, dtype=torch.bfloat16) for k, s in enumerate(shapes)] for r in range(ranks)]

        def fill(r):
            for w, g in zip(weights[r], grads[r]):
                w.grad = g.clone()

        exchange(ranks, opts, weights, fill)
        for k, w in enumerate(mirror):
            got = weights[0][k].grad
            mean = sum(g[k].double() for g in grads) / ranks
            most = sum(g[k].double().abs() for g in grads) / ranks
            assert bool(((got.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + (ranks + 1) * U * most * 1.01).all())
            w.grad = got
        alone.step()
        for ws in weights:
            assert all(torch.equal(a, b) for a, b in zip(ws, mirror))


@pytest.mark.parametrize("distinct", [1, 3, 300, 499, 500, 501, 999, 1000])
def test_summed_slices_keep_no_more_than_twice_their_size(distinct):
    """Every rank's rows are set aside for the sum; a gradient of few distinct rows must not keep them until the next step."""
    count, width = 1000, 64
    ids = torch.arange(count).remainder(distinct).cuda()
    rows = values(50, count, width)
    got = mpi.sum_slices(mpi.IndexedSlices(rows, ids, (5000, width)))
    assert got.indices.tolist() == list(range(distinct)) and got.values.shape == (distinct, width)
    for t in (got.indices, got.values):
        assert t.is_contiguous() and t.untyped_storage().nbytes() <= 2 * t.numel() * t.element_size()
    weight = values(51, 5000, width).requires_grad_(True)
    mpi.embedding(ids, weight, sparse=True).backward(rows)
    assert torch.equal(weight.grad._values(), got.values)
    assert weight.grad._values().untyped_storage().nbytes() <= 2 * got.values.numel() * 4


@pytest.mark.parametrize("fusion", [False, True])
def test_repeated_indices_of_a_16_bit_gradient_are_summed_in_32(fusion):
    """torch's own sparse gradient holds a row per token: 300 ones are 300, not the 256 where bfloat16 stops counting."""
    weights = [torch.zeros(3, 8, dtype=torch.bfloat16, device="cuda").requires_grad_(True) for _ in range(2)]
    opts = [mpi.DistributedOptimizer(torch.optim.SGD([w], lr=1.0), fusion=fusion) for w in weights]

    def fill(r):
        torch.nn.functional.embedding(torch.zeros(300, dtype=torch.int64).cuda(), weights[r], sparse=True).sum().backward()

    exchange(2, opts, weights, fill)
    for w in weights:
        assert torch.equal(w.detach().cpu(), torch.tensor([[-300.0], [0.0], [0.0]]).expand(3, 8).bfloat16())
