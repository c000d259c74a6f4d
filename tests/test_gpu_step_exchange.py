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
