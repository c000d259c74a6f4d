"""GPU tests of how far the products of single fp16 operands (precise=False)
may be off, against the definition in 64 bits."""
import math

import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi
from test_gpu_orthogonalize import A, B, C

pytestmark = pytest.mark.gpu

# Mean size (root of the mean square) of the relative rounding to fp16 of values spread evenly over their logarithm:
# 2^-10 / sqrt(12) over a mantissa between 1 and 2, sqrt(3 / (8 ln 2)) of it.
ROUNDING = 2.0 ** -10 / math.sqrt(12) * math.sqrt(3 / (8 * math.log(2)))


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def outer(seed, rows, cols, count=None):
    gen = torch.Generator().manual_seed(seed)
    batch = () if count is None else (count,)
    return (1e-3 * torch.randn(*batch, rows, 1, generator=gen) * torch.randn(*batch, 1, cols, generator=gen)).cuda()


def exact_there(update, steps=5):
    """exact() of one matrix, on its device."""
    x = update.double()
    tall = x.shape[0] > x.shape[1]
    x = (x.T if tall else x).contiguous() / (x.square().sum().sqrt() + 1e-7)
    for _ in range(steps):
        gram = x @ x.T.contiguous()
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x.T if tall else x


def two_norm(x):
    """By power iteration, from below."""
    v = torch.randn(x.shape[1], 1, generator=torch.Generator().manual_seed(0), dtype=torch.float64).to(x.device)
    for _ in range(60):
        v = x.T.contiguous() @ (x @ v)
        v /= v.norm()
    return float((x @ v).norm())


def off_by(got, want):
    """In the 2-norm."""
    return two_norm(got.double() - want) / two_norm(want)


@pytest.mark.parametrize("shape", [(128, 128), (300, 300), (777, 333), (130, 2000), (1000, 1000), (1000, 1500), (1100, 1300)])
def test_the_linear_term_is_exact(shape):
    """A rank-one update stays of rank one: X = s u v^T with s between 0.7 and 1.13, the polynomial's orbit from 1. Its linear
    term a X is exact to 2^-22 (both planes of X, and what fp16 rounds off the diagonal of B). What is left turns u: the
    roundings E of A's entries by (b + c s^2) E u and those of B's others by (b s^2 + c s^4) E u, each of them, for entries
    of normal u, ROUNDING sqrt(3 / m) in size, over the next s: 5.5, 1.6, 6.1, 1.7 and 6.1 times that in the five steps,
    10.5 together. X's own roundings are averaged over columns too, the one of the last iterate but one (a s / s' = 5.4
    times ROUNDING sqrt(3 / m)) is as large as a step's: all within three times the 10.5. At 128 rows that is 0.10 %, at
    1000 0.036 %. With the rounded diagonal, a itself would be off by up to 2^-12 in every step: 0.2 % at any size."""
    update = outer(1, *shape)
    bound = 3 * 10.5 * ROUNDING * math.sqrt(3 / min(shape))
    assert off_by(mpi.orthogonalize(update, dtype=torch.float32, precise=False), exact_there(update)) <= bound


@pytest.mark.parametrize("shape", [(40, 320, 320), (9, 1024, 1024), (6, 1090, 1090), (3, 2240, 2240)])
def test_the_linear_term_is_exact_whatever_the_tiles(shape):
    update = outer(2, *shape[1:], count=shape[0])
    bound = 3 * 10.5 * ROUNDING * math.sqrt(3 / min(shape[1:]))
    got = mpi.orthogonalize(update, dtype=torch.float32, precise=False)
    for k in (0, shape[0] // 2, shape[0] - 1):
        assert off_by(got[k], exact_there(update[k])) <= bound


@pytest.mark.parametrize("shape", [(2, 1000), (4, 300), (7, 2000), (8, 300), (16, 700), (33, 1000), (65, 300), (128, 512), (300, 300), (1000, 700)])
@pytest.mark.parametrize("kind", ["rank 1", "rank 2", "rank 8", "full", "decaying", "orthogonal"])
def test_the_documented_accuracy(shape, kind):
    """What orthogonalize's documentation says of precise=False."""
    gen = torch.Generator().manual_seed(3)
    normal = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    rows, cols = shape
    if kind.startswith("rank"):
        rank = int(kind[5:])
        update = normal(rows, rank) @ normal(rank, cols)
    elif kind == "full":
        update = normal(rows, cols)
    elif kind == "decaying":
        update = normal(rows, rows) @ (normal(rows, cols) / torch.arange(1, rows + 1).unsqueeze(1))
    else:
        q = torch.linalg.qr(normal(max(shape), min(shape)))[0]
        update = (q if rows > cols else q.T).contiguous()
    update = update.cuda()
    want = exact_there(update)
    got = mpi.orthogonalize(update, dtype=torch.float32, precise=False)
    assert float((got.double() - want).norm() / want.norm()) <= (0.003 if min(shape) >= 8 else 0.006)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_small_matrix_is_as_exact_among_larger_ones(dtype):
    """With products of single operands for the larger ones, a small one takes the same step as alone, bit for bit."""
    shapes = [(64, 256), (300, 200), (20, 30), (65, 64), (128, 64), (64, 257), (2, 2)]
    small = [s for s in shapes if min(s) <= 64 and max(s) <= 256]
    make = lambda some: [torch.nn.Parameter(torch.zeros(s, dtype=dtype, device="cuda")) for s in some]  # noqa: E731
    together, alone = make(shapes), make(small)
    for params in (together, alone):
        for p in params:
            gen = torch.Generator().manual_seed(1000 * p.shape[0] + p.shape[1])
            p.grad = torch.randn(*p.shape, generator=gen).to(dtype).cuda()
    mpi.Muon(together, precise=False).step()
    for p in alone:
        mpi.Muon([p], precise=False).step()
    for q in alone:
        p, = [p for p in together if p.shape == q.shape]
        assert torch.equal(p, q), p.shape
    for p in together:
        want = -0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * exact_there(p.grad)
        off = float((p.detach().double() - want).norm() / want.norm())
        assert off <= (1e-5 if tuple(p.shape) in small else 0.003) + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("shape", [(300, 300), (70, 1000), (1000, 500)])
def test_a_float16_result_is_as_exact_as_its_type(shape):
    """The split products' 1e-5 (1e-6 measured) and half a step of float16 in every entry, whose subnormal ones are off by
    half of 2^-24 at most."""
    update = torch.randn(*shape, generator=torch.Generator().manual_seed(4)).cuda()
    for u in (update.half(), update):
        want = exact_there(u)
        got = mpi.orthogonalize(u, dtype=torch.float16)
        assert got.dtype == torch.float16
        off = float((got.double() - want).norm())
        assert off <= (1e-5 + 2.0 ** -11) * float(want.norm()) + 2.0 ** -25 * math.sqrt(want.numel())
    assert torch.equal(got, mpi.orthogonalize(update, dtype=torch.float16, precise=True))


def test_a_mixed_list_captured_and_replayed():
    """Small matrices and larger ones of one 16-bit list: their launches go into the graph together. Four replays with new
    gradients against the same steps taken eagerly."""
    shapes = [(64, 256), (300, 200), (20, 30), (128, 64), (64, 300)]
    make = lambda: [torch.nn.Parameter(torch.ones(s, dtype=torch.bfloat16, device="cuda")) for s in shapes]  # noqa: E731
    captured, eager = make(), make()
    first, second = mpi.Muon(captured, weight_decay=0.1), mpi.Muon(eager, weight_decay=0.1)

    def fill(seed):
        for k, (p, q) in enumerate(zip(captured, eager)):
            new = torch.randn(*p.shape, generator=torch.Generator().manual_seed(10 * seed + k)).bfloat16().cuda()
            p.grad.copy_(new)
            q.grad.copy_(new)

    for p in captured + eager:
        p.grad = torch.zeros_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        fill(0)
        first.step(), second.step()
        with torch.cuda.graph(graph, stream=side):
            first.step()
    torch.cuda.synchronize()
    for seed in range(1, 5):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        second.step()
        torch.cuda.synchronize()
        for p, q in zip(captured, eager):
            assert torch.equal(p, q) and torch.equal(first.state[p]["momentum_buffer"], second.state[q]["momentum_buffer"])
