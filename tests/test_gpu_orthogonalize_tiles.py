"""GPU tests of every tile that the products of orthogonalize and Muon are cut
into, against the definition in 64 bits. test_step_host_on_cpu.py holds which
shapes take which."""
import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi
from test_gpu_orthogonalize_accuracy import exact_there
from test_step_host_on_cpu import TILES

pytestmark = pytest.mark.gpu

# The norm of the difference over that of the result: what the documentation states for products of single operands; with
# split ones some 2^-22 for each operand and float32 sums of at most 4096 products, 2^-24 sqrt(4096) = 4e-6, in all 1e-5.
BOUND = {False: 0.003, True: 1e-5}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def update_of(shape, seed):
    """Some strong directions over noise."""
    gen = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    return normal(shape[0], shape[1], 8) @ normal(shape[0], 8, shape[2]) + 0.3 * normal(*shape)


def off_by(got, want):
    return float((got.double() - want).norm() / want.norm())


def worst_entry(got, want):
    """The largest difference over the size of the result's entries: a tile in the wrong place is off by about 1."""
    return float((got.double() - want).abs().max() / want.square().mean().sqrt())


@pytest.mark.parametrize("shape, precise", TILES)
def test_tiles(shape, precise):
    count, rows, cols = shape
    update = update_of(shape, 1)
    results = {}
    for steps in (1, 2, 5):
        got = mpi.orthogonalize(update, steps=steps, dtype=torch.float32, precise=precise)
        tall = mpi.orthogonalize(update.mT, steps=steps, dtype=torch.float32, precise=precise)
        for k in {0, count // 2, count - 1}:
            want = exact_there(update[k], steps=steps)
            for x in (got[k], tall[k].T):
                assert off_by(x, want) <= BOUND[precise], (steps, k)
                # entries are off alike: eight times the mean size covers the largest of the some 10^7 there are, 5.3 times
                # for normal ones, and what is not independent
                assert worst_entry(x, want) <= 8 * BOUND[precise], (steps, k)
        results[steps] = got
    # 16-bit results, the same products
    for dtype in (torch.bfloat16, torch.float16):
        got = mpi.orthogonalize(update, dtype=dtype, precise=precise)
        assert torch.equal(got, results[5].to(dtype))


@pytest.mark.parametrize("shape, precise", TILES)
def test_tiles_under_muon(shape, precise):
    """A list of alike matrices takes the tiles of the batch; the new weights from the old ones and the momentum."""
    count, rows, cols = shape
    make = lambda seed: list(update_of(shape, seed).unbind(0))  # noqa: E731
    params = [torch.nn.Parameter(w.clone()) for w in make(2)]
    opt = mpi.Muon(params, lr=0.5, momentum=0.9, weight_decay=0.1, precise=precise, adjust="rms")
    momentum = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    for step in range(2):
        before = [p.detach().double() for p in params]
        for k, (p, g) in enumerate(zip(params, make(3 + step))):
            p.grad = g.clone()
            momentum[k] = 0.9 * momentum[k] + g.double()
        opt.step()
        for k in {0, count // 2, count - 1}:
            moved = 0.5 * 0.2 * max(rows, cols) ** 0.5 * exact_there(params[k].grad.double() + 0.9 * momentum[k])
            want = before[k] * (1 - 0.5 * 0.1) - moved
            off = params[k].detach().double() - want
            assert float(off.norm()) <= BOUND[precise] * float(moved.norm()) + 2.0 ** -22 * float(want.norm())


@pytest.mark.parametrize("precise", [False, True])
def test_a_list_of_unlike_matrices(precise):
    shapes = [(2220, 2400), (1000, 2731), (300, 500), (2240, 2240), (70, 4000), (700, 65), (64, 64), (1, 900)]
    params = [torch.nn.Parameter(torch.zeros(*s, device="cuda")) for s in shapes]
    for k, p in enumerate(params):
        p.grad = update_of((1,) + p.shape, 10 + k)[0].clone()
    mpi.Muon(params, lr=1.0, precise=precise, adjust="shape", nesterov=False).step()
    for p in params:
        want = -max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * exact_there(p.grad)
        assert off_by(p.detach(), want) <= (BOUND[precise] if min(p.shape) >= 8 else 2 * BOUND[precise]), p.shape
