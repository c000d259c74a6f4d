"""GPU tests of the step operators: embedding, embedding_gradient, sum_slices.

Tolerances. Products and sums are taken in 32 bits and rounded once to the
type. With u = 2^-24 (half a step of float32), a sum of n rows is off by at
most n u times the sum of the absolute values, the product with the scale by
u, and the rounding by half a step of the type (bf16 2^-8, fp16 2^-11): the
bounds below add these up. What is below fp16's smallest normal number 2^-14
is rounded to a multiple of 2^-24, half of which is added for that type."""
import numpy as np
import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def values(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def make_ids(seed, tokens, rows, kind, dtype):
    rng = np.random.default_rng(seed)
    if kind == "common":                      # a few ids hold most of the tokens
        ids = (rows * rng.random(tokens) ** 6).astype(np.int64)
    elif kind == "one":                       # all the same
        ids = np.full(tokens, rows - 1)
    elif kind == "outside":                   # nothing is in the table
        ids = rng.choice([-1, rows, rows + 7, -2 ** 31, 2 ** 31 - 1], tokens)
    elif kind == "padded":
        ids = np.where(rng.random(tokens) < 0.3, -1, rng.integers(0, rows, tokens))
    else:
        ids = rng.integers(0, rows, tokens)
    return torch.from_numpy(ids.astype(np.int32 if dtype == torch.int32 else np.int64)).cuda()


def lookup_64(ids, weight, scale):
    ids, weight = ids.cpu().long(), weight.double().cpu()
    inside = (ids >= 0) & (ids < weight.shape[0])
    out = torch.zeros(ids.shape + (weight.shape[1],), dtype=torch.float64)
    out[inside] = weight[ids[inside]] * float(np.float32(scale))
    return out


def sums_64(grad, ids, rows):
    """Sums, sums of absolute values, and counts, by row."""
    grad, ids = grad.double().cpu(), ids.cpu().long()
    inside = (ids >= 0) & (ids < rows)
    total = torch.zeros(rows, grad.shape[1], dtype=torch.float64)
    size = torch.zeros(rows, grad.shape[1], dtype=torch.float64)
    total.index_add_(0, ids[inside], grad[inside])
    size.index_add_(0, ids[inside], grad[inside].abs())
    return total, size, torch.bincount(ids[inside], minlength=rows)


def assert_sums(got, total, size, count, scale, dtype):
    slack = (count + 2).unsqueeze(1) * U * size * abs(scale)
    bound = slack + ((total * scale).abs() + slack) * HALF_STEP[dtype] + TINY[dtype]
    off = (got.double().cpu() - total * scale).abs()
    assert bool((off <= bound).all()), "off by up to %g of the bound" % float((off / bound.clamp_min(1e-300)).max())


SHAPES = [(1, 1, 1), (1, 50, 8), (2, 7, 3), (63, 9, 64), (64, 1000, 65), (257, 33, 1001), (1000, 4000, 129),
          (1024, 300, 256), (1025, 5000, 40), (5000, 777, 515), (8192, 8192, 16), (8193, 100, 24), (12288, 9000, 20), (12289, 300, 20), (20001, 70000, 33)]


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_lookup(shape, dtype):
    tokens, rows, width = shape
    weight = values(1, rows, width, dtype=dtype)
    for kind, id_type, scale in (("any", torch.int64, 1.0), ("padded", torch.int32, float(width) ** 0.5), ("outside", torch.int32, 2.0)):
        ids = make_ids(2, tokens, rows, kind, id_type)
        got = mpi.embedding(ids, weight, scale=scale)
        want = lookup_64(ids, weight, scale)
        assert got.dtype == dtype and got.shape == want.shape
        bound = want.abs() * (HALF_STEP[dtype] + 2 * U) + TINY[dtype]
        assert bool(((got.double().cpu() - want).abs() <= bound).all())


def test_lookup_shapes_and_strides():
    table = values(3, 40, 96)
    weight = table[5:30, 7:50]                                 # a slice of a larger table, misaligned rows
    ids = make_ids(4, 24, 25, "padded", torch.int64).reshape(2, 3, 4)
    want = lookup_64(ids, weight, 0.5).float()
    assert torch.equal(mpi.embedding(ids, weight, scale=0.5).cpu(), want)
    assert torch.equal(mpi.embedding(ids.transpose(0, 2), weight, scale=0.5).cpu(), want.transpose(0, 2))
    by_column = weight.t().contiguous().t()                    # columns not contiguous: copied
    assert torch.equal(mpi.embedding(ids, by_column, scale=0.5).cpu(), want)
    assert mpi.embedding(ids[:0], weight).shape == (0, 3, 4, 43)
    assert mpi.embedding(ids[0, 0, 0], weight).shape == (43,)
    assert torch.equal(mpi.embedding(ids, weight[:0]).cpu(), torch.zeros(2, 3, 4, 43))
    assert mpi.embedding(ids, weight[:, :0]).shape == (2, 3, 4, 0)
    one_row = table[:1].expand(25, 96)                         # rows that are no distance apart
    assert torch.equal(mpi.embedding(ids, one_row).cpu(), lookup_64(ids, one_row, 1.0).float())


def test_lookup_of_infinities_stays_in_their_rows():
    weight = torch.zeros(4, 16).cuda()
    weight[1] = float("inf")
    weight[2] = float("nan")
    out = mpi.embedding(torch.tensor([0, 1, -1, 2, 3]).cuda(), weight, scale=3.0).cpu()
    assert torch.equal(out[[0, 2, 4]], torch.zeros(3, 16))
    assert bool(torch.isinf(out[1]).all()) and bool(torch.isnan(out[3]).all())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(shape, dtype):
    tokens, rows, width = shape
    grad = values(5, tokens, width, dtype=dtype)
    for kind, id_type, scale in (("any", torch.int32, 1.0), ("common", torch.int64, 3.0), ("one", torch.int64, 1.0),
                                 ("padded", torch.int32, 0.25), ("outside", torch.int32, 1.0)):
        ids = make_ids(6, tokens, rows, kind, id_type)
        got = mpi.embedding_gradient(grad, ids, rows, scale=scale)
        assert got.dtype == dtype and got.shape == (rows, width)
        total, size, count = sums_64(grad, ids, rows)
        assert_sums(got, total, size, count, scale, dtype)
        empty = count == 0
        assert torch.equal(got.cpu()[empty], torch.zeros(int(empty.sum()), width, dtype=dtype))
        assert torch.equal(mpi.embedding_gradient(grad, ids, rows, scale=scale), got)     # the same bits again


def test_gradient_adds_in_the_order_of_the_tokens():
    """Up to a piece's length (64 tokens at least) a row's sum is the left fold over its tokens, bit for bit."""
    tokens, rows, width = 3000, 128, 37
    grad, ids = values(7, tokens, width), make_ids(8, tokens, rows, "any", torch.int64)
    assert int(torch.bincount(ids).max()) <= 64
    got = mpi.embedding_gradient(grad, ids, rows).cpu().numpy()
    want = np.zeros((rows, width), np.float32)
    for t, i in enumerate(ids.cpu().numpy()):
        want[i] = want[i] + grad[t].cpu().numpy()
    assert np.array_equal(got, want)


def test_gradient_of_padding_is_left_out_whatever_it_holds():
    ids = torch.tensor([0, -1, 2, 5, 2]).cuda()
    grad = torch.ones(5, 40).cuda()
    grad[1] = float("nan")
    grad[3] = float("inf")
    got = mpi.embedding_gradient(grad, ids, 4).cpu()
    assert torch.equal(got, torch.tensor([1.0, 0.0, 2.0, 0.0]).unsqueeze(1).expand(4, 40))
    grad[4] = float("inf")
    got = mpi.embedding_gradient(grad, ids, 4).cpu()
    assert bool(torch.isinf(got[2]).all()) and torch.equal(got[[0, 1, 3]], torch.tensor([[1.0], [0.0], [0.0]]).expand(3, 40))


def test_gradient_strides():
    ids = make_ids(9, 60, 20, "padded", torch.int64).reshape(5, 12)
    wide = values(10, 5, 12, 70)
    for grad in (wide[..., 3:36], wide[:, :, ::2], wide[:1, :1, :33].expand(5, 12, 33), wide.transpose(0, 1)[:, :, :33].transpose(0, 1)):
        got = mpi.embedding_gradient(grad, ids, 20)
        total, size, count = sums_64(grad.reshape(60, -1), ids.reshape(-1), 20)
        assert_sums(got, total, size, count, 1.0, torch.float32)
    assert torch.equal(mpi.embedding_gradient(wide[:0], ids[:0], 20).cpu(), torch.zeros(20, 70))
    assert torch.equal(mpi.embedding_gradient(wide[:0].half(), ids[:0], 3).cpu(), torch.zeros(3, 70).half())
    assert torch.equal(mpi.embedding_gradient(wide[:0, :, :1].half(), ids[:0], 1).cpu(), torch.zeros(1, 1).half())
    assert mpi.embedding_gradient(wide, ids, 0).shape == (0, 70)
    assert mpi.embedding_gradient(wide[..., :0], ids, 20).shape == (20, 0)


@pytest.mark.parametrize("tokens, ranks, rows, width, id_type", [
    (1, 1, 10, 5, torch.int64), (0, 3, 10, 5, torch.int32), (129, 4, 3000, 300, torch.int64), (700, 3, 90, 33, torch.int32),
    (3000, 8, 5021, 64, torch.int64), (5000, 16, 12, 9, torch.int32),
    (1536, 8, 400, 20, torch.int64)])
def test_sum_slices(tokens, ranks, rows, width, id_type):
    ids = torch.cat([make_ids(20 + r, tokens, rows, "common" if r % 2 else "padded", id_type) for r in range(ranks)])
    grad = values(11, tokens * ranks, width)
    total, size, count = sums_64(grad, ids, rows)
    got = mpi.sum_slices(mpi.IndexedSlices(grad, ids, (rows, width)))
    there = count > 0
    assert got.dense_shape == (rows, width) and got.indices.dtype == id_type
    assert torch.equal(got.indices.cpu().long(), torch.nonzero(there).reshape(-1))
    assert_sums(got.values, total[there], size[there], count[there], 1.0, torch.float32)


def test_sum_slices_of_other_types_and_shapes():
    ids = torch.tensor([3, 1, 3, 3]).cuda()
    for dtype in FLOATS:
        v = torch.arange(24.0).reshape(4, 2, 3).to(dtype).cuda()
        got = mpi.sum_slices(mpi.IndexedSlices(v, ids, (5, 2, 3)))
        assert got.indices.tolist() == [1, 3] and got.values.dtype == dtype
        assert torch.equal(got.values.cpu(), torch.stack([v[1], v[0] + v[2] + v[3]]).cpu())
    got = mpi.sum_slices(mpi.IndexedSlices(torch.arange(4.0).cuda(), ids, (5,)))
    assert got.values.tolist() == [1.0, 5.0]
    none = mpi.sum_slices(mpi.IndexedSlices(torch.ones(4, 2).cuda(), ids, (1, 2)))
    assert none.indices.numel() == 0 and none.values.shape == (0, 2)


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("dtype", FLOATS)
def test_autograd(dtype, sparse):
    ids = make_ids(12, 300, 50, "padded", torch.int64).reshape(3, 100)
    weight = values(13, 50, 72, dtype=dtype).requires_grad_(True)
    grad = values(14, 3, 100, 72, dtype=dtype)
    out = mpi.embedding(ids, weight, scale=1.5, sparse=sparse)
    out.backward(grad)
    assert weight.grad.is_sparse == sparse
    if sparse:
        # distinct and ascending (autograd does not keep the mark that says so)
        assert torch.equal(weight.grad._indices()[0].cpu(), torch.unique(ids[ids >= 0]).cpu())
    total, size, count = sums_64(grad.reshape(300, 72), ids.reshape(-1), 50)
    assert_sums(weight.grad.to_dense() if sparse else weight.grad, total, size, count, 1.5, dtype)
    # a second backward pass adds
    first = weight.grad.to_dense().clone() if sparse else weight.grad.clone()
    mpi.embedding(ids, weight, scale=1.5, sparse=sparse).backward(grad)
    second = weight.grad.to_dense() if sparse else weight.grad
    assert torch.equal(second, first + first)


def test_gradient_against_differences():
    """The lookup is linear and these numbers are small powers of two, so differences are exact."""
    ids = torch.tensor([[2, 0, 2], [-1, 1, 2]]).cuda()
    weight = torch.tensor([[1.0, 0.5], [2.0, -1.0], [0.25, 4.0]]).cuda()
    grad = torch.tensor([[[1.0, 2.0], [0.5, 1.0], [4.0, -1.0]], [[8.0, 8.0], [2.0, 0.25], [-2.0, 1.0]]]).cuda()
    leaf = weight.clone().requires_grad_(True)
    mpi.embedding(ids, leaf, scale=2.0).backward(grad)
    for i in range(3):
        for j in range(2):
            step = torch.zeros_like(weight)
            step[i, j] = 0.5
            up, down = mpi.embedding(ids, weight + step, scale=2.0), mpi.embedding(ids, weight - step, scale=2.0)
            assert float((grad * (up - down)).sum()) == float(leaf.grad[i, j])


def test_no_gradient_where_none_is_wanted():
    ids = torch.tensor([0, 1]).cuda()
    weight = values(15, 3, 4).requires_grad_(True)
    with torch.no_grad():
        assert not mpi.embedding(ids, weight).requires_grad
    assert not mpi.embedding(ids, weight.detach()).requires_grad
    out = (mpi.embedding(ids, weight) * 2).sum()               # an expanded gradient
    out.backward()
    assert torch.equal(weight.grad.cpu(), torch.tensor([[2.0], [2.0], [0.0]]).expand(3, 4))


def test_offsets_beyond_32_bits():
    """A table, a result and a gradient of more than 2^32 bytes and 2^31 elements."""
    rows, width = 530_000, 4100
    table = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    picked = [0, 1, 255_000, 523_776, rows - 1]
    marks = values(16, len(picked), width, dtype=torch.bfloat16)
    for k, r in enumerate(picked):
        table[r] = marks[k]
    got = mpi.embedding(torch.tensor(picked).cuda(), table)
    assert torch.equal(got, marks)
    del table
    # gradient rows far out: positions and rows both
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    ids[picked] = torch.tensor(picked, dtype=torch.int32).cuda()
    grad = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    for k, r in enumerate(picked):
        grad[r] = marks[k]
    dense = mpi.embedding_gradient(grad, ids, rows)
    assert torch.equal(dense[picked], marks)
    assert int(dense[2:1000].count_nonzero()) == 0 and int(dense[-1000:-1].count_nonzero()) == 0


def test_another_stream():
    stream = torch.cuda.Stream()
    ids = make_ids(17, 5000, 300, "common", torch.int64)
    weight, grad = values(18, 300, 128), values(19, 5000, 128)
    want, want_grad = mpi.embedding(ids, weight), mpi.embedding_gradient(grad, ids, 300)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(stream):
            got, got_grad = mpi.embedding(ids, weight), mpi.embedding_gradient(grad, ids, 300)
        here = mpi.embedding_gradient(grad, ids, 300)          # both streams at once
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(got_grad, want_grad) and torch.equal(here, want_grad)


@pytest.mark.parametrize("tokens", [700, 20000])
def test_captured_into_graphs_and_replayed(tokens):
    """Two captured graphs with workspaces of their own, replayed in turn with new inputs, eager work between them."""
    rows, width = 900, 96
    ids = torch.empty(tokens, dtype=torch.int64, device="cuda")
    weight, grad = values(21, rows, width), torch.empty(tokens, width, device="cuda")
    ids.copy_(make_ids(22, tokens, rows, "any", torch.int64))
    grad.copy_(values(23, tokens, width))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            mpi.embedding(ids, weight), mpi.embedding_gradient(grad, ids, rows)     # warm-up
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = mpi.embedding(ids, weight, scale=2.0)
                dense = mpi.embedding_gradient(grad, ids, rows, scale=2.0)
            graphs.append((g, out, dense))
    torch.cuda.synchronize()
    for k in range(4):
        ids.copy_(make_ids(30 + k, tokens, rows, ("common", "padded", "one", "any")[k], torch.int64))
        grad.copy_(values(40 + k, tokens, width))
        want, want_grad = mpi.embedding(ids, weight, scale=2.0), mpi.embedding_gradient(grad, ids, rows, scale=2.0)
        torch.cuda.synchronize()
        for g, out, dense in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(dense, want_grad)


def test_refusals():
    ids, weight = torch.zeros(3, dtype=torch.int64).cuda(), torch.zeros(4, 5).cuda()
    for call in (lambda: mpi.embedding(ids.float(), weight), lambda: mpi.embedding(ids.short(), weight),
                 lambda: mpi.embedding(ids, weight.double()), lambda: mpi.embedding(ids, weight[0]),
                 lambda: mpi.embedding(ids.cpu(), weight), lambda: mpi.embedding(ids, weight.cpu()),
                 lambda: mpi.embedding_gradient(weight, ids, 7), lambda: mpi.embedding_gradient(weight[:3], ids, -1),
                 lambda: mpi.sum_slices(mpi.IndexedSlices(weight, ids, (9, 5))),
                 lambda: mpi.sum_slices(mpi.IndexedSlices(weight[:3], ids, (9, 6))),
                 lambda: mpi.sum_slices(mpi.IndexedSlices(weight[:3], ids)),
                 lambda: mpi.sum_slices(mpi.IndexedSlices(weight[:3], ids, (-1, 5)))):
        with pytest.raises(mpi.InvalidArgumentError):
            call()


@pytest.mark.parametrize("ranks", [1, 4])
def test_sparse_gradients_through_the_exchange(ranks):
    """What a data-parallel step does with an embedding: every rank's sparse gradient, gathered and averaged by
    DistributedOptimizer, summed by index, applied; against the same steps in 64 bits."""
    rows, width, tokens, lr = 60, 24, 200, 0.5
    start = values(50, rows, width)
    weights = [start.clone().requires_grad_(True) for _ in range(ranks)]
    exact = start.double().cpu()
    opts = [mpi.DistributedOptimizer(torch.optim.SGD([w], lr=lr)) for w in weights]
    bound = torch.zeros(rows, width, dtype=torch.float64)
    with mpi.Session(size=ranks) as session:
        for step in range(3):
            pairs, mean = [], torch.zeros(rows, width, dtype=torch.float64)
            for r in range(ranks):
                ids = make_ids(100 * step + r, tokens, rows, "common" if r % 2 else "padded", torch.int64)
                grad = values(100 * step + r + 50, tokens, width)
                with session.as_rank(r):
                    opts[r].zero_grad(set_to_none=True)
                    mpi.embedding(ids, weights[r], scale=2.0, sparse=True).backward(grad)
                    pairs.append(opts[r].compute_gradients())
                total, size, count = sums_64(grad, ids, rows)
                mean += 2.0 * total / ranks
                bound += lr * 2.0 * size / ranks * (count + 2 + ranks + 3).unsqueeze(1) * U
            if ranks > 1:
                session.run([g for p in pairs for g, _ in p])
            for r in range(ranks):
                with session.as_rank(r):
                    opts[r].apply_gradients(pairs[r])
                    assert weights[r].grad.is_sparse and weights[r].grad.is_coalesced()
            exact -= lr * mean
            bound += exact.abs() * 2 * U
    for w in weights:
        assert torch.equal(w, weights[0])
    assert bool(((weights[0].detach().double().cpu() - exact).abs() <= bound).all())


def test_gradient_of_the_gradient():
    """A penalty on the gradient of what the lookup feeds: the gradient is linear, its own gradient the lookup."""
    ids = make_ids(60, 40, 12, "padded", torch.int64)
    weight = values(61, 12, 10).requires_grad_(True)
    mix = values(62, 40, 10).requires_grad_(True)
    out = mpi.embedding(ids, weight, scale=2.0)
    first, = torch.autograd.grad((out * mix).sum(), weight, create_graph=True)
    first.square().sum().backward()
    mirror_w, mirror_m = weight.detach().double().cpu().requires_grad_(True), mix.detach().double().cpu().requires_grad_(True)
    inside = ids.cpu() >= 0
    picked = torch.zeros(40, 10, dtype=torch.float64).index_put((inside,), 2.0 * mirror_w[ids.cpu()[inside]])
    want, = torch.autograd.grad((picked * mirror_m).sum(), mirror_w, create_graph=True)
    want.square().sum().backward()
    assert torch.allclose(mix.grad.double().cpu(), mirror_m.grad, rtol=40 * U, atol=40 * U * float(mirror_m.grad.abs().max()))


def test_the_gradient_called_by_name_is_differentiable():
    """embedding_gradient is linear in grad: the gradient of <embedding_gradient(g), m> is the lookup of m."""
    ids = make_ids(70, 50, 9, "padded", torch.int32)
    grad = values(71, 50, 12).requires_grad_(True)
    mix = values(72, 9, 12)
    (mpi.embedding_gradient(grad, ids, 9, scale=0.5) * mix).sum().backward()
    assert torch.equal(grad.grad, mpi.embedding(ids, mix, scale=0.5))
    with torch.no_grad():
        assert not mpi.embedding_gradient(grad, ids, 9).requires_grad
