"""GPU tests of orthogonalize and Muon against the definition in 64 bits.

Tolerances. The distance is the 2-norm of the difference over that of the
result. A product of n terms in fp16 operands (relative rounding at most
2^-11) with float32 sums: the linear term of a step is exact to 2^-22, and the
rounding of X, A and B inside (b A + c A A) X moves X by at most
(3 |b| + 7 |c|) 2^-11 per step, relative to |X|, if all roundings pull one way:
28.6 2^-11 = 0.014, times five steps 0.07 (the polynomial's slope is below 1 in
size where the singular values have arrived). That is the bound for a matrix of
one row, where one rounding of A and one of B hit every entry. With m rows each
entry of (b A + c A A) X sums m products with roundings of their own, which are
independent: together the 1 / sqrt(m)-th part. From m = 291 on this is below
0.0041, where the roundings of the entries of X themselves (not averaged over m:
mean size 2^-11 / sqrt(12) each, 1 / 3.5 of the most, terms' root of the sum of
squares at most 13: 13 2^-11 / 3.5 sqrt(5)) stay. With split operands 2^-11 becomes
2^-22, plus float32 sums over at most 4096 terms (2^-24 sqrt(4096) = 4e-6):
1e-5. A 16-bit result adds half a step of its type."""
import math

import pytest
import torch

import mpi_collectives as mpi
from mpi_collectives import step_abi

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
SPLIT = 1e-5
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    step_abi.lib()


def exact(update, steps=5, coefficients=(A, B, C), eps=1e-7):
    """On the CPU, in 64 bits."""
    x = update.detach().cpu().double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    triples = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    for a, b, c in triples:
        if x.shape[-2] <= x.shape[-1]:
            gram = x @ x.mT
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        else:
            gram = x.mT @ x
            x = a * x + x @ (b * gram + c * (gram @ gram))
    return x


def distance(got, want):
    want = want.double().cpu()
    return float((got.detach().double().cpu() - want).norm() / want.norm())


def half(shape):
    return max(0.0041, 0.07 / math.sqrt(min(shape[-2:])))


def bound(dtype, precise, shape=(1, 1)):
    return (SPLIT if precise else half(shape)) + HALF_STEP[dtype]


def gradient(seed, *shape, rank=8, noise=0.3, size=1e-4, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    k = min(rank, shape[-1], shape[-2])
    low = torch.randn(*shape[:-1], k, generator=gen) @ torch.randn(*shape[:-2], k, shape[-1], generator=gen)
    return (size * (low + noise * torch.randn(*shape, generator=gen))).to(dtype).cuda()


SHAPES = [(1, 1), (1, 100), (64, 256), (250, 64), (33, 129), (64, 257), (100, 1), (3, 5), (64, 64), (64, 128), (65, 63), (128, 128), (129, 500), (200, 130), (500, 129),
          (1000, 1), (256, 1024), (777, 333), (1000, 1500), (2000, 130)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_orthogonalize(shape, dtype):
    size = 1e-2 if dtype == torch.float16 else 1e-4
    update = gradient(1, *shape, size=size, dtype=dtype)
    want = exact(update)
    for precise in (False, True):
        got = mpi.orthogonalize(update, precise=precise)
        assert got.dtype == dtype and got.shape == update.shape
        assert distance(got, want) <= bound(dtype, precise, shape), precise
        assert torch.equal(mpi.orthogonalize(update, precise=precise), got)      # the same bits again
    got = mpi.orthogonalize(update, dtype=torch.float32)
    assert got.dtype == torch.float32 and distance(got, want) <= bound(torch.float32, True)


@pytest.mark.parametrize("shape, kind", [((64, 256), "rank 1"), ((300, 300), "rank 1"), ((512, 512), "noise"),
                                         ((400, 900), "decaying"), ((1024, 2048), "noise")])
def test_whatever_the_spectrum(shape, kind):
    """Roundings must not grow in directions that the update hardly has."""
    if kind == "rank 1":
        update = gradient(2, *shape, rank=1, noise=0.0)
    elif kind == "noise":
        update = gradient(3, *shape, rank=1, noise=1e3, size=1.0)
    else:
        gen = torch.Generator().manual_seed(4)
        left, right = torch.randn(shape[0], shape[0], generator=gen), torch.randn(shape[0], shape[1], generator=gen)
        update = (left @ (right / torch.arange(1, shape[0] + 1).unsqueeze(1))).cuda()
    want = exact(update)
    assert distance(mpi.orthogonalize(update, precise=False), want) <= half(shape)
    # hi + lo / 2048 holds 22 bits: the first iterate is rounded by 2^-22 at most, which grows by a^5 = 485 where nothing else is
    assert distance(mpi.orthogonalize(update), want) <= SPLIT + 485 * 2.0 ** -22
    for shift in (2.0 ** -60, 2.0 ** 50):                            # exact: the same update at other sizes
        scaled = update * shift
        assert distance(mpi.orthogonalize(scaled, eps=0.0), exact(scaled, eps=0.0)) <= SPLIT + 485 * 2.0 ** -22


def test_batches():
    update = gradient(5, 3, 2, 70, 130)
    got = mpi.orthogonalize(update)
    for i in range(3):
        for j in range(2):
            assert torch.equal(got[i, j], mpi.orthogonalize(update[i, j]))
    many = gradient(6, 300, 20, 33)
    assert distance(mpi.orthogonalize(many), exact(many)) <= SPLIT
    assert mpi.orthogonalize(update[:0]).shape == (0, 2, 70, 130)
    assert mpi.orthogonalize(update[..., :0]).shape == (3, 2, 70, 0)
    assert mpi.orthogonalize(update[..., :0, :]).shape == (3, 2, 0, 130)
    # strides other than the contiguous ones
    for view in (update.mT, update[..., 1::2, 3:], update.permute(1, 3, 0, 2)):
        assert torch.equal(mpi.orthogonalize(view), mpi.orthogonalize(view.contiguous()))


def test_steps_and_coefficients():
    update = gradient(7, 90, 200)
    for steps in (1, 2, 3):
        assert distance(mpi.orthogonalize(update, steps=steps), exact(update, steps=steps)) <= SPLIT
        assert distance(mpi.orthogonalize(update, steps=steps, precise=False), exact(update, steps=steps)) <= half(update.shape)
    cubic = (1.5, -0.5, 0.0)
    assert distance(mpi.orthogonalize(update, steps=20, coefficients=cubic), exact(update, 20, cubic)) <= 4 * SPLIT
    schedule = [(3.4, -4.7, 2.0), (2.8, -3.0, 1.2), (1.875, -1.25, 0.375)]
    assert distance(mpi.orthogonalize(update, steps=3, coefficients=schedule), exact(update, 3, schedule)) <= SPLIT
    x = mpi.orthogonalize(gradient(8, 100, 300), steps=20, coefficients=cubic).double()
    sigma = torch.linalg.svdvals(x.cpu())
    assert float((sigma - 1).abs().max()) < 1e-4                     # it is orthogonal in the end


def test_zeros_infinities_and_nan():
    assert int(mpi.orthogonalize(torch.zeros(70, 90).cuda()).count_nonzero()) == 0
    assert int(mpi.orthogonalize(torch.zeros(70, 90).cuda(), precise=False).count_nonzero()) == 0
    batch = gradient(9, 3, 70, 90)
    clean = mpi.orthogonalize(batch)
    batch[1, 5, 5] = float("nan")
    got = mpi.orthogonalize(batch)
    assert bool(torch.isnan(got[1]).all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])       # its neighbours do not see it
    batch[1, 5, 5] = float("inf")
    assert bool(torch.isnan(mpi.orthogonalize(batch)[1]).any())


def muon_64(w, m, g, lr, momentum, nesterov, decay, adjust):
    w, m, g = w.double().cpu(), m.double().cpu(), g.double().cpu()
    m = momentum * m + g
    o = exact(g + momentum * m if nesterov else m)
    rows, cols = w.shape
    s = math.sqrt(max(1.0, rows / cols)) if adjust == "shape" else 0.2 * math.sqrt(max(rows, cols))
    return w * (1 - lr * decay) - lr * s * o, m, lr * s * o


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("options", [dict(), dict(nesterov=False, weight_decay=0.1), dict(adjust="rms", lr=0.003, momentum=0.9),
                                     dict(precise=False), dict(precise=True, momentum=0.0)])
def test_muon(dtype, options):
    shapes = [(64, 64), (130, 70), (70, 130), (130, 70), (1, 40), (300, 300), (257, 64), (64, 257)]
    params = [torch.nn.Parameter((0.05 * torch.randn(*s, generator=torch.Generator().manual_seed(k))).to(dtype).cuda()) for k, s in enumerate(shapes)]
    params.append(torch.nn.Parameter(torch.ones(2, 2, dtype=dtype).cuda()))      # never gets a gradient
    opt = mpi.Muon(params, **options)
    o = {**dict(lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="shape"), **options}
    precise = options.get("precise", dtype == torch.float32)
    for step in range(3):
        before = []
        for k, p in enumerate(params[:-1]):
            p.grad = gradient(100 * step + k, *p.shape, size=1e-2, dtype=dtype)
            m = opt.state[p].get("momentum_buffer", torch.zeros(p.shape)).clone()
            before.append((p.detach().clone(), m, p.grad))
        opt.step()
        for p, (w, m, g) in zip(params, before):
            want, buffer, moved = muon_64(w, m, g, o["lr"], o["momentum"], o["nesterov"], o["weight_decay"], o["adjust"])
            got = opt.state[p]["momentum_buffer"]
            assert got.dtype == torch.float32
            assert bool(((got.double().cpu() - buffer).abs() <= (buffer.abs() + m.double().cpu().abs()) * 2.0 ** -23).all())
            off = float((p.detach().double().cpu() - want).norm())
            # the step's own error, a few roundings in 32 bits, the rounding to the type
            assert off <= (SPLIT if precise else half(w.shape)) * float(moved.norm()) + (2.0 ** -22 + HALF_STEP[dtype]) * float(want.norm())
    assert torch.equal(params[-1], torch.ones(2, 2, dtype=dtype).cuda())


def test_muon_with_many_matrices_of_many_shapes():
    """More matrices than one launch carries; as one list and one by one they differ by the split products' roundings only."""
    shapes = [(8 + 3 * (k % 30), 16 + 5 * (k % 17)) for k in range(130)]
    make = lambda: [torch.nn.Parameter(gradient(k, *s, size=1.0)) for k, s in enumerate(shapes)]  # noqa: E731
    together, apart = make(), make()
    for p, q in zip(together, apart):
        p.grad = q.grad = gradient(int(p.numel()), *p.shape)
    start = [p.detach().clone() for p in together]
    mpi.Muon(together).step()
    for q in apart:
        mpi.Muon([q]).step()
    for p, q, w in zip(together, apart, start):
        p, q = p.detach(), q.detach()
        assert float((p - q).norm()) <= 2 * SPLIT * float((q - w).norm()) + 2.0 ** -22 * float(q.norm())


def test_muon_strides_state_and_groups():
    make = lambda: torch.nn.Parameter(torch.randn(40, 60, generator=torch.Generator().manual_seed(3)).cuda().t())  # noqa: E731
    p, q = make(), torch.nn.Parameter(make().detach().contiguous())
    assert not p.is_contiguous()
    a, b = mpi.Muon([{"params": [p], "lr": 0.1}]), mpi.Muon([q], lr=0.1)
    for k in range(2):
        q.grad = gradient(k, 60, 40)
        p.grad = q.grad.t().contiguous().t()
        a.step(), b.step()
        assert torch.equal(p, q) and not p.is_contiguous()
    # a saved and loaded state goes on with the same bits, in 16 bits too
    w = torch.nn.Parameter(torch.randn(50, 50, generator=torch.Generator().manual_seed(4)).bfloat16().cuda())
    c = mpi.Muon([w], lr=0.1)
    w.grad = gradient(5, 50, 50, dtype=torch.bfloat16)
    c.step()
    v = torch.nn.Parameter(w.detach().clone())
    d = mpi.Muon([v], lr=0.7)
    d.load_state_dict(c.state_dict())
    assert d.state[v]["momentum_buffer"].dtype == torch.float32 and d.param_groups[0]["lr"] == 0.1
    v.grad = w.grad = gradient(6, 50, 50, dtype=torch.bfloat16)
    c.step(), d.step()
    assert torch.equal(v, w) and torch.equal(c.state[w]["momentum_buffer"], d.state[v]["momentum_buffer"])


def test_streams_and_graphs():
    update = gradient(10, 200, 300)
    w = torch.nn.Parameter(torch.zeros(200, 300).cuda())
    w.grad = torch.zeros_like(w)
    opt = mpi.Muon([w], lr=0.5)
    static = torch.zeros_like(update)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        opt.step()
        for _ in range(2):
            mpi.orthogonalize(static)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = mpi.orthogonalize(static)
                opt.step()
            graphs.append((g, out))
    torch.cuda.synchronize()
    v = torch.nn.Parameter(w.detach().clone())
    eager = mpi.Muon([v], lr=0.5)
    eager.load_state_dict(opt.state_dict())
    for k in range(4):
        new = gradient(20 + k, 200, 300)
        static.copy_(new)
        for g, out in graphs:
            w.grad.copy_(new * (k + 1))
            v.grad = new * (k + 1)
            eager.step()
            want = mpi.orthogonalize(new)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(w, v)
    # two streams at once
    want = mpi.orthogonalize(update)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            there = mpi.orthogonalize(update)
        here = mpi.orthogonalize(update)
        torch.cuda.synchronize()
        assert torch.equal(there, want) and torch.equal(here, want)


def test_refusals():
    u = torch.zeros(4, 4).cuda()
    vector, cube = torch.nn.Parameter(torch.zeros(4).cuda()), torch.nn.Parameter(torch.zeros(2, 4, 4).cuda())
    for call in (lambda: mpi.orthogonalize(u[0]), lambda: mpi.orthogonalize(u.long()), lambda: mpi.orthogonalize(u.cpu()),
                 lambda: mpi.orthogonalize(u, dtype=torch.float64), lambda: mpi.orthogonalize(u, steps=0),
                 lambda: mpi.orthogonalize(u, steps=65), lambda: mpi.orthogonalize(u, coefficients=(1.0, 2.0)),
                 lambda: mpi.orthogonalize(u, steps=3, coefficients=[(1.0, 2.0, 3.0)] * 2),
                 lambda: mpi.Muon([vector]), lambda: mpi.Muon([cube]), lambda: mpi.Muon([torch.nn.Parameter(u.double())]),
                 lambda: mpi.Muon([torch.nn.Parameter(u)], adjust="none"), lambda: mpi.Muon([torch.nn.Parameter(u)], steps=65)):
        with pytest.raises(mpi.InvalidArgumentError):
            call()
    w = torch.nn.Parameter(u.clone())
    w.grad = torch.zeros(4, 4).to_sparse().cuda()
    with pytest.raises(mpi.InvalidArgumentError):
        mpi.Muon([w]).step()
    on_cpu = torch.nn.Parameter(torch.zeros(4, 4))
    on_cpu.grad = torch.zeros(4, 4)
    with pytest.raises(mpi.InvalidArgumentError):
        mpi.Muon([on_cpu]).step()


@pytest.mark.parametrize("fusion", [False, True])
def test_a_training_step_through_the_exchange(fusion):
    """Embedding with a sparse gradient, two matrices with Muon, gradients exchanged by DistributedOptimizer, three virtual
    ranks: the replicas stay identical and follow the same steps in 64 bits."""
    ranks, rows, width, classes, tokens = 3, 50, 48, 20, 64
    start = [torch.randn(s, generator=torch.Generator().manual_seed(k)).mul_(0.2) for k, s in enumerate([(rows, width), (width, 96), (96, classes)])]
    nets = [[t.clone().cuda().requires_grad_(True) for t in start] for _ in range(ranks)]
    nets = [[net[0], torch.nn.Parameter(net[1].detach()), torch.nn.Parameter(net[2].detach())] for net in nets]
    opts = [(mpi.DistributedOptimizer(torch.optim.SGD(net[:1], lr=0.5)),
             mpi.DistributedOptimizer(mpi.Muon(net[1:], lr=0.05, weight_decay=0.1), fusion=fusion)) for net in nets]
    mirror = [t.double().requires_grad_(True) for t in start]
    buffers = [torch.zeros_like(t) for t in mirror[1:]]

    def loss_of(ids, target, table, first, second, lookup):
        hidden = torch.tanh(lookup(ids, table) @ first)
        return torch.nn.functional.cross_entropy(hidden @ second, target)

    with mpi.Session(size=ranks) as session:
        for step in range(3):
            pairs = []
            for t in mirror:
                t.grad = None
            for r in range(ranks):
                gen = torch.Generator().manual_seed(10 * step + r)
                ids, target = torch.randint(0, rows, (tokens,), generator=gen), torch.randint(0, classes, (tokens,), generator=gen)
                with session.as_rank(r):
                    for o in opts[r]:
                        o.zero_grad(set_to_none=True)
                    loss_of(ids.cuda(), target.cuda(), *nets[r], lambda i, t: mpi.embedding(i, t, scale=2.0, sparse=True)).backward()
                    pairs.append([o.compute_gradients() for o in opts[r]])
                (loss_of(ids, target, *mirror, lambda i, t: 2.0 * t[i]) / ranks).backward()
            if not fusion:
                session.run([[g for g, _ in p] for both in pairs for p in both])
            else:
                session.run()
            for r in range(ranks):
                with session.as_rank(r):
                    for o, p in zip(opts[r], pairs[r]):
                        o.apply_gradients(p)
            with torch.no_grad():
                mirror[0] -= 0.5 * mirror[0].grad
                for k in (1, 2):
                    mirror[k].copy_(muon_64(mirror[k], buffers[k - 1], mirror[k].grad, 0.05, 0.95, True, 0.1, "shape")[0])
                    buffers[k - 1] = 0.95 * buffers[k - 1] + mirror[k].grad
    for net in nets[1:]:
        for p, q in zip(net, nets[0]):
            assert torch.equal(p, q)
    for p, want in zip(nets[0], mirror):
        # float32 gradients are some 2^-20 off, and a step turns and stretches them by at most 485 (a^5); three steps
        assert distance(p, want.detach()) <= 3 * 485 * 2.0 ** -20


def test_muon_tells_autograd_and_refuses_a_captured_first_step():
    w = torch.nn.Parameter(gradient(30, 70, 90))
    opt = mpi.Muon([w])
    loss = (w * w).sum()                    # its backward pass needs the weights as they are now
    w.grad = gradient(31, 70, 90)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    v = torch.nn.Parameter(w.detach().clone())
    v.grad = gradient(32, 70, 90)
    before = v.detach().clone()
    opt = mpi.Muon([v])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        with pytest.raises(mpi.InvalidArgumentError):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(v, before) and not opt.state[v]


@pytest.mark.parametrize("shape", [(140_000, 64, 256), (1100, 2048, 1024)])
def test_batches_beyond_32_bits(shape):
    """More than 2^31 elements and 2^32 bytes: the last matrix comes out as it does alone."""
    one = gradient(40, *shape[1:], dtype=torch.bfloat16)
    batch = torch.zeros(shape, dtype=torch.bfloat16, device="cuda")
    batch[-1] = one
    batch[0] = one
    got = mpi.orthogonalize(batch)
    want = mpi.orthogonalize(one)
    assert distance(want, exact(one)) <= bound(torch.bfloat16, False, shape)
    tolerance = 2 * bound(torch.bfloat16, False, shape)   # a list of another size may take other tiles, in another order
    assert distance(got[-1], want) <= tolerance and distance(got[0], want) <= tolerance
    assert not bool(got[1].any()) and not bool(got[-2].any())


def test_more_matrices_than_workgroups_of_a_launch():
    """2^32 lanes are 8388608 workgroups of 512: a batch of more is several launches."""
    count = (1 << 23) + 5
    batch = torch.ones(count, 1, 2, device="cuda")
    batch[:, 0, 1] = torch.arange(count, device="cuda") % 7
    got = mpi.orthogonalize(batch, steps=2)
    want = mpi.orthogonalize(batch[:7], steps=2)
    assert torch.equal(got[:7 * 1000].view(1000, 7, 1, 2), want.expand(1000, 7, 1, 2))
    last = torch.arange(count - 7, count, device="cuda") % 7
    assert torch.equal(got[-7:], want[last])
    middle = torch.arange((1 << 22) - 7, (1 << 22) + 7, device="cuda")
    assert torch.equal(got[middle], want[middle % 7])


def test_a_matrix_beyond_32_bits():
    """One matrix of more than 2^31 elements, a single step; its ends against X a + X (b A + c A A). That X is the rounded
    update over its norm; all of it is a sum of about 2100 products of which X's own rounding is the largest."""
    rows, cols = 1 << 20, 2100
    update = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for k in range(0, rows, 1 << 17):
        update[k:k + (1 << 17)] = torch.randn(1 << 17, cols, generator=torch.Generator("cuda").manual_seed(k), device="cuda")
    got = mpi.orthogonalize(update, steps=1)
    gram, size = torch.zeros(cols, cols, dtype=torch.float64, device="cuda"), 0.0
    for k in range(0, rows, 1 << 15):
        part = update[k:k + (1 << 15)].float()
        gram += (part.T.contiguous() @ part).double()
        size += float(part.square().sum(dtype=torch.float64))
    gram /= size
    inner = B * gram + C * gram @ gram
    for at in (slice(0, 300), slice(rows // 2, rows // 2 + 300), slice(rows - 300, rows)):
        x = update[at].double() / math.sqrt(size)
        assert distance(got[at], A * x + x @ inner) <= bound(torch.bfloat16, False, (rows, cols))
