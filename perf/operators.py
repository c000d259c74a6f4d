"""The operators of a training step around the gradient exchange, as cases that can be timed and checked:

  lookup         an embedding lookup with scaling (decoding, long batches)
  train          the same lookup and, through autograd, its dense gradient
  slices         the sum of the gathered rows of an IndexedSlices, one row for each distinct index
  orthogonalize  five Newton-Schulz steps on one matrix or a batch of them
  muon           one optimizer step on a list of matrices: momentum, Newton-Schulz, decay, update

`run` computes them with elementary torch operations where `own` is false, and with mpi_collectives where it is true.
"""
import math
import os
import sys

import torch

own = False

A, B, C = 3.4445, -4.7750, 2.0315   # the quintic's coefficients
EPS = 1e-7
STEPS = 5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def _mpi():
    path = os.path.join(os.getcwd(), "tensorflow-allreduce_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mpi_collectives
    return mpi_collectives


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the first layer of a decoding step: one token for each of 16 running sequences
        dict(name="lookup decode", op="lookup", tokens=16, rows=32000, width=2048, dtype="bfloat16", ids="int64"),
        # the first layer of a long training batch: 32 sequences of 4096 tokens, a large vocabulary
        dict(name="lookup long batch", op="lookup", tokens=131072, rows=131072, width=4096, dtype="bfloat16", ids="int64"),
        # a small model's step: forward and dense gradient, float32 as the ring reduces it
        dict(name="train small", op="train", tokens=1024, rows=8192, width=512, dtype="float32", ids="int64"),
        # a padded batch of odd sizes: ids of -1 are padding
        dict(name="train ragged", op="train", tokens=10007, rows=50021, width=1001, dtype="bfloat16", ids="int32"),
        # a large step: 16 sequences of 4096 tokens
        dict(name="train large", op="train", tokens=65536, rows=131072, width=2048, dtype="bfloat16", ids="int64"),
        # what an allgather of four ranks' small sparse gradients delivers
        dict(name="slices small", op="slices", ranks=4, tokens=129, rows=32000, width=300, dtype="float32", ids="int64"),
        # what eight ranks with two sequences of 4096 tokens each deliver
        dict(name="slices 8 ranks", op="slices", ranks=8, tokens=8192, rows=50021, width=1024, dtype="float32", ids="int64"),
        # the matrices of single attention heads, as one batch: float32 updates, a bfloat16 result
        dict(name="orthogonalize heads", op="orthogonalize", batch=48, rows=64, cols=128, dtype="float32", result="bfloat16"),
        # one matrix of odd sizes in float32
        dict(name="orthogonalize odd f32", op="orthogonalize", batch=1, rows=1000, cols=2731, dtype="float32", result="float32"),
        # the largest projection of a wide model
        dict(name="orthogonalize wide", op="orthogonalize", batch=1, rows=4096, cols=16384, dtype="bfloat16", result="bfloat16"),
        # the 54 matrices of the ResNet-50 set that the ring's benchmark reduces, float32 as the ring delivers them
        dict(name="muon resnet50", op="muon", set="resnet50", width=0, depth=0, dtype="float32"),
        # four blocks (four square projections, two of a feed-forward layer), bfloat16 weights, float32 momentum
        dict(name="muon blocks", op="muon", set="blocks", width=1024, depth=4, dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "train", "slices", "orthogonalize", "muon"])
    kind = rng.choice(["float32", "bfloat16", "float16"])
    ids = rng.choice(["int32", "int64"])
    if op == "lookup":
        width = _log(rng, 17, 4096)
        most = min(262144, (1 << 30) // (width * _SIZE[kind]))
        return dict(op=op, tokens=_log(rng, 1, most), rows=_log(rng, 1000, 131072), width=width, dtype=kind, ids=ids)
    if op == "train":
        width = _log(rng, 17, 2048)
        most = min(131072, (1 << 28) // (width * _SIZE[kind]))
        rows = _log(rng, 1000, min(131072, (1 << 29) // (width * _SIZE[kind])))
        return dict(op=op, tokens=_log(rng, 1, most), rows=rows, width=width, dtype=kind, ids=ids)
    if op == "slices":
        ranks = rng.choice([1, 2, 3, 4, 6, 8, 16])
        width = _log(rng, 1, 1024)
        tokens = _log(rng, 1, 65536 // ranks)
        return dict(op=op, ranks=ranks, tokens=tokens, rows=_log(rng, 100, 131072), width=width, dtype="float32", ids=ids)
    if op == "orthogonalize":
        rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
        batch = _log(rng, 1, max(1, min(64, (1 << 24) // (rows * cols))))
        kind = rng.choice(["float32", "bfloat16"])
        return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=kind, result=rng.choice([kind, "bfloat16"]))
    return dict(op=op, set="blocks", width=_log(rng, 64, 1400), depth=rng.randint(1, 4),
                dtype=rng.choice(["float32", "bfloat16"]))


def _matrices(case):
    """The shapes of a muon case."""
    if case["set"] == "blocks":
        w = case["width"]
        return ([(w, w)] * 4 + [(4 * w, w), (w, 4 * w)]) * case["depth"]
    shapes, cin = [(7 * 7 * 3, 64)], 64
    for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
        for b in range(blocks):
            shapes += [(cin, width), (9 * width, width), (width, 4 * width)]
            if b == 0:
                shapes.append((cin, 4 * width))
            cin = 4 * width
    return shapes + [(2048, 1000)]


# ---- inputs -----------------------------------------------------------------------------------

def _tokens(gen, case, count):
    """Token ids as text has them: a few are very common, most are rare; one in 32 is padding (-1)."""
    u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64)
    ids = (case["rows"] * u ** 4).long().clamp_(max=case["rows"] - 1)
    pad = torch.rand(count, generator=gen, device="cuda") < 1 / 32
    return ids.masked_fill(pad, -1).to(torch.int32 if case["ids"] == "int32" else torch.int64)


def _slices(case):
    """How many rows a slices case gathers, and how many of their indices are distinct."""
    count = case["ranks"] * case["tokens"]
    return count, min(case["rows"], (count + 1) // 2)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _update(gen, *shape):
    """A gradient as training has it: a few strong directions over noise, of small magnitude."""
    rank = min(16, shape[-1], shape[-2])
    left = _normal(gen, *shape[:-1], rank)
    right = _normal(gen, *shape[:-2], rank, shape[-1])
    return 1e-4 * (left @ right + _normal(gen, *shape))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"case": case}
    kind = _TYPES[case["dtype"]]
    if case["op"] in ("lookup", "train"):
        state["ids"] = _tokens(gen, case, case["tokens"])
        state["weight"] = _normal(gen, case["rows"], case["width"], dtype=kind)
        state["scale"] = math.sqrt(case["width"])
        if case["op"] == "train":
            state["weight"].requires_grad_(True)
            state["grad"] = _normal(gen, case["tokens"], case["width"], dtype=kind)
    elif case["op"] == "slices":
        # every rank's rows one behind the other; each of `distinct` tokens occurs, the common ones often
        count, distinct = _slices(case)
        ids = torch.randperm(case["rows"], generator=gen, device="cuda")[:distinct]
        again = (distinct * torch.rand(count - distinct, generator=gen, device="cuda", dtype=torch.float64) ** 4).long()
        indices = torch.cat([ids, ids[again.clamp_(max=distinct - 1)]])
        indices = indices[torch.randperm(count, generator=gen, device="cuda")]
        state["indices"] = indices.to(torch.int32 if case["ids"] == "int32" else torch.int64)
        state["values"] = _normal(gen, count, case["width"])
    elif case["op"] == "orthogonalize":
        shape = (case["batch"], case["rows"], case["cols"]) if case["batch"] > 1 else (case["rows"], case["cols"])
        state["update"] = _update(gen, *shape).to(kind)
    else:
        shapes = _matrices(case)
        # weights and momentum in one buffer each, as a program keeps them that reduces or saves them at once
        counts = [m * n for m, n in shapes]
        state["weights"] = torch.empty(sum(counts), device="cuda", dtype=kind)
        state["buffers"] = torch.empty(sum(counts), device="cuda", dtype=torch.float32)
        params = [torch.nn.Parameter(w.view(s)) for w, s in zip(state["weights"].split(counts), shapes)]
        state["params"] = params
        state["momentum"] = [b.view(s) for b, s in zip(state["buffers"].split(counts), shapes)]
        for p, b in zip(params, state["momentum"]):
            p.data.copy_(_normal(gen, *p.shape).mul_(p.shape[1] ** -0.5))
            p.grad = _update(gen, *p.shape).to(kind)
            b.copy_(5 * _update(gen, *p.shape))
        if own:
            opt = _mpi().Muon(params, lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS)
            for p, m in zip(params, state["momentum"]):
                opt.state[p]["momentum_buffer"] = m
            state["optimizer"] = opt
    return state


# ---- one pass ---------------------------------------------------------------------------------

def _plain_lookup(ids, weight, scale):
    inside = ((ids >= 0) & (ids < weight.shape[0])).unsqueeze(-1)
    rows = weight[ids.long().clamp(0, weight.shape[0] - 1)].float() * scale
    return torch.where(inside, rows, 0.0).to(weight.dtype)


def _plain_gradient(grad, ids, rows, scale):
    at = torch.where((ids >= 0) & (ids < rows), ids, rows).long()
    total = torch.zeros(rows + 1, grad.shape[1], device=grad.device, dtype=torch.float32)
    total.index_add_(0, at, grad.float())
    return (total[:rows] * scale).to(grad.dtype)


def _plain_newton_schulz(update):
    x = update.float()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    for _ in range(STEPS):
        gram = x @ x.mT.contiguous()
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x.mT.contiguous() if tall else x


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        mpi = _mpi()
        if op == "lookup":
            return mpi.embedding(state["ids"], state["weight"], scale=state["scale"])
        if op == "train":
            out = mpi.embedding(state["ids"], state["weight"], scale=state["scale"])
            return out, torch.autograd.grad(out, state["weight"], state["grad"])[0]
        if op == "slices":
            total = mpi.sum_slices(mpi.IndexedSlices(state["values"], state["indices"], (case["rows"], case["width"])))
            return total.indices, total.values
        if op == "orthogonalize":
            return mpi.orthogonalize(state["update"], steps=STEPS, dtype=_TYPES[case["result"]])
        state["optimizer"].step()
        return state["weights"], state["buffers"]

    with torch.no_grad():
        if op == "lookup":
            return _plain_lookup(state["ids"], state["weight"], state["scale"])
        if op == "train":
            out = _plain_lookup(state["ids"], state["weight"], state["scale"])
            return out, _plain_gradient(state["grad"], state["ids"], case["rows"], state["scale"])
        if op == "slices":
            inside = (state["indices"] >= 0) & (state["indices"] < case["rows"])
            indices, at = torch.unique(state["indices"][inside], return_inverse=True)
            total = torch.zeros(indices.numel(), case["width"], device="cuda")
            return indices, total.index_add_(0, at, state["values"][inside])
        if op == "orthogonalize":
            return _plain_newton_schulz(state["update"]).to(_TYPES[case["result"]])
        for p, m in zip(state["params"], state["momentum"]):
            g = p.grad.float()
            m.mul_(MOMENTUM).add_(g)
            step = _plain_newton_schulz(g + MOMENTUM * m)
            grow = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            p.copy_((p * (1 - LR * DECAY) - (LR * grow) * step).to(p.dtype))
        return state["weights"], state["buffers"]


# ---- what a pass cannot do without ------------------------------------------------------------

def _newton_schulz_flops(rows, cols):
    """The Gram matrix and its square are symmetric: half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op in ("lookup", "train"):
        id_size = 4 if case["ids"] == "int32" else 8
        distinct = min(case["tokens"], case["rows"])
        read = case["tokens"] * id_size + distinct * case["width"] * size
        moved = read + case["tokens"] * case["width"] * size
        flops = case["tokens"] * case["width"]
        if op == "train":
            moved += (case["tokens"] + case["rows"]) * case["width"] * size
            flops *= 2
        return {"bytes": moved, "flops": flops}
    if op == "slices":
        count, distinct = _slices(case)
        return {"bytes": (count + distinct) * (case["width"] * size + (4 if case["ids"] == "int32" else 8)),
                "flops": count * case["width"]}
    if op == "orthogonalize":
        one = case["rows"] * case["cols"]
        return {"bytes": case["batch"] * one * (size + _SIZE[case["result"]]),
                "flops": case["batch"] * _newton_schulz_flops(case["rows"], case["cols"])}
    shapes = _matrices(case)
    return {"bytes": sum(m * n for m, n in shapes) * (3 * size + 8),
            "flops": sum(_newton_schulz_flops(m, n) for m, n in shapes)}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _exact_sums(values, index, distinct):
    """Sums of the rows of `values` by their place in `distinct` (ascending), by differences of a running sum over the
    rows in order of their index."""
    order = torch.argsort(index, stable=True)
    end = torch.searchsorted(index[order].contiguous(), distinct, right=True)
    out = torch.empty(distinct.numel(), values.shape[1], device="cuda", dtype=torch.float64)
    for c in range(0, values.shape[1], 256):
        run_sum = torch.cumsum(values[:, c:c + 256].double()[order], 0)
        run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
        at_end = run_sum[end]
        out[:, c:c + 256] = torch.diff(at_end, dim=0, prepend=torch.zeros_like(at_end[:1]))
    return out


def _exact_newton_schulz(update):
    x = update.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    if x.shape[-2] > x.shape[-1]:   # the smaller Gram matrix, from the other side
        for _ in range(STEPS):
            gram = torch.matmul(x.mT.contiguous(), x)
            poly = torch.baddbmm(B * gram, gram, gram, alpha=C) if gram.dim() == 3 else torch.addmm(B * gram, gram, gram, alpha=C)
            x = A * x + torch.matmul(x, poly)
        return x
    for _ in range(STEPS):
        gram = torch.matmul(x, x.mT.contiguous())
        poly = torch.baddbmm(B * gram, gram, gram, alpha=C) if gram.dim() == 3 else torch.addmm(B * gram, gram, gram, alpha=C)
        x = A * x + torch.matmul(poly, x)
    return x


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("lookup", "train"):
            ids, weight, rows = state["ids"].long(), state["weight"], case["rows"]
            out = torch.zeros(case["tokens"], case["width"], device="cuda", dtype=torch.float64)
            hit = torch.nonzero((ids > -1) & (ids < rows)).reshape(-1)
            out[hit] = torch.index_select(weight, 0, ids[hit]).double() * state["scale"]
            if op == "lookup":
                return out
            every = torch.arange(rows, device="cuda")
            return out, _exact_sums(state["grad"][hit], ids[hit], every) * state["scale"]
        if op == "slices":
            index = state["indices"].long()
            hit = torch.nonzero((index > -1) & (index < case["rows"])).reshape(-1)
            distinct = torch.unique(index[hit])
            return distinct.to(state["indices"].dtype), _exact_sums(state["values"][hit], index[hit], distinct)
        if op == "orthogonalize":
            return _exact_newton_schulz(state["update"])
        weights, buffers = [], []
        for p, m in zip(state["params"], state["momentum"]):
            g = p.grad.double()
            buffers.append(MOMENTUM * m.double() + g)
            o = _exact_newton_schulz(g + MOMENTUM * buffers[-1])
            weights.append(p.double() - LR * (DECAY * p.double() + math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * o))
        return torch.cat([w.reshape(-1) for w in weights]), torch.cat([b.reshape(-1) for b in buffers])
