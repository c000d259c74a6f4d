"""Operators of a training step around the gradient exchange, over torch
tensors on the GPU: the embedding lookup and its gradient, the sum of the rows
that allreduce(IndexedSlices) gathers, and the orthogonalised update of a
matrix with the optimizer that uses it.

They run on torch's current stream of the tensors' device, allocate through
torch and synchronise nothing (except where a result's size depends on the
data: sum_slices, and the sparse gradient of embedding). torch.compile breaks
its graph around them and runs them as they are; what records a trace instead
(jit.trace, make_fx, torch.export) is refused.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import step_abi
from ._plugin import InvalidArgumentError

_FLOATS = {torch.float32: step_abi.F32, torch.bfloat16: step_abi.BF16, torch.float16: step_abi.F16}
_IDS = {torch.int32: step_abi.I32, torch.int64: step_abi.I64}


class IndexedSlices:
    """A sparse representation of a set of tensor slices at given indices
    (the tf.IndexedSlices the reference's allreduce accepts)."""

    def __init__(self, values, indices, dense_shape=None):
        self.values, self.indices, self.dense_shape = values, indices, dense_shape


def _refuse(why, *args):
    raise InvalidArgumentError(why % args)


_MODES = tuple(getattr(torch._C._TorchDispatchModeKey, k) for k in ("PROXY", "FAKE", "FUNCTIONAL"))


def _check_run(what):
    """Refuses to be traced. The kernels are launched past torch's dispatcher: a trace would hold the empty result and not
    what fills it."""
    if torch._C._get_tracing_state() is not None or torch._C._len_torch_dispatch_stack() and any(
            torch._C._get_dispatch_mode(k) is not None for k in _MODES):
        _refuse("%s: it launches kernels of its own, which a trace (jit.trace, make_fx, torch.export) does not hold", what)


def _check_tensor(t, name, types, what):
    if not isinstance(t, torch.Tensor):
        _refuse("%s: %s must be a torch.Tensor, got %s", what, name, type(t).__name__)
    if t.dtype not in types:
        _refuse("%s: %s has type %s; it takes %s", what, name, t.dtype, ", ".join(str(k) for k in types))
    if not t.is_cuda:
        _refuse("%s: %s is on %s; there are GPU kernels only", what, name, t.device)


def _same_device(what, a, b):
    if a.get_device() != b.get_device():
        _refuse("%s: tensors on %s and %s", what, a.device, b.device)


def _rows_of(t):
    """`t` as rows whose columns are contiguous and which are t.stride(0) apart, copied only if it is not."""
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _as_stored(t):
    """t with the values that its memory holds: a view can stand for the negative of them (the imaginary part of a conjugate)."""
    return t.resolve_neg() if t.is_neg() else t


def _is_dual(t):
    """Whether t carries a tangent of forward-mode differentiation."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _in_memory(tangent):
    """A tangent as the kernels read it: one that is known to be zero has no memory."""
    return torch.zeros(tangent.shape, dtype=tangent.dtype, device=tangent.device) if tangent._is_zerotensor() else tangent


# The current stream and device as plain numbers: these calls are a large part of a small operator's time, and in a
# backward pass, which runs on a thread of autograd's own, every Python object that is touched comes from another core.
_stream_of = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_empty = torch.empty


def _on_device(fn, tensor, *args):
    """fn(*args) with the tensor's device as the current one."""
    with torch.cuda.device(tensor.device):
        return fn(*args)


def _lookup(ids, weight, scale):
    index = weight.get_device()
    if index != _current_device():
        return _on_device(_lookup, weight, ids, weight, scale)
    rows, width = weight.shape
    stride = width
    if not weight.is_contiguous():
        weight, stride = _rows_of(weight)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    dtype = weight.dtype
    out = _empty((*ids.shape, width), dtype=dtype, device=weight.device)
    status = (step_abi._lib or step_abi.lib()).step_embedding_lookup(
        ids.data_ptr(), _IDS[ids.dtype], ids.numel(), weight.data_ptr(), _FLOATS[dtype], rows, width, stride, scale,
        out.data_ptr(), _stream_of(index))
    if status:
        step_abi.check(status, "embedding")
    return out


def embedding_gradient(grad, ids, rows, scale=1.0):
    """The dense gradient of `embedding` with respect to its table: row v of the
    result is scale * the sum of the rows of `grad` whose id is v, 0 if there is
    none.

    Arguments:
        grad: gradient of the lookup's result, ids.shape + (width,), float32,
              bfloat16 or float16. Its last dimension should be contiguous (it
              is copied otherwise).
        ids: int32 or int64 tensor; ids outside [0, rows) contribute nothing.
        rows: rows of the table.
        scale: as in `embedding`.

    Sums are taken in 32 bits in the order of the tokens and rounded once to
    grad's type; the same call gives the same bits every time. The result is
    differentiable with respect to grad, backwards and forwards."""
    what = "embedding_gradient"
    _check_run(what)
    _check_tensor(grad, "grad", _FLOATS, what)
    _check_tensor(ids, "ids", _IDS, what)
    _same_device(what, grad, ids)
    rows = int(rows)
    if rows < 0:
        _refuse("%s: rows is %d", what, rows)
    grad = _as_stored(grad)
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        _refuse("%s: a gradient of shape %s for ids of shape %s", what, tuple(grad.shape), tuple(ids.shape))
    if grad.requires_grad and torch.is_grad_enabled() or _is_dual(grad):
        return _EmbeddingGradient.apply(grad, ids, rows, float(scale))
    return _gradient(grad, ids, rows, float(scale))


def _gradient(grad, ids, rows, scale):
    index = grad.get_device()
    if index != _current_device():
        return _on_device(_gradient, grad, grad, ids, rows, scale)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    tokens, width = ids.numel(), grad.shape[-1]
    stride = width
    if not grad.is_contiguous():
        grad, stride = _rows_of(grad.reshape(tokens, width))
    dtype, device = grad.dtype, grad.device
    out = _empty((rows, width), dtype=dtype, device=device)
    L = step_abi._lib or step_abi.lib()
    size = L.step_embedding_gradient_workspace(tokens, rows, width)
    ws = _empty(size, dtype=torch.uint8, device=device)
    status = L.step_embedding_gradient(
        ids.data_ptr(), _IDS[ids.dtype], tokens, grad.data_ptr(), _FLOATS[dtype], rows, width, stride, scale,
        out.data_ptr(), ws.data_ptr(), size, _stream_of(index))
    if status:
        step_abi.check(status, "embedding_gradient")
    return out


def can_sum_slices(slices):
    """Whether sum_slices takes the tensors of `slices`: their types, on a GPU, of sizes that fit its 32-bit places and its
    launches. (A lane sums 16 bytes of the runs that begin in eight rows, and may have as many idle ones beside it: 2^36 bytes
    of rows, of at least 16 each, are a quarter of the 2^32 lanes of a launch.)"""
    values, indices = slices.values, slices.indices
    if not (values.is_cuda and values.dtype in _FLOATS and indices.is_cuda and indices.dtype in _IDS and indices.dim() == 1):
        return False
    row = math.prod(values.shape[1:])
    return (slices.dense_shape is not None and int(slices.dense_shape[0]) < 1 << 31 and row <= 65535 * 256 * 4 and
            indices.shape[0] < 1 << 31 and indices.shape[0] * max(row * values.element_size(), 16) <= 1 << 36)


def sum_slices(slices):
    """An IndexedSlices with one row for each distinct index, in ascending order:
    the sum of the rows of `slices` that have it. This is what makes a gradient
    of what allreduce(IndexedSlices) delivers, where every rank's rows stand one
    behind the other.

    Arguments:
        slices: IndexedSlices with values of shape (n, ...), float32, bfloat16 or
                float16, indices of shape (n,), int32 or int64, and dense_shape
                set. Rows whose index is outside [0, dense_shape[0]) are left out.

    Sums are taken in 32 bits in the order of the rows and rounded once; the
    same call gives the same bits every time. The number of distinct indices is
    read from the GPU, so the call waits for its stream and cannot be captured
    into a graph. No gradient flows through it, backwards or forwards."""
    what = "sum_slices"
    _check_run(what)
    if not isinstance(slices, IndexedSlices):
        _refuse("%s: an IndexedSlices is needed, got %s", what, type(slices).__name__)
    values, indices = slices.values, slices.indices
    _check_tensor(values, "values", _FLOATS, what)
    _check_tensor(indices, "indices", _IDS, what)
    _same_device(what, values, indices)
    values = _as_stored(values)
    if slices.dense_shape is None:
        _refuse("%s: dense_shape is needed", what)
    shape = tuple(int(d) for d in slices.dense_shape)
    if indices.dim() != 1 or values.dim() < 1 or values.shape[0] != indices.shape[0] or tuple(values.shape[1:]) != shape[1:]:
        _refuse("%s: values of shape %s, indices of shape %s, dense_shape %s", what, tuple(values.shape),
                tuple(indices.shape), shape)
    if shape[0] < 0:
        _refuse("%s: dense_shape is %s", what, shape)
    if torch.cuda.is_current_stream_capturing():
        _refuse("%s: the size of the result depends on the data: it cannot be captured into a graph", what)
    out_ids, out_values = _sum_slices(values, indices, shape[0], 1.0)
    return IndexedSlices(out_values, out_ids, shape)


def _sum_slices(values, indices, rows, scale):
    index = values.get_device()
    if index != _current_device():
        return _on_device(_sum_slices, values, values, indices, rows, scale)
    shape, dtype, device = tuple(values.shape[1:]), values.dtype, values.device
    tokens, width = indices.shape[0], math.prod(shape)
    flat, stride = _rows_of(values.reshape(tokens, width))
    indices = indices.contiguous()
    most = min(tokens, rows)
    out_ids = _empty(most, dtype=indices.dtype, device=device)
    out = _empty((most, width), dtype=dtype, device=device)
    count = _empty(1, dtype=torch.int64, device=device)
    L = step_abi._lib or step_abi.lib()
    size = L.step_sum_slices_workspace(tokens, rows, width)
    ws = _empty(size, dtype=torch.uint8, device=device)
    step_abi.check(L.step_sum_slices(
        indices.data_ptr(), _IDS[indices.dtype], tokens, flat.data_ptr(), _FLOATS[dtype], rows, width, stride, scale,
        out_ids.data_ptr(), out.data_ptr(), count.data_ptr(), ws.data_ptr(), size, _stream_of(index)), "sum_slices")
    n = count.item()
    out_ids, out = out_ids[:n], out[:n].view((n,) + shape)
    # a gradient lives until the next step: where it is less than half of what was set aside, it does not keep the rest alive
    return (out_ids.clone(), out.clone()) if 2 * n < most else (out_ids, out)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, sparse):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.set_materialize_grads(False)
        ctx.call = (weight.shape[0], scale, sparse)
        return _lookup(ids, weight, scale)

    @staticmethod
    def backward(ctx, grad):
        if grad is None:
            return None, None, None, None
        rows, scale, sparse = ctx.call
        ids, = ctx.saved_tensors
        grad = _as_stored(grad)
        if grad.requires_grad or _is_dual(grad):
            return None, _EmbeddingGradient.apply(grad, ids, rows, scale), None, None
        if not sparse:
            return None, _gradient(grad, ids, rows, scale), None, None
        if torch.cuda.is_current_stream_capturing():
            _refuse("embedding: the size of a sparse gradient depends on the data: it cannot be captured into a graph")
        index, values = _sum_slices(grad.reshape(ids.numel(), grad.shape[-1]), ids.reshape(-1), rows, scale)
        return None, torch.sparse_coo_tensor(index.long().unsqueeze(0), values, (rows, grad.shape[-1]),
                                             is_coalesced=True, check_invariants=False), None, None

    @staticmethod
    def jvp(ctx, _ids, tangent, _scale, _sparse):
        ids, = ctx.saved_tensors
        return embedding(ids, _in_memory(tangent), ctx.call[1])


class _EmbeddingGradient(torch.autograd.Function):
    """The gradient as a function of its own, for gradients of gradients: it is linear, and its transpose the lookup."""

    @staticmethod
    def forward(ctx, grad, ids, rows, scale):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.rows, ctx.scale = rows, scale
        return _gradient(grad, ids, rows, scale)

    @staticmethod
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return embedding(ids, grad, ctx.scale), None, None, None

    @staticmethod
    def jvp(ctx, tangent, _ids, _rows, _scale):
        ids, = ctx.saved_tensors
        return embedding_gradient(_in_memory(tangent), ids, ctx.rows, ctx.scale)


def embedding(ids, weight, scale=1.0, sparse=False):
    """Rows of a table by id, times a scale: ids.shape + (width,), in the table's type.

    Arguments:
        ids: int32 or int64 tensor of any shape. An id outside [0, rows) reads
             nothing: its row is zero and it has no part in the gradient, so an
             id of -1 is padding.
        weight: the table, (rows, width), float32, bfloat16 or float16; rows may be
                any distance apart (a slice of a larger table).
        scale: a number every row is multiplied by (sqrt(width), say), in 32 bits
               before the one rounding to the table's type.
        sparse: False: weight's gradient is dense (see embedding_gradient). True:
                it is a sparse tensor with one row per distinct id, which
                DistributedOptimizer exchanges as an IndexedSlices; its size
                depends on the data, so that backward pass waits for its stream
                and cannot be captured into a graph. Where gradients of
                gradients are asked for (create_graph, or a gradient that carries
                a tangent) it is dense all the same.

    The lookup is linear in the table and differentiable backwards and, by
    torch.autograd.forward_ad, forwards.

    A forward and backward pass can be captured into a graph. As with every
    function of torch, no eager graph of the same leaves may be alive then:
    autograd would join its stream into the capture.
    """
    what = "embedding"
    _check_run(what)
    _check_tensor(ids, "ids", _IDS, what)
    _check_tensor(weight, "weight", _FLOATS, what)
    _same_device(what, ids, weight)
    weight = _as_stored(weight)
    if weight.dim() != 2:
        _refuse("%s: a table of shape %s; it has two dimensions", what, tuple(weight.shape))
    if weight.requires_grad and torch.is_grad_enabled() or _is_dual(weight):
        return _Embedding.apply(ids, weight, float(scale), bool(sparse))
    return _lookup(ids, weight, float(scale))


# The quintic whose five steps bring every singular value between 0.003 and 1 to within 0.7 .. 1.2.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)
_MOST_STEPS = 64


def _coefficients(coefficients, steps, what):
    """`steps` triples (a, b, c) as a C array; one triple stands for every step."""
    if not 1 <= steps <= _MOST_STEPS:
        _refuse("%s: %r steps; 1 to %d are possible", what, steps, _MOST_STEPS)
    rows = list(coefficients)
    if len(rows) == 3 and not any(hasattr(r, "__len__") for r in rows):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        _refuse("%s: coefficients are (a, b, c) or one such triple for each of %d steps", what, steps)
    flat = [float(v) for r in rows for v in r]
    return (ctypes.c_float * len(flat))(*flat)


def orthogonalize(update, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, dtype=None, precise=None):
    """Brings the singular values of a matrix near 1 and keeps its singular vectors,
    by Newton-Schulz steps: X = U / (|U| + eps) with the Frobenius norm, then
    `steps` times A = X X^T, X = a X + (b A + c A A) X.

    Arguments:
        update: tensor of shape (..., rows, cols), float32, bfloat16 or float16;
                leading dimensions are a batch of matrices.
        steps: number of steps.
        coefficients: (a, b, c), or one such triple for each step. They have to
                keep the singular values below 2 (X X^T below 4 in every entry).
        eps: added to the norm, so that a zero matrix gives zeros.
        dtype: type of the result; update's by default.
        precise: False: products of float16 operands with float32 sums, the rest
                of each iterate kept beside them: the norm of the difference is
                0.05 to 0.3 % of the result's, whatever update's rank (up to
                0.6 % with fewer than eight rows or columns); bfloat16's own
                rounding is 0.17 %, float16's 0.02 %. True: products of split
                operands, three times the work: about 1e-6 off. Default: False
                if the result is bfloat16, else True. Matrices of at most 64 x
                256 (or the transposed) are always precise.

    An update with an infinity or NaN gives NaN. No gradient flows through the
    result, backwards or forwards."""
    what = "orthogonalize"
    _check_run(what)
    _check_tensor(update, "update", _FLOATS, what)
    if update.dim() < 2:
        _refuse("%s: an update of shape %s; it has two dimensions at least", what, tuple(update.shape))
    dtype = update.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        _refuse("%s: a result of type %s", what, dtype)
    table = _coefficients(coefficients, steps, what)
    precise = dtype != torch.bfloat16 if precise is None else bool(precise)
    index = update.get_device()
    if index != _current_device():
        return _on_device(orthogonalize, update, update, steps, coefficients, eps, dtype, precise)
    update = _as_stored(update.detach()).contiguous()
    out = _empty(update.shape, dtype=dtype, device=update.device)
    rows, cols = update.shape[-2:]
    count = update.numel() // (rows * cols) if update.numel() else 0
    one = step_abi.Matrix(update.data_ptr(), None, out.data_ptr(), rows, cols, count, 0.0)
    L = step_abi._lib or step_abi.lib()
    size = L.step_orthogonalize_workspace(one, 1, precise)
    ws = _empty(size, dtype=torch.uint8, device=update.device)
    step_abi.check(L.step_orthogonalize(one, 1, _FLOATS[update.dtype], _FLOATS[dtype], precise, steps, table, float(eps),
                                        ws.data_ptr(), size, _stream_of(index)), what)
    return out


class Muon(torch.optim.Optimizer):
    """Optimizer for the matrices of a model: momentum, then the orthogonalised
    update (see `orthogonalize`), with decoupled weight decay:

        M <- momentum M + G
        U  = G + momentum M  (nesterov)  or  M
        W <- W (1 - lr weight_decay) - lr s orthogonalize(U)

    A step can be captured into a graph once every momentum exists, that is after
    a step of its own; lr and the other options are then those of the capture.

    Made to be wrapped by DistributedOptimizer. All matrices of a step go through
    each product in one launch. Embeddings, biases and other vectors belong to
    another optimizer.

    Arguments:
        params: matrices (two-dimensional), float32, bfloat16 or float16, on the
                GPU, or dicts of parameter groups with these options.
        lr: learning rate.
        momentum, nesterov: as above. The momentum is held in float32.
        weight_decay: as above.
        steps, coefficients, eps: as in `orthogonalize`.
        adjust: what s is. "shape": sqrt(max(1, rows / cols)). "rms":
                0.2 sqrt(max(rows, cols)), which gives the update the size that
                Adam's usually has.
        precise: as in `orthogonalize`, matrix by matrix; by default True for
                float32 weights (0.3 % of an update is far below what 16-bit
                weights round).
    """

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=NEWTON_SCHULZ, eps=1e-7, adjust="shape", precise=None):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, adjust=adjust, precise=precise))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            if group["adjust"] not in ("shape", "rms"):
                _refuse("Muon: adjust is %r; it is \"shape\" or \"rms\"", group["adjust"])
            _coefficients(group["coefficients"], group["steps"], "Muon")
            for p in group["params"]:
                if p.dim() != 2 or p.dtype not in _FLOATS:
                    _refuse("Muon: a parameter of shape %s and type %s; it takes matrices of type %s", tuple(p.shape),
                            p.dtype, ", ".join(str(k) for k in _FLOATS))
        except InvalidArgumentError:
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def step(self, closure=None):
        """One step for every parameter that has a gradient."""
        _check_run("Muon.step")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is not None:
                    alike.setdefault((p.device, p.dtype), []).append(p)
            for (device, dtype), params in alike.items():
                if device.type != "cuda":
                    _refuse("Muon: a weight on %s; there are GPU kernels only", device)
                with torch.cuda.device(device):
                    self._step(group, device, dtype, params)
        return loss

    def _step(self, group, device, dtype, params):
        rule = 0.2 if group["adjust"] == "rms" else None
        table = (step_abi.Matrix * len(params))()
        moved, keep = [], []      # weights that are not contiguous, with the copies that take the step; tensors in use
        for p, row in zip(params, table):
            g = p.grad
            if p.is_neg():
                _refuse("Muon: a weight that stands for the negative of its memory (resolve_neg makes one that does not)")
            if g.is_sparse:
                _refuse("Muon: a sparse gradient; it takes matrices with dense ones")
            if g.dtype != dtype or g.device != device:
                _refuse("Muon: a weight of type %s on %s with a gradient of type %s on %s", dtype, device, g.dtype, g.device)
            state = self.state[p]
            m = state.get("momentum_buffer")
            if m is None:
                if torch.cuda.is_current_stream_capturing():
                    _refuse("Muon: a first step cannot be captured into a graph, whose replays would begin with a momentum "
                            "of zero again; take one before")
                m = state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=device)
            elif m.dtype != torch.float32 or m.device != device or m.shape != p.shape or not m.is_contiguous():
                _refuse("Muon: a momentum buffer of shape %s and type %s on %s", tuple(m.shape), m.dtype, m.device)
            w = p
            if not p.is_contiguous():
                w = p.contiguous()
                moved.append((p, w))
            if not g.is_contiguous() or g.is_neg():
                g = _as_stored(g).contiguous()
                keep.append(g)
            rows, cols = p.shape
            row.grad, row.momentum, row.out = g.data_ptr(), m.data_ptr(), w.data_ptr()
            row.rows, row.cols, row.count = rows, cols, 1 if rows and cols else 0
            row.rate = group["lr"] * (rule * math.sqrt(max(rows, cols)) if rule else math.sqrt(max(1.0, rows / cols)) if cols else 0.0)
        steps = group["steps"]
        precise = dtype == torch.float32 if group["precise"] is None else bool(group["precise"])
        L = step_abi._lib or step_abi.lib()
        size = L.step_orthogonalize_workspace(table, len(params), precise)
        ws = _empty(size, dtype=torch.uint8, device=device)
        step_abi.check(L.step_muon(
            table, len(params), _FLOATS[dtype], precise, steps, _coefficients(group["coefficients"], steps, "Muon"),
            group["eps"], group["momentum"], bool(group["nesterov"]), 1.0 - group["lr"] * group["weight_decay"],
            ws.data_ptr(), size, _stream_of(device.index)), "Muon.step")
        for p, w in moved:
            p.copy_(w)
        torch.autograd.graph.increment_version(params)  # a backward pass that still needs the old weights has to notice

    def load_state_dict(self, state_dict):
        """Unlike the base class, which gives every buffer its parameter's type, this keeps the momentum in float32."""
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                m = state_dict["state"].get(key, {}).get("momentum_buffer")
                if m is not None:
                    self.state[p]["momentum_buffer"] = m.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()
