"""Distillation: a teacher's top logits (`top_logits`) and the loss of a student against them (`distill_loss_topk`), autograd over
the C ABI (segk_top_logits, segk_distill).  CPU tensors are served by the same formulas in torch ops (`_host_*`)."""
import math
from typing import NamedTuple, Optional

import torch

from . import ops
from ._lib import call, query
from .ops import _env, dt

MEAN, EACH, SKIP = 1, 2, 4          # flag bits of segk_distill
MAX_K = 64
PLANE_FEW, PLANE_CLASSES, PLANE_TOP, PLANE_POSITIONS, PLANE_INNER = 32, 256, 8, 16384, 16
REST_FLOOR = 2.0 ** -20             # a rest of the teacher's mass up to this is rounding and counts as none


class TopLogits(NamedTuple):
    """What is kept of a teacher's logits: the k greatest of each position in descending order, their classes (int32; -1 or any
    other value that is no class marks an entry that does not exist), and the logsumexp of all classes at the temperature the
    loss will use (None: the kept logits are renormalised).  `values` and `indices` have the logits' shape with k in place of the
    class dimension, `lse` the shape without it.  Batches like any named tuple in a DataLoader (whose default collation takes no None: without lse, store (values, indices))."""
    values: torch.Tensor
    indices: torch.Tensor
    lse: Optional[torch.Tensor] = None

    def to(self, *args, **kw):
        v = self.values.to(*args, **kw)
        nb = bool(kw.get("non_blocking", False))
        return TopLogits(v, self.indices.to(v.device, non_blocking=nb), None if self.lse is None else self.lse.to(v.device, non_blocking=nb))

    def cuda(self, device=None):
        return self.to(torch.device("cuda" if device is None else device))

    def cpu(self):
        return self.to(torch.device("cpu"))


def _check(logits, dim, temperature):
    if logits.dim() < 1 or not logits.dtype.is_floating_point:
        raise TypeError(f"logits of floating point type are expected, got {logits.dtype} with {logits.dim()} dimensions")
    if not -logits.dim() <= dim < logits.dim():
        raise IndexError(f"dimension {dim} is out of range for logits with {logits.dim()} dimensions")
    if not (isinstance(temperature, (int, float)) and 2.0 ** -40 <= temperature <= 2.0 ** 40):
        raise ValueError(f"temperature has to be a number between 2^-40 and 2^40, got {temperature}")
    return dim % logits.dim()


def _in_place(C, outer, inner, size, selected):
    """Whether class planes [N, C, ...] are read as they are, not copied into rows; selected: as many are selected (0: the loss).

    Up to PLANE_FEW classes always (a thread holds them).  Up to PLANE_CLASSES, and PLANE_TOP selected, where the positions fill the chip: until
    they do a thread for each costs the same time however few they are, about in proportion to the classes (and, of the selection, half as
    much again beyond 2 kept), while the copy's grows with the positions.  In place / copied, fp32 (bf16), us: 128 x 128 positions, loss
    with gradient, 8 kept: 33 classes 32/50 (34/61), 80 38/53 (47/59), 150 47/62 (66/70), 256 69/70 (94/72), 64 kept of 80 134/134
    (145/182); selection of 1: 80 classes 13/19 (18/19), 150 22/28 (30/27), 256 33/37 (48/32); of 8: 80 23/23 (28/33), 150 40/32 (48/32), 256
    63/41 (78/36); 192 x 192: 150 40/61 (48/61), 256 70/82 (78/64).  An image has a workgroup of its own, so those of few positions
    leave it idle: 16384 images of 2 x 2 (4096 of 4 x 4) positions, 80 classes, loss with gradient 334/126 (104/128).  With
    PLANE_POSITIONS 0 whatever the kernels can read is read in place."""
    if inner == 1 or C <= PLANE_FEW:
        return True
    full = (164 if size == 4 else 102) * (2 / 3 if selected > 2 else 1)      # classes of which PLANE_POSITIONS are enough
    return C <= PLANE_CLASSES and selected <= PLANE_TOP and inner >= min(PLANE_INNER, PLANE_POSITIONS) and outer * inner >= PLANE_POSITIONS * max(1.0, C / full)


def _canonical(x, dim, selected=0, keep=False):
    """(tensor, outer, C, inner, ld, moved): x as `outer` images of C x `inner`, in place where its strides allow it.  Classes in front
    of other dimensions are moved to the end (a copy) where _in_place does not hold; never with `keep`."""
    shape = x.shape
    if dim == 1 and len(shape) == 2 and x.is_contiguous():            # the usual rows, for the sake of a short call
        return x, shape[0], shape[1], 1, shape[1], False
    C, outer, inner = shape[dim], math.prod(shape[:dim]), math.prod(shape[dim + 1:])
    moved = not (keep or _in_place(C, outer, inner, x.element_size(), selected))
    if moved:
        x, outer, inner = x.movedim(dim, -1), outer * inner, 1
    if x.is_contiguous():
        return x, outer, C, inner, C * inner, moved
    x = x.reshape(outer, C, inner)
    if (C > 1 and x.stride(1) != inner) or (inner > 1 and x.stride(2) != 1) or (outer > 1 and x.stride(0) < C * inner):
        x = x.contiguous()
    return x, outer, C, inner, (x.stride(0) if outer > 1 else C * inner), moved


def top_logits(logits, k, dim=1, temperature=1.0):
    """The k greatest logits along `dim` (1 <= k <= min(64, classes)) as TopLogits(values, indices int32, lse): descending, ties to
    the lower class, NaN as the greatest; lse = logsumexp(logits / temperature) over all classes, fp32 (NaN where a logit is NaN or
    +infinity).  float32, bfloat16 and float16 logits; values keep their type.  Not differentiable: a teacher's answer is data.

    The class dimension may stand anywhere: last (rows of any number of classes, read where they are) or in front of others as in
    [N, C, H, W] (up to 32 classes, many positions of up to 256 if k <= 8, read where they are; others are copied once into rows)."""
    dim = _check(logits, dim, temperature)
    C = logits.shape[dim]
    if not 1 <= k <= min(MAX_K, C):
        raise ValueError(f"k has to be between 1 and min({MAX_K}, {C} classes), got {k}")
    z = logits.detach() if logits.requires_grad else logits
    if not z.is_cuda or z.numel() == 0:
        return _host_top(z.detach(), k, dim, temperature)            # detached from a forward-mode derivative as well
    before, behind = z.shape[:dim], z.shape[dim + 1:]
    z, outer, C, inner, ld, moved = _canonical(z.float() if z.dtype == torch.float16 else z, dim, k)
    device, rest = z.device, before + behind
    kept = rest + (k,) if moved else before + (k,) + behind
    values = torch.empty(kept, dtype=z.dtype, device=device)
    indices = torch.empty(kept, dtype=torch.int32, device=device)
    lse = torch.empty(rest, dtype=torch.float32, device=device)
    dev, st = _env(z)
    with ops._streamed("top logits", z.numel() * z.element_size()):
        call("segk_top_logits", z.data_ptr(), dt(z.dtype), outer, C, inner, ld, k, temperature, values.data_ptr(), indices.data_ptr(),
             lse.data_ptr(), dev, st)
    if moved:
        values, indices = values.movedim(-1, dim), indices.movedim(-1, dim)
    return TopLogits(values if z.dtype == logits.dtype else values.to(logits.dtype), indices, lse)


class _DistillFn(torch.autograd.Function):
    """(student logits, target) -> loss.  Where a scalar's gradient will be wanted, the forward pass writes it for an upstream
    gradient of 1 while the row is still in registers; the backward pass hands it over, recomputed only if upstream is not 1.  That needs
    one forward pass for each backward pass: where only one of them is captured into a graph, or each into its own, a replayed backward
    pass would find what an earlier replay left, so it computes a gradient of its own."""

    @staticmethod
    def forward(ctx, logits, values, indices, lse, dim, temperature, weight, reduction, want_grad):
        z, outer, C, inner, ld, moved = _canonical(logits.float() if logits.dtype == torch.float16 else logits, dim)
        k = values.shape[dim]
        if moved:
            values, indices = values.movedim(dim, -1), indices.movedim(dim, -1)
        values = values if values.is_contiguous() else values.contiguous()
        indices = indices if indices.is_contiguous() else indices.contiguous()
        lse = lse if lse is None or lse.is_contiguous() else lse.contiguous()
        shape = logits.shape
        meta = (outer, C, inner, ld, moved, k, dim, float(temperature), float(weight), reduction, shape, logits.dtype)
        each = reduction == "none"
        out = torch.empty(shape[:dim] + shape[dim + 1:] if each else (), dtype=torch.float32, device=z.device)
        dz = _DistillFn._gradient(meta, z) if want_grad and not each else None
        # a workspace of its own for every call: launches on other streams and replays of captured graphs never share one
        ws = torch.empty(query("segk_distill_workspace", outer, C, inner), dtype=torch.uint8, device=z.device)
        args = _DistillFn._launch(meta, z, values, indices, lse, None, MEAN if reduction == "mean" else 0, None if each else out, out if each else None, dz, ws)
        if want_grad:
            # the gradient among them, as large as the logits: offloading and recomputation (hooks on saved tensors) get hold of it
            ctx.save_for_backward(z, values, indices, lse, dz, None if each else ws)
            ctx.meta, ctx.first, ctx.args, ctx.stride, ctx.capture = meta, dz is not None, args, z.stride(), query("segk_capture_id", args[23])
        return out

    @staticmethod
    def _gradient(meta, z):
        """Memory for dlogits, [outer][C][inner] (rows with the classes last if they were moved), in the caller's shape."""
        moved, dim, shape = meta[4], meta[6], meta[10]
        return torch.empty(shape[:dim] + shape[dim + 1:] + (shape[dim],) if moved else shape, dtype=z.dtype, device=z.device)

    @staticmethod
    def _launch(meta, z, values, indices, lse, upstream, flags, loss, each, dz, ws):
        outer, C, inner, ld, moved, k, dim, T, weight, reduction, shape, in_dtype = meta
        p = ops._p
        dev, st = _env(z)
        args = [z.data_ptr(), dt(z.dtype), outer, C, inner, ld, values.data_ptr(), dt(values.dtype), indices.data_ptr(), indices.element_size(),
                p(lse), k, T, weight, flags, p(upstream), p(loss), p(each), p(dz), C * inner, ws.data_ptr(), ws.numel(), dev, st]
        with ops._streamed("distillation loss", z.numel() * z.element_size() * (2 if dz is not None else 1)):
            call("segk_distill", *args)
        return args

    @staticmethod
    def backward(ctx, g):
        # the wrapper only matters where somebody may differentiate again
        return _once(ctx, g) if torch.is_grad_enabled() else _DistillFn._gradients(ctx, g)

    @staticmethod
    def _gradients(ctx, g):
        z, values, indices, lse, dz, ws = ctx.saved_tensors
        outer, C, inner, ld, moved, k, dim, T, weight, reduction, shape, in_dtype = meta = ctx.meta
        first, ctx.first = ctx.first, False                      # handed over once; a second backward pass computes its own
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.float().contiguous()
        args = ctx.args
        if not first or query("segk_capture_id", _env(z)[1]) != ctx.capture or not dz.is_contiguous() or not ws.is_contiguous():
            dz = None
        else:
            dz = dz.data             # what the caller does to its gradient is no change to a saved tensor: that one is not read again
        if z.data_ptr() != args[0] or z.stride() != ctx.stride:   # hooks on saved tensors brought back a copy, maybe in another layout
            z, _, _, _, ld, _ = _canonical(z.reshape(outer, C, inner), 1, keep=True)
            meta = (outer, C, inner, ld) + meta[4:]
            values, indices, lse = (t if t is None else t.contiguous() for t in (values, indices, lse))
            args = None
        if dz is None:
            dz = _DistillFn._gradient(meta, z)
            ws = torch.empty(query("segk_distill_workspace", outer, C, inner), dtype=torch.uint8, device=z.device)
            _DistillFn._launch(meta, z, values, indices, lse, g, EACH if reduction == "none" else MEAN if reduction == "mean" else 0, None, None, dz, ws)
        elif args is None:
            _DistillFn._launch(meta, z, values, indices, lse, g, SKIP | (MEAN if reduction == "mean" else 0), None, None, dz, ws)
        else:
            # the forward pass's arguments once more: this runs in autograd's thread, where every line costs several times its usual time
            args[14] |= SKIP
            args[6], args[8], args[10] = values.data_ptr(), indices.data_ptr(), ops._p(lse)
            args[15], args[16], args[18], args[20], args[23] = g.data_ptr(), None, dz.data_ptr(), ws.data_ptr(), _env(z)[1]
            call("segk_distill", *args)
        if moved:
            dz = dz.movedim(-1, dim)
        return (dz if dz.dtype == in_dtype else dz.to(in_dtype),) + (None,) * 8


_once = torch.autograd.function.once_differentiable(_DistillFn._gradients)


def distill_loss_topk(pred, target, temperature=1.0, reduction="mean", dim=1, weight=1.0):
    """Distillation loss of the student's logits `pred` against a teacher's top logits.

    With q = softmax(pred / T) over all classes along `dim`, a position contributes
        T^2 [ sum_j p_j (log p_j - log q_(i_j)) + r (log r - log R) ]
    where, if target.lse is None, p = softmax(values / T) over the kept entries and r = 0; otherwise p_j = exp(value_j / T - lse) and
    r = 1 - sum p is what the teacher gave to the other classes together, R what the student gives them (`lse` has to be taken at
    the same temperature).  Entries whose index is no class do not exist; a position without entries (padding) has loss 0 and
    gradient 0.  reduction: 'mean' over the positions that have an entry (0 if there are none), 'sum', or 'none' (a map).
    `weight` scales loss and gradient; it costs nothing, where multiplying the returned loss costs another pass over the logits.

    pred: float32, bfloat16 or float16, any strides; target: TopLogits or a tuple (values, indices[, lse]) with float32 / bfloat16 /
    float16 values and int32 / int64 indices.  Differentiable once, backwards (on the CPU in any mode).  Returns float32; the gradient has
    pred's type.  Sums run in float32 (in float64 on the CPU).  log p carries the rounding of the kept lse, 2^-24 |lse|, so logits / T of some thousands leave no exact probabilities.
    Student and teacher differ by d / T in log q where their logits differ by d, and that is known to about 2^-22: loss and
    gradient are good to about T 2^-22 / d of themselves.  Where every class is kept with an lse, the rounding of the lse adds up to
    T^2 2^-22 (1 + |lse|): leave the lse away there."""
    dim = _check(pred, dim, temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError('Reduction parameter unknown.')
    values, indices, lse = target if isinstance(target, TopLogits) else TopLogits(*target)
    shape, C = pred.shape, pred.shape[dim]
    k = values.shape[dim] if values.dim() == pred.dim() else 0
    want = shape[:dim] + (k,) + shape[dim + 1:]
    if values.shape != want or indices.shape != want:
        raise ValueError(f"values and indices need the logits' shape {tuple(shape)} with the kept entries in dimension {dim}, got "
                         f"{tuple(values.shape)} and {tuple(indices.shape)}")
    if not 1 <= k <= min(MAX_K, C):
        raise ValueError(f"between 1 and min({MAX_K}, {C} classes) kept entries are expected, got {k}")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices have to be int32 or int64, got {indices.dtype}")
    if not values.dtype.is_floating_point:
        raise TypeError(f"values of floating point type are expected, got {values.dtype}")
    if lse is not None and (lse.shape != shape[:dim] + shape[dim + 1:] or not lse.dtype.is_floating_point):
        raise ValueError(f"lse has to have the logits' shape without dimension {dim} and a floating point type, got {tuple(lse.shape)} {lse.dtype}")
    device = pred.device
    if values.device != device or indices.device != device or (lse is not None and lse.device != device):
        raise ValueError("logits and target have to be on the same device")
    if any(t is not None and (t.requires_grad or ops.has_tangent(t)) for t in (values, lse)):
        raise ValueError("the target is data: detach the teacher's logits")
    if not pred.is_cuda or pred.numel() == 0:
        return _host_distill(pred, values, indices, lse, dim, temperature, weight, reduction)
    if values.dtype == torch.float16:
        values = values.float()
    dt(torch.float32 if pred.dtype == torch.float16 else pred.dtype), dt(values.dtype)       # refuses what the kernels do not read
    want_grad = torch.is_grad_enabled() and pred.requires_grad
    if lse is not None and lse.dtype != torch.float32:
        lse = lse.float()
    if ops.has_tangent(pred):
        raise NotImplementedError("distill_loss_topk has no forward-mode derivative on the GPU")
    if isinstance(weight, torch.Tensor) and (weight.requires_grad or ops.has_tangent(weight)):
        raise ValueError("weight is a number on the GPU, and gets no derivative: multiply the loss by it, or detach it")
    if not want_grad:                                        # no node to be made (3 us)
        return _DistillFn.forward(None, pred, values, indices, lse, dim, temperature, weight, reduction, False)
    return _DistillFn.apply(pred, values, indices, lse, dim, temperature, weight, reduction, True)


# ------------------------------------------------------------------------------------ host tensors
def _host_top(z, k, dim, temperature):
    w = z.float() if z.dtype in (torch.float16, torch.bfloat16) else z
    if z.numel() == 0:
        shape = z.shape[:dim] + (k,) + z.shape[dim + 1:]
        return TopLogits(z.new_empty(shape), torch.empty(shape, dtype=torch.int32, device=z.device),
                         torch.empty(z.shape[:dim] + z.shape[dim + 1:], dtype=torch.float32, device=z.device))
    indices = torch.sort(w, dim=dim, descending=True, stable=True).indices.narrow(dim, 0, k)
    lse = torch.logsumexp(w / temperature, dim)
    # two-byte types are gathered as integers: torch's gather on the CPU turns their NaNs into other ones
    raw = z.view(torch.int16) if z.element_size() == 2 else z
    return TopLogits(torch.gather(raw, dim, indices).view(z.dtype), indices.to(torch.int32), lse.masked_fill(lse == math.inf, math.nan).float())


def _host_distill(pred, values, indices, lse, dim, T, weight, reduction):
    # in 64 bits: the terms of a row cancel to 1 / T of themselves, and a temperature costs nothing that way
    z = pred.double().movedim(dim, -1) / T
    t = values.movedim(dim, -1).to(z.dtype) / T
    at = indices.movedim(dim, -1).to(torch.int64)
    valid = (at >= 0) & (at < z.shape[-1])
    counted = valid.any(-1)
    z = torch.where(counted.unsqueeze(-1), z, torch.zeros((), dtype=z.dtype))          # unread: NaN there does not matter
    at = torch.where(valid, at, torch.zeros((), dtype=at.dtype))
    minus = torch.tensor(-math.inf, dtype=z.dtype)
    t = torch.where(valid, t, minus)
    logq = torch.log_softmax(z, -1)
    if lse is None:
        top = t.amax(-1, keepdim=True)
        e = torch.where(t == minus, torch.zeros((), dtype=z.dtype), torch.exp(t - top))
        s = e.sum(-1, keepdim=True)
        p = torch.where(s == 0, torch.zeros((), dtype=z.dtype), e / s)
    else:
        p = torch.where(valid, torch.exp(t - lse.to(z.dtype).unsqueeze(-1)), torch.zeros((), dtype=z.dtype))
    term = p * (torch.log(torch.where(p == 0, torch.ones((), dtype=z.dtype), p)) - torch.where(p == 0, torch.zeros((), dtype=z.dtype), torch.gather(logq, -1, at)))
    row = term.sum(-1)
    if lse is not None:
        kept = torch.zeros_like(z, dtype=torch.int32).scatter_add_(-1, at, valid.to(torch.int32)) > 0
        r = 1 - p.sum(-1)
        has = (r > REST_FLOOR) & ~kept.all(-1) & counted
        outside = torch.logsumexp(torch.where(kept & has.unsqueeze(-1), minus, logq), -1)
        r = torch.where(has, r, torch.ones((), dtype=z.dtype))
        row = row + torch.where(has, r * (torch.log(r) - outside), torch.zeros((), dtype=z.dtype))
    row = torch.where(counted, row * (T * T * weight), torch.zeros((), dtype=z.dtype))
    if reduction == "none":
        return row.to(torch.float32 if pred.dtype != torch.float64 else torch.float64)
    total = row.sum()
    total = total / counted.sum().clamp(min=1) if reduction == "mean" else total
    return total.to(torch.float32 if pred.dtype != torch.float64 else torch.float64)
