"""Microscaled 4-bit floating point: packing, unpacking and the linear layer on packed operands, over the C ABI (segk_mxfp4_*), for
serving linear layers (nn.Linear, 1x1 convolutions over channels-last pixels) whose trained weights are held in 4 bits.  Functions for a
caller's own layers: the networks of models/ run theirs in fp32.  CPU tensors are served by the same definitions in torch ops (`_host_*`)."""
import math

import torch

from . import ops
from ._lib import call, query
from .ops import _env, dt

GROUP, SLICE = 32, 128      # values that share a scale; values of one slice of a packed row


class MXFP4:
    """A packed matrix [rows, cols]: `codes` uint8 [rows, S * 64] with two values a byte (even column in the low half), `scales`
    uint8 [S, rows, 4], S = ceil(cols / 128); a scale byte b stands for 2^(b - 127), 255 for NaN.  Rows are padded with zeros."""
    __slots__ = ("codes", "scales", "cols")

    def __init__(self, codes, scales, cols):
        slices = -(-int(cols) // SLICE)
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales are uint8 tensors")
        if cols < 1 or codes.dim() != 2 or codes.shape[1] != slices * (SLICE // 2) or scales.shape != (slices, codes.shape[0], 4):
            raise ValueError(f"{cols} columns need codes [rows, {slices * (SLICE // 2)}] and scales [{slices}, rows, 4], got "
                             f"{tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales have to be on the same device")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales have to be contiguous")
        if codes.is_cuda and (codes.data_ptr() % 16 or scales.data_ptr() % 4):
            raise ValueError("codes have to be 16-byte aligned and scales 4-byte aligned")
        self.codes, self.scales, self.cols = codes, scales, int(cols)

    @classmethod
    def _of(cls, codes, scales, cols):
        """What mxfp4_quantize allocated: its shapes need no check."""
        q = object.__new__(cls)
        q.codes, q.scales, q.cols = codes, scales, cols
        return q

    rows = property(lambda s: s.codes.shape[0])
    shape = property(lambda s: (s.codes.shape[0], s.cols))
    device = property(lambda s: s.codes.device)

    def to(self, device):
        return MXFP4(self.codes.to(device), self.scales.to(device), self.cols)

    def row_scales(self):
        """The scale bytes as [rows, S * 4]: one for each 32 columns, in order."""
        return self.scales.transpose(0, 1).reshape(self.rows, self.scales.shape[0] * 4)

    def __repr__(self):
        return f"MXFP4({self.rows} x {self.cols}, {self.device})"


def _rows(x, what):
    """(x as a 2-D matrix with contiguous rows, its leading dimension); fp16 is read as fp32, which holds its values."""
    if not isinstance(x, torch.Tensor) or not x.dtype.is_floating_point or x.dim() < 1:
        raise TypeError(f"{what} has to be a floating point tensor with at least one dimension")
    if x.shape[-1] < 1:
        raise ValueError(f"{what} has no columns")
    if x.requires_grad:
        if torch.is_grad_enabled():
            raise RuntimeError(f"{what} requires a gradient and 4-bit rounding has none: call under torch.no_grad() or detach it")
        x = x.detach()
    if ops.has_tangent(x):
        raise RuntimeError(f"{what} carries a forward-mode derivative and 4-bit rounding has none: detach it")
    if x.dtype == torch.float16:
        x = x.float()
    dt(x.dtype)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    rows, cols = x.shape
    if x.is_contiguous():
        return x, cols
    if cols > 1 and x.stride(1) != 1 or rows > 1 and x.stride(0) < cols:
        x = x.contiguous()
    return x, (x.stride(0) if rows > 1 else cols)


def mxfp4_quantize(x):
    """Pack a float32 / bfloat16 / float16 matrix (leading dimensions are flattened, rows may be strided) as MXFP4: for each 32
    values of a row the scale 2^e, e = floor(log2(max |x|)) - 2, and x / 2^e to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to
    the even code, beyond 6 to 6.  A NaN or an infinity makes its 32 values NaN."""
    x, ld = _rows(x, "x")
    rows, cols = x.shape
    if not x.is_cuda:
        return MXFP4(*_host_quantize(x), cols)
    slices, device = -(-cols // SLICE), x.device
    codes = torch.empty((rows, slices * (SLICE // 2)), dtype=torch.uint8, device=device)
    scales = torch.empty((slices, rows, 4), dtype=torch.uint8, device=device)
    if rows:
        dev, st = _env(x)
        with ops._streamed("4-bit packing", x.numel() * (x.element_size() + 0.53125)):
            call("segk_mxfp4_quantize", dt(x.dtype), x.data_ptr(), ld, rows, cols, codes.data_ptr(), scales.data_ptr(), dev, st)
    return MXFP4._of(codes, scales, cols)


def mxfp4_dequantize(q, dtype=torch.float32):
    """The matrix that `q` stands for, exact in float32 and in bfloat16."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"float32 or bfloat16 hold these values exactly, not {dtype}")
    rows, cols = q.shape
    if not q.codes.is_cuda:
        return _host_dequantize(q).to(dtype)
    y = torch.empty((rows, cols), dtype=dtype, device=q.codes.device)
    if rows:
        dev, st = _env(q.codes)
        with ops._streamed("4-bit unpacking", y.numel() * (y.element_size() + 0.53125)):
            call("segk_mxfp4_dequantize", dt(dtype), q.codes.data_ptr(), q.scales.data_ptr(), rows, cols, y.data_ptr(), cols, dev, st)
    return y


def mxfp4_linear(x, w, bias=None, out_dtype=None):
    """x w^T + bias with both operands in 4 bits, float32 accumulation: the serving form of nn.Linear with packed weights.

    x: [..., K] float32 / bfloat16 / float16, packed on the fly exactly as mxfp4_quantize does, or an MXFP4; w: MXFP4 [N, K]; bias: [N].
    Returns [..., N] in out_dtype (default: x's type, float32 for a packed x).  Not differentiable."""
    if not isinstance(w, MXFP4):
        raise TypeError("w has to be an MXFP4 (mxfp4_quantize packs a weight)")
    N, K = w.shape
    packed = isinstance(x, MXFP4)
    if out_dtype is None:
        out_dtype = torch.float32 if packed else x.dtype
    if out_dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"out_dtype has to be float32, bfloat16 or float16, not {out_dtype}")
    if packed:
        lead, M, kx = (x.rows,), x.rows, x.cols
    else:
        lead, kx = x.shape[:-1], x.shape[-1]
        x, ld = _rows(x, "x")
        M = x.shape[0]
    if kx != K:
        raise ValueError(f"x has {kx} columns and w {K}")
    device = w.codes.device
    if x.device != device:
        raise ValueError("x and w have to be on the same device")
    if bias is not None:
        if bias.shape != (N,) or bias.device != device or not bias.dtype.is_floating_point:
            raise ValueError(f"bias has to be a floating point tensor [{N}] on the device of w")
        if bias.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("bias requires a gradient: call under torch.no_grad() or detach it")
        if ops.has_tangent(bias):
            raise RuntimeError("bias carries a forward-mode derivative: detach it")
        if bias.dtype != torch.float32 or bias.requires_grad or not bias.is_contiguous():
            bias = bias.detach().float().contiguous()
    if not w.codes.is_cuda:
        xq = _host_dequantize(x if packed else MXFP4(*_host_quantize(x), K))
        y = xq @ _host_dequantize(w).t()
        return (y if bias is None else y + bias).to(out_dtype).reshape(lead + (N,))
    y = torch.empty((M, N), dtype=torch.float32 if out_dtype == torch.float16 else out_dtype, device=device)
    if M and N:
        nbytes = 0 if packed else query("segk_mxfp4_linear_workspace", M, K, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None     # one for every call: nothing is shared
        dev, st = _env(w.codes)
        with ops._streamed("4-bit linear", M * K * (0.53125 if packed else x.element_size()) + N * K * 0.53125 + M * N * y.element_size()):
            call("segk_mxfp4_linear", None if packed else x.data_ptr(), 0 if packed else dt(x.dtype), 0 if packed else ld,
                 x.codes.data_ptr() if packed else None, x.scales.data_ptr() if packed else None, M, K, w.codes.data_ptr(), w.scales.data_ptr(), N,
                 ops._p(bias), y.data_ptr(), dt(y.dtype), N, ops._p(ws), nbytes, dev, st)
    if y.dtype != out_dtype:
        y = y.to(out_dtype)
    return y if len(lead) == 1 else y.reshape(lead + (N,))


# ------------------------------------------------------------------------------------ host tensors
def _host_quantize(x):
    rows, cols = x.shape
    slices = -(-cols // SLICE)
    v = torch.nn.functional.pad(x.float(), (0, slices * SLICE - cols)).view(rows, slices * 4, GROUP)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.frexp(top).exponent - 3
    e = torch.where((top > 0) & ~bad, e, -127).clamp(-127, 127)
    y = torch.ldexp(v.abs().double(), -e.unsqueeze(-1))
    y = torch.where(bad.unsqueeze(-1), 0.0, y)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp(max=6)                       # torch.round: ties to even multiples of the step
    code = torch.where(y < 2, 2 * y, torch.where(y < 4, y + 2, y / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v) & ~bad.unsqueeze(-1)).to(torch.uint8) << 3).view(rows, slices * SLICE)
    scale = torch.where(bad, 255, e + 127).to(torch.uint8).view(rows, slices, 4)
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), scale.transpose(0, 1).contiguous()


def _host_dequantize(q):
    width = q.codes.shape[1] * 2
    code = torch.stack([q.codes & 15, q.codes >> 4], -1).view(q.rows, width)
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    v = torch.cat([table, -table])[code.long()].view(q.rows, width // GROUP, GROUP)
    s = q.row_scales()
    f = torch.where(s == 255, math.nan, torch.ldexp(torch.ones(()), s.to(torch.int32) - 127))
    return (v * f.unsqueeze(-1)).view(q.rows, width)[:, :q.cols].contiguous()
