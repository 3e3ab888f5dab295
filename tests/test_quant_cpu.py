"""4-bit packing and the linear layer on packed operands: definitions and refusals on host tensors, refusals of the C entry points."""
import pytest
import torch

from segk.quant import MXFP4, mxfp4_dequantize, mxfp4_linear, mxfp4_quantize

TABLE = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def four_bit(x):
    """[rows, cols] as the definition packs it, in 64 bits: nearest table entry by distance, ties to the even code."""
    x = x.double()
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % 32)).view(rows, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2
    unit = torch.exp2(torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127))
    d = ((v / unit).abs().unsqueeze(-1) - TABLE).abs()
    d = d + torch.tensor([0, 1, 0, 1, 0, 1, 0, 1]) * 1e-9            # of two at the same distance the even one
    y = TABLE[d.argmin(-1)] * torch.sign(v) * unit
    return y.view(rows, -1)[:, :cols]


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (4, 33), (5, 128), (2, 129), (7, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_host_packing_is_the_definition(rows, cols, dtype):
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    q = mxfp4_quantize(x)
    assert q.shape == (rows, cols) and q.codes.shape == (rows, -(-cols // 128) * 64) and q.scales.shape == (-(-cols // 128), rows, 4)
    assert torch.equal(mxfp4_dequantize(q).double(), four_bit(x))
    assert torch.equal(mxfp4_dequantize(mxfp4_quantize(mxfp4_dequantize(q))), mxfp4_dequantize(q))       # packing keeps what is packed


def test_ties_saturation_zeros_and_non_finite_values():
    x = torch.zeros(4, 32)
    x[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, 7.5])
    x[2, 3] = float("nan")
    x[3, 4] = float("-inf")
    q = mxfp4_quantize(x)
    assert mxfp4_dequantize(q)[0, :10].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 0.0, 6.0]
    assert q.row_scales()[:, 0].tolist() == [127, 0, 255, 255] and not mxfp4_dequantize(q)[1].any() and mxfp4_dequantize(q)[2:].isnan().all()


def test_host_linear_and_its_shapes():
    g = torch.Generator().manual_seed(0)
    w, x, b = torch.randn(9, 200, generator=g), torch.randn(2, 3, 200, generator=g), torch.randn(9, generator=g)
    q = mxfp4_quantize(w)
    y = mxfp4_linear(x, q, b)
    want = four_bit(x.view(6, 200)) @ four_bit(w).t() + b.double()
    assert y.shape == (2, 3, 9) and float((y.view(6, 9).double() - want).abs().max()) < 200 * 2.0 ** -24 * 36 * float(want.abs().max() + 1)
    assert mxfp4_linear(mxfp4_quantize(x), q).shape == (6, 9) and mxfp4_linear(x.bfloat16(), q).dtype == torch.bfloat16
    assert mxfp4_linear(x[:0], q).shape == (0, 3, 9) and mxfp4_quantize(torch.zeros(0, 5)).shape == (0, 5)


def test_refusals():
    w = mxfp4_quantize(torch.randn(4, 40))
    x = torch.randn(3, 40)
    with pytest.raises(TypeError, match="MXFP4"):
        mxfp4_linear(x, torch.randn(4, 40))
    with pytest.raises(ValueError, match="columns"):
        mxfp4_linear(torch.randn(3, 41), w)
    with pytest.raises(ValueError, match="bias"):
        mxfp4_linear(x, w, torch.zeros(5))
    with pytest.raises(RuntimeError, match="gradient"):
        mxfp4_linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="gradient"):
        mxfp4_linear(x, w, torch.zeros(4, requires_grad=True))
    with pytest.raises(RuntimeError, match="gradient"):
        mxfp4_quantize(torch.zeros(2, 3, requires_grad=True))
    with torch.no_grad():
        mxfp4_quantize(torch.zeros(2, 3, requires_grad=True))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        mxfp4_quantize(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(TypeError, match="floating"):
        mxfp4_quantize(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="no columns"):
        mxfp4_quantize(torch.zeros(2, 0))
    with pytest.raises(TypeError, match="exactly"):
        mxfp4_dequantize(w, torch.float16)
    with pytest.raises(TypeError, match="out_dtype"):
        mxfp4_linear(x, w, out_dtype=torch.float64)
    with pytest.raises(TypeError, match="uint8"):
        MXFP4(w.codes.int(), w.scales, 40)
    for codes, scales, cols in ((w.codes[:, :32], w.scales, 40), (w.codes, w.scales[:, :3], 40), (w.codes, w.scales, 129), (w.codes, w.scales, 0)):
        with pytest.raises(ValueError, match="columns need"):
            MXFP4(codes, scales, cols)
    with pytest.raises(ValueError, match="contiguous"):
        MXFP4(w.codes.t().contiguous().t(), w.scales, 40)
    with pytest.raises(ValueError, match="same device"):
        MXFP4(w.codes, w.scales.to("meta"), 40)


def test_c_entry_points_refuse_bad_arguments_without_a_gpu():
    from segk import _lib
    F32, BF16 = _lib.SEGK_F32, _lib.SEGK_BF16
    base = dict(dt=F32, x=4096, ld=64, rows=4, cols=64, c=4096, s=4096, d=0, st=None)
    for kw, text in ((dict(dt=5), "dtype"), (dict(x=None), "null"), (dict(rows=0), "shape"), (dict(cols=0), "shape"), (dict(cols=1 << 30, ld=1 << 30), "shape"),
                     (dict(ld=63), "ld"), (dict(x=4098), "aligned"), (dict(c=None), "null"), (dict(c=4104), "16-byte"), (dict(s=4098), "4-byte")):
        with pytest.raises(_lib.SegkError, match=text):
            _lib.call("segk_mxfp4_quantize", *{**base, **kw}.values())
        o = {**base, **kw}
        with pytest.raises(_lib.SegkError, match=text):
            _lib.call("segk_mxfp4_dequantize", o["dt"], o["c"], o["s"], o["rows"], o["cols"], o["x"], o["ld"], 0, None)
    base = dict(x=4096, dt=BF16, ld=64, xc=None, xs=None, M=4, K=64, wc=4096, ws=4096, N=8, b=None, y=4096, ydt=F32, ldy=8, ws_=4096, wsb=1 << 20, d=0, st=None)
    for kw, text in ((dict(x=None), "either"), (dict(xc=4096), "either"), (dict(M=0), "shape"), (dict(K=0), "shape"), (dict(N=0), "shape"), (dict(wc=None), "null"),
                     (dict(wc=4100), "16-byte"), (dict(y=None), "null"), (dict(ydt=3), "dtype"), (dict(ldy=7), "ld"), (dict(M=5, wsb=16), "SEGK_EWORKSPACE"),
                     (dict(M=5, ws_=None), "SEGK_EWORKSPACE"), (dict(M=5, ws_=4104), "16-byte"), (dict(x=None, xc=4096), "null"), (dict(dt=2), "dtype"), (dict(ld=10), "ld")):
        with pytest.raises(_lib.SegkError, match=text):
            _lib.call("segk_mxfp4_linear", *{**base, **kw}.values())
    assert _lib.query("segk_mxfp4_codes_bytes", 3, 129) == 3 * 128 and _lib.query("segk_mxfp4_scales_bytes", 3, 129) == 24
    assert _lib.query("segk_mxfp4_codes_bytes", 0, 5) == 0


def test_more_outputs_than_one_launch_holds_are_refused_without_a_gpu():
    """A launch has fewer than 2^32 threads, 512 for each 256 x 256 tile; refused before anything is launched."""
    from segk import _lib
    for M, N in ((1 << 27, 1 << 27), (256 * (1 << 12), 256 * (1 << 11)), ((1 << 28) - 1, 65281)):
        for packed in (False, True):
            with pytest.raises(_lib.SegkError, match="too many outputs"):
                _lib.call("segk_mxfp4_linear", None if packed else 4096, _lib.SEGK_BF16, 64, 4096 if packed else None, 4096 if packed else None, M, 64, 4096, 4096, N,
                          None, 4096, _lib.SEGK_BF16, N, 4096, 1 << 60, 0, None)


def forward_mode_is_refused(device):
    import torch.autograd.forward_ad as fwd
    w = mxfp4_quantize(torch.randn(4, 40, device=device))
    x, b = torch.randn(3, 40, device=device), torch.zeros(4, device=device)
    want = mxfp4_linear(x, w, b)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: mxfp4_quantize(dual), lambda: mxfp4_linear(dual, w), lambda: mxfp4_linear(x, w, fwd.make_dual(b, torch.ones_like(b)))):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call()
        assert torch.equal(mxfp4_linear(dual.detach(), w, b), want)


def test_forward_mode_is_refused():
    """4-bit rounding has no derivative: a dual number is refused like a tensor that requires a gradient, also under no_grad."""
    forward_mode_is_refused("cpu")
