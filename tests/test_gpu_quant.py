"""4-bit packing, unpacking and the linear layer on packed operands on the GPU against their definitions in 64 bits, and the chain
in which they are used: a 4-bit layer answers, its top logits are kept, a student learns from them."""
import pytest
import torch

from distill_oracle import loss_and_gradient, top
from loss.distill import distill_loss_topk, top_logits
from segk.quant import MXFP4, mxfp4_dequantize, mxfp4_linear, mxfp4_quantize
from test_quant_cpu import forward_mode_is_refused, four_bit

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def matrix(rows, cols, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 1000 + cols)
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 31), (5, 32), (2, 33), (4, 127), (300, 128), (7, 129), (33, 1000), (5, 1664), (1000, 37), (2, 20000)])
def test_packing(rows, cols, dtype):
    x = matrix(rows, cols, dtype)
    host = mxfp4_quantize(x)
    for y in (x.cuda(), torch.nn.functional.pad(x, (1, 2)).cuda()[:, 1:-2], x.t().contiguous().cuda().t()):
        q = mxfp4_quantize(y)
        assert torch.equal(q.codes.cpu(), host.codes) and torch.equal(q.scales.cpu(), host.scales)
    want = four_bit(x)
    for t in (F32, BF16):
        assert torch.equal(mxfp4_dequantize(q, t).cpu().double(), want)


def test_packing_of_every_bfloat16_value():
    """Every finite bf16 value, next to each of several largest values that set its scale; then whole blocks of every value."""
    b = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    b = b[torch.isfinite(b)]
    for top in (1.0, 1.5, 3.9, 2.0 ** -120, 2.0 ** -125, 2.0 ** -126, 2.0 ** -130, 2.0 ** 127, None):
        v = b if top is None else b[b.abs() <= top]
        n = v.numel() // 31 * 31
        last = torch.full((n // 31, 1), 0.0 if top is None else top, dtype=BF16)
        x = torch.cat([v[:n].view(-1, 31), last], 1).contiguous()
        for y in (x, x.float()):
            host, q = mxfp4_quantize(y), mxfp4_quantize(y.cuda())
            assert torch.equal(q.codes.cpu(), host.codes) and torch.equal(q.scales.cpu(), host.scales)
            assert torch.equal(mxfp4_dequantize(q, y.dtype).cpu(), mxfp4_dequantize(host, y.dtype))


def test_non_finite_values_and_zeros():
    x = matrix(6, 200)
    x[0] = 0
    x[1, 40] = float("nan")
    x[2, 199] = float("inf")
    x[3, 64:96] = -0.0
    host, q = mxfp4_quantize(x), mxfp4_quantize(x.cuda())
    assert torch.equal(q.codes.cpu(), host.codes) and torch.equal(q.scales.cpu(), host.scales)
    y = mxfp4_dequantize(q).cpu()
    bad = torch.zeros(6, 200, dtype=torch.bool)
    bad[1, 32:64] = bad[2, 192:] = True
    assert torch.equal(y.isnan(), bad)
    w = mxfp4_quantize(matrix(20, 200).cuda())
    for rows in (slice(0, 6), slice(1, 3)):
        out = mxfp4_linear(x[rows].cuda(), w).cpu()
        assert torch.equal(out.isnan().all(1), bad[rows].any(1)) and torch.equal(out.isnan().any(1), bad[rows].any(1))


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 1664, 1000), (1, 8192, 512), (2, 100, 33), (4, 513, 80), (5, 640, 1030), (8, 4096, 250), (15, 129, 17), (16, 256, 64),
          (17, 300, 65), (33, 1000, 127), (37, 1664, 1000), (64, 384, 128), (65, 2000, 129), (100, 77, 300), (128, 512, 128), (129, 1280, 255), (200, 3000, 100),
          (255, 640, 257), (256, 896, 256), (257, 1152, 513), (300, 64, 2000), (1000, 32, 90), (513, 2048, 512), (2049, 130, 130), (1, 20000, 40), (520, 8192, 300), (4, 20000, 50),
          (2, 300, 5000), (20, 1100, 4500), (3, 2500, 4097),
          # the kernels' borders: more than 512 workgroups of 16 x 16, a side of 64, 128 or 256 with 256 tiles
          (1, 260, 9000), (2, 129, 8200), (33, 300, 4100), (64, 513, 8197), (100, 1000, 1500), (150, 128, 1111), (300, 1100, 777), (512, 100, 256),
          (513, 300, 256), (65, 400, 32773), (129, 200, 33000), (200, 384, 65540), (130, 100, 65283)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(M, K, N, dtype):
    x, w, b = matrix(M, K, dtype), matrix(N, K, seed=1), torch.randn(N, generator=torch.Generator().manual_seed(2))
    qw = mxfp4_quantize(w.cuda())
    a, c = four_bit(x), four_bit(w)
    want, size = a @ c.t() + b.double(), a.abs() @ c.abs().t() + b.double().abs()
    y = mxfp4_linear(x.cuda(), qw, b.cuda())
    # products of two 4-bit values are exact; K additions in fp32, each off by half a step of a partial sum, then one rounding
    tol = (K + 8) * 2.0 ** -24 * size
    assert y.dtype == dtype
    assert bool(((y.cpu().double() - want).abs() <= tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)).all())
    packed = mxfp4_linear(mxfp4_quantize(x.cuda()), qw, b.cuda(), out_dtype=dtype)
    assert torch.equal(packed, y)                                                   # packing on the fly is the same packing
    assert torch.equal(mxfp4_linear(x.cuda(), qw, b.cuda()), y)                     # and the order of the sums is fixed
    plain = mxfp4_linear(torch.nn.functional.pad(x, (3, 1)).cuda()[:, 3:-1], qw, out_dtype=F32)
    assert bool(((plain.cpu().double() - a @ c.t()).abs() <= (K + 8) * 2.0 ** -23 * size).all())


def test_linear_forms():
    w = matrix(70, 300)
    qw, qh = mxfp4_quantize(w.cuda()), mxfp4_quantize(w)
    x = matrix(24, 300, torch.float16)
    y = mxfp4_linear(x.view(2, 3, 4, 300).cuda(), qw)
    assert y.shape == (2, 3, 4, 70) and y.dtype == torch.float16
    host = mxfp4_linear(x, qh, out_dtype=F32)
    torch.testing.assert_close(mxfp4_linear(x.cuda(), qw, out_dtype=F32).cpu(), host, rtol=0, atol=300 * 2.0 ** -23 * float(four_bit(x).abs().max() * four_bit(w).abs().max()) * 30)
    assert mxfp4_linear(x[:0].cuda(), qw).shape == (0, 70)
    moved = MXFP4(qh.codes.cuda(), qh.scales.cuda(), 300)
    assert torch.equal(mxfp4_linear(x.cuda(), moved), mxfp4_linear(x.cuda(), qw))
    assert torch.equal(mxfp4_linear(x.cuda(), qw, torch.ones(70, device="cuda", dtype=BF16), F32), mxfp4_linear(x.cuda(), qw, torch.ones(70, device="cuda"), F32))
    with pytest.raises(ValueError, match="same device"):
        mxfp4_linear(x, qw)
    with pytest.raises(ValueError, match="bias"):
        mxfp4_linear(x.cuda(), qw, torch.zeros(70))
    with pytest.raises(ValueError, match="aligned"):
        MXFP4(torch.empty(70 * 192 + 8, dtype=torch.uint8, device="cuda")[8:].view(70, 192), qw.scales, 300)


def test_rows_behind_the_last_stay_as_they_were():
    """The C entry point writes the M rows and N columns it was asked for and nothing else."""
    from segk import _lib
    M, K, N, ld = 19, 300, 37, 45
    x, qw = matrix(M, K).cuda(), mxfp4_quantize(matrix(N, K).cuda())
    y = torch.full((M + 3, ld), 7.0, device="cuda")
    ws = torch.empty(_lib.query("segk_mxfp4_linear_workspace", M, K, N), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for m in (1, 3, 16, M):
        y.fill_(7.0)
        _lib.call("segk_mxfp4_linear", x.data_ptr(), 0, K, None, None, m, K, qw.codes.data_ptr(), qw.scales.data_ptr(), N, None, y.data_ptr(), 0, ld,
                  ws.data_ptr(), ws.numel(), 0, st)
        assert bool((y[m:] == 7).all()) and bool((y[:, N:] == 7).all()) and torch.equal(y[:m, :N], mxfp4_linear(x[:m], qw))
    z = torch.full((M + 2, K + 5), 7.0, device="cuda")
    q = mxfp4_quantize(x)
    _lib.call("segk_mxfp4_dequantize", 0, q.codes.data_ptr(), q.scales.data_ptr(), M, K, z.data_ptr(), K + 5, 0, st)
    assert bool((z[M:] == 7).all()) and bool((z[:, K:] == 7).all()) and torch.equal(z[:M, :K], mxfp4_dequantize(q))


def test_many_rows_few_outputs():
    """More rows than a grid dimension of 65535 workgroups of 16 covers: pixels through a 1x1 layer."""
    M, K, N = 1_200_000, 32, 24
    x, w = matrix(64, K, BF16), matrix(N, K)
    y = mxfp4_linear(x.cuda().repeat(M // 64, 1), mxfp4_quantize(w.cuda()))
    want = four_bit(x) @ four_bit(w).t()
    assert y.shape == (M, N) and bool((y.view(-1, 64, N) == y[:64]).all())
    size = four_bit(x).abs() @ four_bit(w).abs().t()
    assert bool(((y[:64].cpu().double() - want).abs() <= (K + 8) * 2.0 ** -24 * size + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -10)).all())


@pytest.mark.parametrize("M,K,N", [(2, 700, 900), (40, 700, 900), (40, 700, 9000), (1, 300, 9000), (2050, 256, 2052), (4096, 384, 4100)])
def test_every_kernel_in_a_captured_graph(M, K, N):
    """The kernels for few rows and every tile size, captured without a call before and replayed on new inputs."""
    qw = mxfp4_quantize(matrix(N, K).cuda())
    x = matrix(M, K, BF16).cuda()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        y = mxfp4_linear(x, qw)
    for seed in (1, 2, 3):
        new = matrix(M, K, BF16, seed=seed).cuda()
        x.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, mxfp4_linear(new, qw))


def test_chain_other_stream_and_captured_graph():
    """Teacher's last layer in 4 bits -> its top logits -> loss and gradient of a student's logits, eager, on another stream and as
    two captured graphs."""
    M, K, N = 96, 700, 1500
    qw, b = mxfp4_quantize((matrix(N, K) / 26).cuda()), torch.zeros(N, device="cuda")

    def chain(features, student):
        teacher = mxfp4_linear(features, qw, b)
        target = top_logits(teacher, 8, temperature=2.0)
        loss = distill_loss_topk(student, target, temperature=2.0)
        return teacher, *target, loss, torch.autograd.grad(loss, student)[0]
    f, s = matrix(M, K).cuda(), torch.randn(M, N, device="cuda").requires_grad_()
    want = [t.detach().clone() for t in chain(f, s)]
    a, c = four_bit(f.cpu()), four_bit(matrix(N, K) / 26)
    assert bool(((want[0].cpu().double() - a @ c.t()).abs() <= K * 2.0 ** -23 * (a.abs() @ c.abs().t())).all())
    # each link against its definition, with the bounds derived in distill_oracle.py
    values, indices = top(want[0].cpu(), 8)
    assert torch.equal(want[1].cpu(), values) and torch.equal(want[2].cpu(), indices)
    lse = torch.logsumexp(want[0].cpu().double() / 2, 1)
    assert bool(((want[3].cpu().double() - lse).abs() <= 2.0 ** -21 * (8 + 3 * want[0].cpu().double().abs().amax(1) / 2)).all())
    loss, grad, counted, lerr, gerr = loss_and_gradient(s.detach().cpu(), values, indices, want[3].cpu(), 2.0)
    assert bool(counted.all()) and abs(float(want[4]) - float(loss.mean())) <= float(lerr.mean()) + 2.0 ** -23 * float(loss.mean())
    assert bool(((want[5].cpu().double() - grad / M).abs() <= (gerr + 2.0 ** -21 * grad.abs()) / M).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.detach().clone() for t in chain(f, s)]
        fs, ss = f.clone(), s.detach().clone().requires_grad_()
        chain(fs, ss)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(fs, ss)
        graphs.append((g, out))
    for seed in (1, 2, 3):
        nf, ns = matrix(M, K, seed=seed).cuda(), torch.randn(M, N, device="cuda").requires_grad_()
        with torch.no_grad():
            fs.copy_(nf)
            ss.copy_(ns)
        want = [t.detach().clone() for t in chain(nf, ns)]
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c.detach()) for a, c in zip(want, out))


def test_forward_mode():
    forward_mode_is_refused("cuda")
