"""Top logits and the distillation loss on the GPU against the definitions in 64 bits (tests/distill_oracle.py, which also derives
the error bounds)."""
import math

import pytest
import torch

from distill_oracle import cancellation_bounds, half_step, loss_and_gradient, top
from loss.distill import TopLogits, distill_loss_topk, top_logits
from test_distill_cpu import nan_among_the_values

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def problem(P, V, k, seed=0, dtype=F32, ignored=0.0, T=1.0, values_dtype=None):
    g = torch.Generator().manual_seed(seed)
    t = (2.5 * torch.randn(P, V, generator=g)).to(dtype)
    z = (0.5 * t.float() + 1.5 * torch.randn(P, V, generator=g)).to(dtype)
    values, indices = torch.topk(t.float(), k, 1)
    lse = torch.logsumexp(t.float() / T, 1)
    indices = indices.to(torch.int32)
    if ignored:
        indices[torch.rand(P, generator=g) < ignored] = -1
    return z, values.to(values_dtype or dtype), indices, lse


def check(z, values, indices, lse, T, weight=1.0, dim=1, upstream=1.0, cuda=None, gtol_extra=0.0):
    """All reductions, loss and gradient, of [P, V] problems; `cuda` turns the host logits into the device tensor to be used."""
    cuda = cuda or (lambda x: x.cuda())
    loss, grad, counted, lerr, gerr = loss_and_gradient(z, values, indices, lse, T, weight)
    n = max(1, int(counted.sum()))
    target = TopLogits(values.cuda(), indices.cuda(), None if lse is None else lse.cuda())
    eps = half_step(z.dtype) + gtol_extra
    for reduction, scale in (("mean", 1.0 / n), ("sum", 1.0), ("none", 1.0)):
        x = cuda(z).detach().requires_grad_()
        got = distill_loss_topk(x, target, temperature=T, reduction=reduction, weight=weight, dim=dim)
        assert got.dtype == F32
        want, tol = (loss, lerr) if reduction == "none" else (loss.sum() * scale, lerr.sum() * scale)
        err = (got.detach().double().cpu() - want).abs()
        assert bool((err <= tol + 2.0 ** -23 * want.abs()).all()), (reduction, float(err.max()), float(tol.max()))
        (got * upstream).sum().backward()
        g = x.grad.double().cpu()
        # the gradient's rounding to its type; once more to fp32 and for the scale factors before it
        bound = scale * abs(upstream) * (gerr + (eps + 2.0 ** -21) * grad.abs())
        err = (g - grad * (scale * upstream)).abs()
        # below the smallest normal number the type's step is fixed, tiny * eps (fp16: 2^-14 * 2^-10 = 2^-24): half of it
        fixed = max(2.0 ** -133, torch.finfo(z.dtype).tiny * half_step(z.dtype))
        assert x.grad.dtype == z.dtype and bool((err <= bound + fixed).all()), (reduction, float((err - bound).max()))
        with torch.no_grad():
            again = distill_loss_topk(x, target, temperature=T, reduction=reduction, weight=weight, dim=dim)
        assert torch.equal(again, got.detach())


# every tier of the rows (one wave, 256 and 1024 threads, in registers or read twice), rows that end inside a 16-byte piece, and the
# thread-per-position kernel (up to 8 classes)
WIDTHS = [1, 2, 3, 5, 8, 9, 31, 64, 80, 127, 255, 256, 257, 512, 513, 1000, 1025, 2047, 4096, 4097, 8191, 8193, 16383, 16385, 32767, 32769, 65535, 65537, 131071, 131073]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", WIDTHS)
def test_rows(V, dtype):
    k = min(V, 1 + V % 13, 64)
    z, values, indices, lse = problem(5, V, k, seed=V, dtype=dtype, ignored=0.25, T=2.0)
    check(z, values, indices, lse, 2.0)
    check(z, values, indices, None, 1.0, weight=0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [4100, 8193, 16385, 32769, 65537, 131073])
def test_many_long_rows(V, dtype):
    """Rows that one workgroup each works on (few rows are shared by several): every row of a group of five again and again."""
    z, values, indices, lse = problem(5, V, 6, seed=V, dtype=dtype, T=2.0)
    indices[3] = -1
    loss, grad, counted, lerr, gerr = loss_and_gradient(z, values, indices, lse, 2.0)
    again = lambda t: t.repeat(40, *([1] * (t.dim() - 1))).cuda()   # noqa: E731
    x = again(z).requires_grad_()
    got = distill_loss_topk(x, TopLogits(again(values), again(indices), again(lse)), temperature=2.0, reduction="none")
    got.sum().backward()
    assert bool(((got.detach().double().cpu().view(40, 5) - loss).abs() <= lerr + 2.0 ** -23 * loss).all())
    # (rows of odd length begin at other places of a 16-byte piece and add up in another order: within the bounds, not to the bit)
    bound, grad = (gerr + (half_step(dtype) + 2.0 ** -21) * grad.abs()).cuda(), grad.cuda()
    assert bool(((x.grad.view(40, 5, V).double() - grad).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,k", [(70, 64), (64, 64), (5000, 64), (40, 40), (6, 6)])
def test_many_entries(V, k, dtype):
    z, values, indices, lse = problem(6, V, k, seed=k, dtype=dtype, T=1.5)
    check(z, values, indices, lse, 1.5)
    check(z, values, indices, None, 1.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [6, 100, 3001])
def test_entries_that_repeat_or_do_not_exist(V, dtype):
    z, values, indices, lse = problem(6, V, 5, seed=V, dtype=dtype)
    indices[0, :3] = indices[0, 3]                       # four entries of one class
    indices[1] = torch.tensor([-1, V, -(1 << 31), (1 << 31) - 1, 2], dtype=torch.int32)
    indices[2] = indices[2, 0]
    indices[3, 1:] = V
    indices[4] = -7
    lse = lse + 2.0                                      # keeps the sum of the p below 1 where entries repeat
    check(z, values, indices, lse, 1.0)
    check(z, values, indices, None, 1.0)
    wide = indices.to(torch.int64)
    wide[5, 0] += 1 << 32                                # no class, although its low half is one
    check(z, values, wide, lse, 1.0)
    values[0, 0] = -math.inf                             # a kept class without mass
    values[2] = torch.finfo(dtype).min
    check(z, values, indices, lse, 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [7, 90, 1500, 70001])
def test_masked_logits(V, dtype):
    z, values, indices, lse = problem(6, V, 4, seed=V, dtype=dtype)
    kept = torch.zeros(6, V, dtype=torch.bool).scatter_(1, indices.long(), True)
    g = torch.Generator().manual_seed(1)
    mask = (torch.rand(6, V, generator=g) < 0.5) & ~kept
    mask[:, (~kept).float().argmax(1)] = False           # one class outside stays
    mask &= ~kept
    for low in (-math.inf, float(torch.finfo(dtype).min)):
        y = torch.where(mask, torch.tensor(low, dtype=dtype), z)
        # the lowest value takes no part in sums; the bounds go by the logits that do
        loss, grad, counted, lerr, gerr = loss_and_gradient(torch.where(mask, torch.tensor(-math.inf, dtype=dtype), z), values, indices, lse, 1.0)
        x = y.cuda().requires_grad_()
        got = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()), reduction="none")
        assert bool(((got.detach().double().cpu() - loss).abs() <= lerr + 2.0 ** -23 * loss).all())
        got.sum().backward()
        err = (x.grad.double().cpu() - grad).abs()
        assert bool((err <= gerr + (half_step(dtype) + 2.0 ** -21) * grad.abs()).all()) and not x.grad.cpu()[mask].any()
    # everything outside the kept classes masked: the student gives them nothing
    y = torch.where(kept, z, torch.tensor(-math.inf, dtype=dtype))
    check(y, values, indices, None, 1.0)
    x = y.cuda()
    got = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()), reduction="none")
    assert torch.isinf(got).all()                        # the teacher gave them something
    # one NaN or infinity spoils its own row only
    for bad in (math.nan, math.inf):
        y = z.clone()
        y[2, (~kept[2]).float().argmax()] = bad
        x = y.cuda().requires_grad_()
        got = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()), reduction="none")
        got.sum().backward()
        others = [i for i in range(6) if i != 2]
        assert torch.isnan(got[2]) and torch.isnan(x.grad[2]).any() and torch.isfinite(got[others]).all() and torch.isfinite(x.grad[others]).all()


def test_rows_without_entries_are_not_read():
    z, values, indices, lse = problem(4, 1000, 4)
    z[1] = math.nan
    indices[1] = -1
    x = z.cuda().requires_grad_()
    loss = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()))
    loss.backward()
    assert torch.isfinite(loss) and not x.grad[1].any() and x.grad[0].any()
    x = z.cuda().requires_grad_()
    loss = distill_loss_topk(x, TopLogits(values.cuda(), torch.full_like(indices, 1000).cuda(), None))
    loss.backward()
    assert float(loss.detach()) == 0 and not x.grad.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,side,k", [(2, 4, 8, 2), (1, 3, 7, 3), (2, 8, 6, 4), (3, 7, 12, 2), (1, 16, 5, 5), (2, 21, 9, 3), (1, 32, 4, 32), (2, 33, 3, 4), (1, 2, 64, 1), (1, 1, 6, 1)])
def test_planes(N, C, side, k, dtype):
    z, values, indices, lse = problem(N * side * side, C, k, seed=C, dtype=dtype, ignored=0.2, T=2.0)
    planes = lambda t: t.view(N, side, side, -1).permute(0, 3, 1, 2).contiguous()  # noqa: E731
    loss, grad, counted, lerr, gerr = loss_and_gradient(z, values, indices, lse, 2.0)
    n = max(1, int(counted.sum()))
    target = TopLogits(planes(values).cuda(), planes(indices).cuda(), lse.view(N, side, side).cuda())
    for form in (lambda t: t, lambda t: t.to(memory_format=torch.channels_last), lambda t: torch.nn.functional.pad(t, (0, 3))[..., :side]):
        for reduction, scale in (("mean", 1 / n), ("sum", 1.0), ("none", 1.0)):
            x = form(planes(z).cuda()).detach().requires_grad_()
            got = distill_loss_topk(x, target, temperature=2.0, reduction=reduction)
            want, tol = (loss.view(N, side, side), lerr.view(N, side, side)) if reduction == "none" else (loss.sum() * scale, lerr.sum() * scale)
            assert got.shape == want.shape and bool(((got.detach().double().cpu() - want).abs() <= tol + 2.0 ** -23 * want.abs()).all())
            got.sum().backward()
            g = x.grad.permute(0, 2, 3, 1).reshape(-1, C).double().cpu()
            assert bool(((g - grad * scale).abs() <= scale * (gerr + (half_step(dtype) + 2.0 ** -21) * grad.abs()) + 2.0 ** -133).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,side,k", [(2, 33, 5, 4), (1, 64, 9, 64), (3, 80, 7, 8), (1, 150, 12, 3), (2, 255, 6, 9), (1, 256, 17, 64), (1, 257, 4, 5), (4, 40, 32, 2)])
def test_planes_of_many_classes(N, C, side, k, dtype, monkeypatch):
    monkeypatch.setattr("segk.distill.PLANE_POSITIONS", 0)                # read in place, few as they are
    test_planes(N, C, side, k, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_positions_of_many_classes(dtype):
    """As many as are read in place, against the formulas on the host in 64 bits."""
    g = torch.Generator().manual_seed(2)
    z, t = torch.randn(1, 80, 130, 130, generator=g).to(dtype), (2 * torch.randn(1, 80, 130, 130, generator=g)).to(dtype)
    got, host = top_logits(t.cuda(), 5, temperature=2.0), top_logits(t, 5, temperature=2.0)
    assert torch.equal(got.values.cpu(), host.values) and torch.equal(got.indices.cpu(), host.indices)
    x, y = z.cuda().requires_grad_(), z.double().requires_grad_()
    a, b = distill_loss_topk(x, got, temperature=2.0), distill_loss_topk(y, TopLogits(host.values.double(), host.indices, got.lse.cpu().double()), temperature=2.0)
    a.backward()
    b.backward()
    # as derived in distill_oracle.py, |logit| / T <= 5: u = 2^-21 (8 + 3 * 5); a position's loss T^2 u (3 + 10), its gradient T u (M q + p + 2 share)
    u = 2.0 ** -21 * 23
    assert abs(float(a.detach()) - float(b.detach())) <= 4 * u * 13 + 2.0 ** -23 * float(b.detach())
    err = (x.grad.cpu().double() - y.grad).abs() * 130 * 130
    assert bool((err <= 2 * u * 4 + (half_step(dtype) + 2.0 ** -21) * y.grad.abs() * 130 * 130).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("N,C,side,k", [(2, 4, 8, 3), (2, 32, 8, 6), (2, 33, 7, 5), (1, 150, 9, 12), (1, 256, 8, 64)])
def test_planes_with_repeated_missing_and_masked_entries(N, C, side, k, given, dtype, monkeypatch):
    monkeypatch.setattr("segk.distill.PLANE_POSITIONS", 0)
    P = N * side * side
    z, values, indices, lse = problem(P, C, k, seed=C, dtype=dtype)
    g = torch.Generator().manual_seed(k)
    indices[0::4, 1] = indices[0::4, 0]                                   # a class twice, with another value
    indices[1::4] = torch.where(torch.rand(indices[1::4].shape, generator=g) < 0.5, C, indices[1::4].int()).int()     # entries that do not exist
    indices[2::7] = -1                                                    # positions without entries
    z[2::7] = math.nan
    z[3::4, 0] = torch.finfo(dtype).min                                   # masked logits, where no teacher's mass is
    gone = torch.arange(C).expand(P, C).clone()
    for j in range(k):
        gone.scatter_(1, indices[:, j:j + 1].long().clamp(0, C - 1), -1)
    z = torch.where((gone[:, -1:] >= 0) & (torch.arange(P) % 5 == 0)[:, None] & (torch.arange(C) == C - 1), -math.inf, z.float()).to(dtype)
    lse = lse + 0.1 if given else None                                    # repeated entries stay below 1 together, mostly
    clean = torch.where(torch.isnan(z), torch.zeros((), dtype=dtype), z)
    loss, grad, counted, lerr, gerr = loss_and_gradient(clean, values, indices, lse, 1.0)
    planes = lambda t: t.view(N, side, side, -1).permute(0, 3, 1, 2).contiguous()  # noqa: E731
    target = TopLogits(planes(values).cuda(), planes(indices).cuda(), None if lse is None else lse.view(N, side, side).cuda())
    x = planes(z).cuda().requires_grad_()
    got = distill_loss_topk(x, target, reduction="none")
    got.sum().backward()
    # Class 0 may be one with mass: (finfo.min - maximum) log2(e) is beyond fp32 then and the loss infinite, where 64 bits hold 10^38
    huge, ok = loss > 2.0 ** 100, loss <= 2.0 ** 100
    assert bool((got.detach().cpu().view(-1)[huge] > 2.0 ** 100).all())
    assert bool(((got.detach().cpu().double().view(-1) - loss).abs() <= lerr + 2.0 ** -23 * loss.abs())[ok].all())
    dx = x.grad.permute(0, 2, 3, 1).reshape(P, C).cpu().double()
    assert bool(((dx - grad).abs() <= gerr + (half_step(dtype) + 2.0 ** -21) * grad.abs() + 2.0 ** -133)[ok].all()) and not dx[~counted].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,side", [(2, 33, 5), (1, 64, 9), (3, 150, 7), (1, 256, 12), (1, 257, 3)])
def test_top_of_planes_of_many_classes(N, C, side, dtype, monkeypatch):
    monkeypatch.setattr("segk.distill.PLANE_POSITIONS", 0)
    g = torch.Generator().manual_seed(C)
    z = torch.randint(-3, 4, (N, C, side, side), generator=g).to(dtype) / 2          # ties everywhere
    z[0, C // 2, 0, 0] = z[0, C - 1, 0, 0] = math.nan
    z[0, 3, 0, 1] = math.inf
    z[0, :, 1, 1] = -math.inf
    z[0, : C - 2, 1, 0] = -math.inf
    for k in (1, 2, 3, 8, 9, 33):
        for form in (lambda t: t, lambda t: torch.nn.functional.pad(t, (0, 3))[..., :side]):
            got, host = top_logits(form(z.cuda()), k, temperature=2.0), top_logits(z, k, temperature=2.0)
            assert torch.equal(got.indices.cpu(), host.indices)
            same = got.values.cpu().eq(host.values) | (got.values.cpu().isnan() & host.values.isnan())
            assert bool(same.all()) and got.values.dtype == dtype
            want = torch.logsumexp(z.double() / 2, 1)
            lse, fine = got.lse.cpu().double(), torch.isfinite(want)
            assert bool(((lse - want).abs() <= 2.0 ** -21 * (8 + 3 * 1.5 / 2))[fine].all())
            assert float(lse[0, 1, 1]) == -math.inf and math.isnan(float(lse[0, 0, 0])) and math.isnan(float(lse[0, 0, 1]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [5, 77, 1030, 9001])
def test_strides_offsets_and_dimensions(V, dtype):
    z, values, indices, lse = problem(6, V, 3, seed=V, dtype=dtype)
    wide = lambda x: torch.nn.functional.pad(x, (3, 2), value=9.0).cuda()[:, 3:-2]   # noqa: E731  rows that begin anywhere
    check(z, values, indices, lse, 1.0, cuda=wide)
    check(z, values, indices, lse, 1.0, cuda=lambda x: x.t().contiguous().cuda().t())          # classes strided
    x = z.view(2, 3, V).cuda().requires_grad_()
    y = z.cuda().requires_grad_()
    target = TopLogits(values.cuda(), indices.cuda(), lse.cuda())
    a = distill_loss_topk(x, TopLogits(target.values.view(2, 3, 3), target.indices.view(2, 3, 3), target.lse.view(2, 3)), dim=-1)
    b = distill_loss_topk(y, target)
    (a + b).backward()
    assert torch.equal(a, b) and torch.equal(x.grad.view(6, V), y.grad)
    one = z[:1].expand(6, V).cuda()                                                              # stride 0
    same = TopLogits(target.values[:1].expand(6, 3), target.indices[:1].expand(6, 3), target.lse[:1].expand(6))
    alone = distill_loss_topk(one[:1], TopLogits(target.values[:1], target.indices[:1], target.lse[:1]), reduction="none")
    # the copies begin at other places of a 16-byte piece and add up in another order: either result is within lerr of the exact one
    lerr = float(loss_and_gradient(z[:1], values[:1], indices[:1], lse[:1], 1.0)[3])
    assert float((distill_loss_topk(one, same, reduction="none") - alone).abs().max()) <= 2 * lerr


def test_half_precision_logits_and_values_types():
    z, values, indices, lse = problem(4, 333, 6, dtype=torch.float16)
    check(z, values, indices, lse, 1.0)
    z, values, indices, lse = problem(4, 333, 6, dtype=BF16, values_dtype=F32)
    check(z, values, indices.long(), lse, 1.0)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        distill_loss_topk(z.double().cuda(), TopLogits(values.cuda(), indices.cuda(), None))
    with pytest.raises(ValueError, match="same device"):
        distill_loss_topk(z.cuda(), TopLogits(values, indices, None))


@pytest.mark.parametrize("shape", [(7, 50), (3, 4, 8, 8), (5, 3000)])
def test_upstream_gradients_and_a_second_backward_pass(shape):
    C = shape[1]
    P = math.prod(shape) // C
    z, values, indices, lse = problem(P, C, 3, T=2.0)
    to = lambda t, c: t.view(shape[0], *shape[2:], c).movedim(-1, 1).contiguous().cuda() if len(shape) > 2 else t.view(-1, c).cuda()  # noqa: E731
    target = TopLogits(to(values, 3), to(indices, 3), lse.view(shape[0], *shape[2:]).cuda())
    if len(shape) == 2:
        check(z, values, indices, lse, 2.0, upstream=-3.0)
    for reduction in ("mean", "sum", "none"):
        x = to(z, C).requires_grad_()
        loss = distill_loss_topk(x, target, temperature=2.0, reduction=reduction)
        total = loss.sum()
        g1, = torch.autograd.grad(total, x, retain_graph=True)
        keep = g1.clone()
        g2, = torch.autograd.grad(total, x, retain_graph=True)
        g3, = torch.autograd.grad(2 * total, x)              # a power of two: exact
        assert torch.equal(keep, g2) and torch.equal(2 * keep, g3) and torch.equal(keep, g1)
    x = to(z, C).requires_grad_()
    w = torch.rand(target.lse.shape, device="cuda")
    (distill_loss_topk(x, target, temperature=2.0, reduction="none") * w).sum().backward()
    y = to(z, C).requires_grad_()
    g, = torch.autograd.grad(distill_loss_topk(y, target, temperature=2.0, reduction="sum"), y)
    # T (M q - p) is a difference of two products of at most T = 2 each, whose factors (weight, T, upstream, 1 / sum) are multiplied in
    # another order: up to four roundings of 2^-24 * 2 on either side of the difference and on either side of this comparison
    torch.testing.assert_close(x.grad, g * w.unsqueeze(1), rtol=2.0 ** -20, atol=2 * 2 * 4 * 2.0 ** -24 * 2)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("classes_last", [True, False])
def test_saved_tensors_that_come_back_as_copies(classes_last, reduction):
    """Offloaded activations: the backward pass sees other memory, and contiguous where the logits were a padded view."""
    g = torch.Generator().manual_seed(3)
    shape = (6, 200) if classes_last else (2, 5, 12, 8)
    z = torch.randn(shape, generator=g).cuda()
    t = top_logits(2 * torch.randn(shape, generator=g).cuda(), 3)

    def gradient(offload):
        leaf = z.clone().requires_grad_()
        view = torch.nn.functional.pad(leaf, (1, 2))[..., 1:-2] * 1.5 if classes_last else torch.nn.functional.pad(leaf, (0, 0, 0, 0, 0, 3))[:, :5]
        view = torch.nn.functional.pad(view, (0, 4))[..., :shape[-1]] if classes_last else view
        with torch.autograd.graph.save_on_cpu() if offload else torch.enable_grad():
            loss = distill_loss_topk(view, t, reduction=reduction)
        del view
        junk = [torch.full(shape, 1e30, device="cuda") for _ in range(4)]          # takes the freed memory
        first, = torch.autograd.grad(loss.sum() * 2.0, leaf, retain_graph=True)
        second, = torch.autograd.grad(loss.sum(), leaf)
        assert len(junk) == 4
        return first, second
    for a, b in zip(gradient(True), gradient(False)):
        assert torch.equal(a, b) and a.any()


def test_a_second_differentiation_is_refused():
    z, values, indices, lse = problem(4, 50, 3)
    x = z.cuda().requires_grad_()
    loss = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()))
    want, = torch.autograd.grad(loss, x, retain_graph=True)
    g, = torch.autograd.grad(loss, x, create_graph=True)
    assert torch.equal(g.detach(), want)
    with pytest.raises(RuntimeError, match="does not require grad"):           # torch's upstream gradient, a constant 1
        torch.autograd.grad(g.sum(), x)
    g, = torch.autograd.grad(loss2 := distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda())) ** 2, x, create_graph=True)
    assert torch.allclose(g.detach(), 2 * loss.detach() * want, rtol=2.0 ** -20) and loss2.requires_grad
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_gradient_against_differences_of_the_definition():
    z, values, indices, lse = problem(5, 400, 7, T=1.5)
    x = z.cuda().requires_grad_()
    distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()), temperature=1.5, reduction="sum").backward()
    _, _, _, _, gerr = loss_and_gradient(z, values, indices, lse, 1.5)
    g = torch.Generator().manual_seed(2)
    for _ in range(3):
        d = torch.randn(z.shape, generator=g, dtype=torch.float64)
        up, down = (loss_and_gradient(z.double() + s * 1e-5 * d, values, indices, lse, 1.5)[0].sum() for s in (1, -1))
        got = float((x.grad.double().cpu() * d).sum())
        # central difference: 1e-10 times third derivatives, 1e-16 * loss / 1e-5
        assert abs(float(up - down) / 2e-5 - got) <= float((gerr * d.abs()).sum()) + 2.0 ** -23 * abs(got) + 1e-7


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", WIDTHS)
def test_top_rows(V, dtype):
    g = torch.Generator().manual_seed(V)
    z = (3 * torch.randn(4, V, generator=g)).to(dtype)
    for k in {1, min(V, 5), min(V, 64)}:
        for x in (z.cuda(), torch.nn.functional.pad(z, (1, 4)).cuda()[:, 1:-4]):
            values, indices, lse = top_logits(x, k, temperature=2.0)
            host = top_logits(z, k, temperature=2.0)
            assert torch.equal(values.cpu(), host.values) and torch.equal(indices.cpu(), host.indices) and values.dtype == dtype
            want = torch.logsumexp(z.double() / 2, 1)
            # exp arguments up to 1.45 * |z| / 2 in base 2, log of the sum: as derived for the loss
            assert bool(((lse.double().cpu() - want).abs() <= 2.0 ** -21 * (8 + 3 * z.double().abs().amax(1) / 2)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [8, 70, 700, 5000, 40000, 140000])
def test_top_rows_where_order_is_hard(V, dtype):
    g = torch.Generator().manual_seed(V)
    rows = [torch.zeros(V), torch.full((V,), -math.inf), torch.full((V,), torch.finfo(dtype).min), torch.arange(V) / V, -torch.arange(V) / V,
            torch.randint(0, 3, (V,), generator=g).float(), torch.randn(V, generator=g), torch.randn(V, generator=g), torch.randn(V, generator=g),
            torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0), -torch.rand(V, generator=g) - 1]
    z = torch.stack(rows).to(dtype)
    z[6, V // 2] = math.nan
    z[6, V - 1] = math.nan
    z[7, V // 3] = math.inf
    z[8, : V - 2] = -math.inf
    for k in {1, min(V, 3), min(V, 64)}:
        values, indices, lse = top_logits(z.cuda(), k)
        host = top_logits(z, k)
        assert torch.equal(indices.cpu(), host.indices)
        assert torch.equal(values.cpu().view(torch.int16 if dtype == BF16 else torch.int32), host.values.view(torch.int16 if dtype == BF16 else torch.int32))
        assert float(lse[1]) == -math.inf and math.isnan(float(lse[6])) and math.isnan(float(lse[7])) and abs(float(lse[0]) - math.log(V)) < 2.0 ** -20 * 12


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,side", [(2, 4, 8), (1, 3, 5), (2, 8, 12), (1, 13, 7), (1, 32, 6), (2, 40, 5), (1, 1, 4)])
def test_top_planes(N, C, side, dtype):
    g = torch.Generator().manual_seed(C)
    z = torch.randint(-3, 4, (N, C, side, side), generator=g).to(dtype) / 2          # ties everywhere
    z[0, 0, 0, 0] = math.nan
    for k in {1, min(C, 3), C}:
        if k > 64:
            continue
        for x in (z.cuda(), z.cuda().to(memory_format=torch.channels_last)):
            values, indices, lse = top_logits(x, k)
            host = top_logits(z, k)
            assert torch.equal(indices.cpu(), host.indices) and torch.equal(torch.nan_to_num(values.cpu(), 99.0), torch.nan_to_num(host.values, 99.0))
            torch.testing.assert_close(lse.cpu(), host.lse, rtol=2.0 ** -20, atol=2.0 ** -20, equal_nan=True)


def test_other_stream_and_captured_graph():
    z, values, indices, lse = problem(64, 2000, 8, T=2.0)
    target = TopLogits(values.cuda(), indices.cuda(), lse.cuda())

    def step(x):
        t = top_logits(x, 4, temperature=2.0)
        loss = distill_loss_topk(x, target, temperature=2.0)
        return (*t, loss, torch.autograd.grad(loss, x)[0])
    x = z.cuda().requires_grad_()
    want = [t.clone() for t in step(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.clone() for t in step(x)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    static = z.cuda().requires_grad_()
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(static)
        graphs.append((g, out))
    for seed in (5, 6, 7):
        new = problem(64, 2000, 8, seed=seed)[0].cuda()
        with torch.no_grad():
            static.copy_(new)
        want = [t.clone() for t in step(new.requires_grad_())]
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("T", [2.0 ** -40, 1e-3, 2.0 ** 40])
def test_extreme_temperatures(T):
    """At the ends of the range the softmax is one class, or uniform."""
    for V in (6, 300):
        z = torch.arange(V, dtype=F32).repeat(4, 1)
        x = z.cuda().requires_grad_()
        t = top_logits(x, 3, temperature=T)
        assert t.indices.cpu().tolist() == [[V - 1, V - 2, V - 3]] * 4
        loss = distill_loss_topk(x, t, temperature=T)
        loss.backward()
        assert torch.isfinite(t.lse).all() and torch.isfinite(loss) and torch.isfinite(x.grad).all()
        # The student is the teacher: both give every class the same, up to rounding of probabilities, 2^-18.  The kept lse and
        # z / T are of the size V / T in fp32: rounded at 1 / T, at its product with log2(e), at those with z and with lse, at
        # lse as kept and at their difference, log p is off by d <= 8 * 2^-24 V / T (nothing is off where T is a power of two
        # and z / T exact).  d weighs in p log p, and as a rest of up to d that the teacher seems to have left:
        # d (log d - log R), log R >= -(3 + log V) / T; 1e-3 and 300: e^d - 1 < 1.1 d.
        d = 0.0 if math.log2(T).is_integer() else 8 * 2.0 ** -24 * V / T
        off = 2.0 ** -18 + 1.1 * d * (2 + (0 if d == 0 else abs(math.log(d)) + (3 + math.log(V)) / T))
        assert abs(float(loss.detach())) <= T * T * off and float(x.grad.abs().max()) <= T * (2.0 ** -18 + 4 * d)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P", [1, 3, 129])
@pytest.mark.parametrize("V,k", [(16384, 64), (33793, 64), (40963, 5), (66049, 1), (131585, 33), (262147, 64)])
def test_top_of_long_rows(V, k, P, dtype):
    """Ties, NaN and infinities in long rows."""
    g = torch.Generator().manual_seed(V)
    base = 2 * torch.randn(3, V, generator=g)
    base[1] = torch.randint(-2, 3, (V,), generator=g).float()                # ties everywhere
    base[2] = -math.inf
    base[2, ::V // 40] = base[0, ::V // 40]                                   # 40 or 41 finite logits: fewer than 64
    for last in (None, math.nan, math.inf):
        z = base.clone()
        if last is not None:
            z[0, V - 1] = last
            z[1, V // 2] = last
        z = z.to(dtype).repeat(-(-P // 3), 1)[:P]
        host = top_logits(z[:3], k, temperature=2.0)
        got = top_logits(z.cuda(), k, temperature=2.0)
        for lo in range(0, P, 3):
            n = min(3, P - lo)
            same = got.values[lo:lo + n].cpu().eq(host.values[:n]) | (got.values[lo:lo + n].cpu().isnan() & host.values[:n].isnan())
            assert bool(same.all()) and torch.equal(got.indices[lo:lo + n].cpu(), host.indices[:n])
        want = torch.logsumexp(z[:3].double() / 2, 1)
        for row in range(min(P, 3)):
            lse = got.lse[row::3].cpu()
            if not math.isfinite(want[row]):
                assert lse.isnan().all()
            else:
                top = float(z[row][z[row].isfinite()].double().abs().max())
                assert bool(((lse.double() - want[row]).abs() <= 2.0 ** -21 * (8 + 3 * top / 2)).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [70, 500, 1000, 2000, 4000, 9000])
def test_as_many_as_can_be_kept(V, dtype):
    """k = 64 of rows whose threads are hardly more: many candidates, in order, in reverse, equal, or in runs."""
    g = torch.Generator().manual_seed(V)
    rows = [torch.randn(V, generator=g), torch.arange(V) / 64.0, -torch.arange(V) / 64.0, torch.zeros(V), torch.randint(0, 4, (V,), generator=g).float(),
            (torch.arange(V) // 64).float(), torch.where(torch.arange(V) < V - 66, -math.inf, torch.randn(V, generator=g)), torch.arange(V).fmod(65.0)]
    z = torch.stack(rows).to(dtype)
    for k in (33, 63, 64):
        host, got = top_logits(z, k), top_logits(z.cuda(), k)
        assert torch.equal(got.values.cpu(), host.values) and torch.equal(got.indices.cpu(), host.indices)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1024, 2048, 8192, 16384, 32768, 65536, 131072])
def test_rows_that_fill_a_kernel_exactly(V, dtype):
    """Lengths at which a row just fits the registers of a kernel, if it begins and ends with a 16-byte piece, and does not otherwise."""
    z, values, indices, lse = problem(20, V, 7, seed=V, dtype=dtype)          # 20 rows: not shared by workgroups below 16384 pieces

    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        return flat[1:].view(x.shape).copy_(x)

    def padded(x):
        return torch.nn.functional.pad(x.cuda(), (0, 1))[:, :V]
    want = torch.topk(z.double(), 7, 1).values
    for form in (lambda x: x.cuda(), shifted, padded):
        got = top_logits(form(z), 7)
        assert torch.equal(got.values.cpu().double(), want) and torch.equal(z.gather(1, got.indices.cpu().long()), got.values.cpu())
        assert bool(((got.lse.cpu().double() - torch.logsumexp(z.double(), 1)).abs() <= 2.0 ** -21 * (8 + 3 * z.double().abs().amax(1))).all())
        check(z, values, indices, lse, 1.0, cuda=form)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P,V", [(4607, 9), (4608, 9), (8191, 16), (8192, 16), (16384, 32), (16383, 32), (5, 200), (1027, 80)])
def test_many_short_rows(P, V, dtype):
    """Both sides of the border between a thread and a wave for each row, and rows that do not fill the last workgroup."""
    z, values, indices, lse = problem(P, V, 3, seed=V, dtype=dtype, ignored=0.1)
    got = top_logits(z.cuda(), 3)
    want = torch.topk(z.double(), 3, 1)
    assert torch.equal(got.values.cpu().double(), want.values)
    assert torch.equal(z.gather(1, got.indices.cpu().long()), got.values.cpu())
    check(z, values, indices, lse, 1.0)


@pytest.mark.parametrize("weight", [1.0, -2.0])
@pytest.mark.parametrize("P,V", [(1, 40), (70, 40), (1100, 40), (16384, 12), (16385, 12), (40000, 12), (20, 140000), (3, 300000)])
def test_positions_counted_for_a_mean(P, V, weight):
    """The mean with a gradient (counted before) and without (counted with the sum), over rows of loss 0 and rows without entries."""
    z, values, indices, lse = problem(min(P, 100), V, 3, seed=P, ignored=0.2)
    indices[0::3] = -1                                           # whole rows, and single entries of others
    values[1::3], indices[1::3], lse[1::3] = 0.0, -1, 0.0
    indices[1::3, 0] = 5                                         # p = 1 at class 5 ...
    z[1::3] = -200.0
    z[1::3, 5] = 200.0                                           # ... and the student agrees: loss 0
    agreed = torch.arange(P) % len(z) % 3 == 1                    # where these rows are repeated to
    n = -(-P // len(z))
    z, values, indices, lse = (torch.cat([t] * n)[:P].cuda() for t in (z, values, indices, lse))
    loss = distill_loss_topk(z, TopLogits(values, indices, lse), weight=weight, reduction="none")
    zero, has = loss[agreed.cuda()], (indices >= 0).any(1)
    assert not zero.any() and not loss[~has].any()
    want = loss.double().sum() / max(1, int(has.sum()))
    for idx in (indices, indices.long()):
        x = z.clone().requires_grad_()
        counted = distill_loss_topk(x, TopLogits(values, idx, lse), weight=weight)
        with torch.no_grad():
            plain = distill_loss_topk(z, TopLogits(values, idx, lse), weight=weight)
        # both sum in double, over at most 256 parts that are rounded to fp32, and round the quotient
        tol = 2.0 ** -23 * float(loss.abs().double().sum()) / max(1, int(has.sum()))
        assert abs(float(counted.detach()) - float(want)) <= tol and float(plain) == float(counted.detach())


@pytest.mark.parametrize("N,side", [(3, 8), (2, 66), (1, 21), (5, 130), (1, 1700)])
def test_positions_counted_in_planes(N, side):
    """A constant loss per counted position: the mean gives the number away.  Entries behind the first decide some positions."""
    g = torch.Generator().manual_seed(side)
    indices = torch.randint(-1, 3, (N, 3, side, side), generator=g, dtype=torch.int32)
    indices[:, :, : side // 2] = torch.where(torch.rand(N, 3, side // 2, side, generator=g) < 0.7, -1, 2).int()
    z = torch.zeros(N, 3, side, side)
    z[:, 1] = 1.0
    values = torch.zeros(N, 3, side, side)
    has = (indices >= 0).any(1)
    flat = torch.empty(indices.numel() + 1, dtype=torch.int32, device="cuda")
    odd = flat[1:].view(indices.shape).copy_(indices)             # not aligned to 16 bytes
    x = z.cuda().requires_grad_()
    for idx in (indices.cuda(), indices.long().cuda(), odd):
        target = TopLogits(values.cuda(), idx, None)
        total = distill_loss_topk(x, target, reduction="sum")
        mean = distill_loss_topk(x, target)
        n = float(total.detach().double() / mean.detach().double())
        assert abs(n / int(has.sum()) - 1) <= 2.0 ** -22          # two roundings to fp32; the number has to be exact
        ga, = torch.autograd.grad(total, x)
        gb, = torch.autograd.grad(mean, x)
        # the scale is rounded once and the product once, on both sides
        assert bool(((gb.double() * int(has.sum()) - ga.double()).abs() <= 2.0 ** -21 * ga.double().abs()).all())
        assert not gb.permute(0, 2, 3, 1)[~has.cuda()].any()


def test_far_rows_of_a_large_tensor():
    """Element offsets beyond 2^31."""
    V, P = 131072, 16400
    z = torch.zeros(P, V, dtype=BF16, device="cuda")
    host = problem(3, V, 6, dtype=BF16)
    z[-3:] = host[0].cuda()
    values, indices, lse = top_logits(z, 6)
    near = top_logits(z[-3:].clone(), 6)
    assert torch.equal(values[-3:], near.values) and torch.equal(indices[-3:], near.indices) and torch.equal(lse[-3:], near.lse)
    assert indices[:-3].cpu().eq(torch.arange(6, dtype=torch.int32)).all()
    keep = TopLogits(torch.zeros(P, 6, device="cuda", dtype=BF16), torch.full((P, 6), -1, device="cuda"), torch.zeros(P, device="cuda"))
    keep.values[-3:], keep.indices[-3:], keep.lse[-3:] = host[1].cuda(), host[2].cuda().long(), host[3].cuda()
    x = z.requires_grad_()
    g, = torch.autograd.grad(distill_loss_topk(x, keep), x)
    y = z[-3:].detach().clone().requires_grad_()
    w, = torch.autograd.grad(distill_loss_topk(y, TopLogits(*(t[-3:] for t in keep))), y)
    assert torch.equal(g[-3:], w) and not g[:4].any() and not g[-4].any()


@pytest.mark.parametrize("T", [1.0, 8.0, 20.0, 64.0, 256.0])
@pytest.mark.parametrize("shape,k", [((40, 1000), 8), ((64, 80), 8), ((4700, 9), 3), ((16, 6), 2), ((16, 6), 6), ((2, 70000), 5),
                                     ((2, 4, 8, 12), 2), ((1, 5, 7, 9), 3), ((1, 21, 8, 8), 4), ((1, 21, 8, 8), 21), ((2, 80, 128, 64), 3)])
def test_high_temperatures(shape, k, T):
    """The loss where its terms cancel: rows of a wave, of a thread and shared by workgroups, class planes of each kind; a given logsumexp,
    one at which nothing is left outside, and renormalised."""
    C = shape[1]
    P = math.prod(shape) // C
    n = min(P, 64)
    z, values, indices, lse = problem(n, C, k, seed=C + k, T=T)
    again = -(-P // n)

    def planes(x):                                               # the positions of [P, c] as [N, c, H, W]
        x = x.repeat((again,) + (1,) * (x.dim() - 1))[:P]
        if len(shape) == 2:
            return x.cuda()
        rest = (shape[0],) + shape[2:]
        return x.reshape(rest).cuda() if x.dim() == 1 else x.reshape(rest + (-1,)).movedim(-1, 1).contiguous().cuda()

    def back(x):
        return (x if len(shape) == 2 else x.reshape(-1) if x.dim() == len(shape) - 1 else x.movedim(1, -1).reshape(P, -1)).detach().cpu().double()[:n]
    for given in (lse, None):
        loss, grad, _, _, _ = loss_and_gradient(z, values, indices, given, T)
        lerr, gerr = cancellation_bounds(z, values, indices, given, T)
        x = planes(z).requires_grad_()
        target = TopLogits(planes(values), planes(indices), None if given is None else planes(given))
        got = distill_loss_topk(x, target, temperature=T, reduction="none")
        err = (back(got) - loss).abs()
        assert bool((err <= lerr).all()), (float((err / loss).max()), float((lerr / loss).max()))
        if given is None or k < C:                               # both sides add up to 1: no term is negative
            assert float(got.detach().min()) >= 0
        plain = distill_loss_topk(x.detach(), target, temperature=T, reduction="sum")
        x2 = x.detach().requires_grad_()
        total = distill_loss_topk(x2, target, temperature=T, reduction="sum")
        every = got.detach().double().sum().cpu()
        for s in (plain, total.detach()):
            assert abs(float(s) - float(every)) <= 2.0 ** -20 * float(got.detach().abs().double().sum())
        got.sum().backward()
        total.backward()
        for g in (x.grad, x2.grad):
            assert bool(((back(g) - grad).abs() <= gerr + 2.0 ** -24 * grad.abs()).all())


@pytest.mark.parametrize("shape", [((1 << 26) + 5, 33), ((1 << 24) + 3, 4, 1, 2), ((1 << 24) + 3, 40, 1, 2)])
def test_more_threads_than_one_launch_may_have(shape, monkeypatch):
    """Rows, and images of few positions, whose threads number 2^32 and more (a launch has fewer): the same bits as parts of them give
    (by the same kernel: a part's planes are not copied into rows for being few)."""
    from segk import distill
    monkeypatch.setattr(distill, "PLANE_POSITIONS", 0)
    g = torch.Generator(device="cuda").manual_seed(1)
    N = shape[0]
    teacher, student = (torch.empty(shape, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
    target = top_logits(teacher, 2, temperature=2.0)
    x = student.requires_grad_()
    each = distill_loss_topk(x, target, temperature=2.0, reduction="none")
    up = torch.rand(each.shape, generator=g, device="cuda")
    grad, = torch.autograd.grad(each, x, up)
    mean = distill_loss_topk(x, target, temperature=2.0)
    grad_mean, = torch.autograd.grad(mean, x)
    with torch.no_grad():
        plain = distill_loss_topk(x, target, temperature=2.0)
    want = float(each.detach().double().mean())
    for got in (mean, plain):                                    # sums of up to 1024 losses in fp32 before those in double
        assert abs(float(got.detach()) - want) <= 2.0 ** -20 * want
    for lo in (0, N // 8 - 500, N // 4 - 500, N // 2 - 500, 3 * (N // 4) - 500, N - 1000):
        part = slice(lo, lo + 1000)
        top_part = top_logits(teacher[part], 2, temperature=2.0)
        assert all(torch.equal(a[part], b) for a, b in zip(target, top_part))
        y = x.detach()[part].requires_grad_()
        few = distill_loss_topk(y, top_part, temperature=2.0, reduction="none")
        assert torch.equal(few, each[part])
        assert torch.equal(torch.autograd.grad(few, y, up[part], retain_graph=True)[0], grad[part])
        # the scale is rounded once, the product once more, then to bf16, on both sides
        sums = torch.autograd.grad(few.sum(), y)[0].double() / each.numel()
        assert bool(((grad_mean[part].double() - sums).abs() <= 2.0 ** -6 * sums.abs() + 2.0 ** -133).all())


@pytest.mark.parametrize("shape", [(6, 40), (2, 4, 3, 5)])
def test_forward_mode_is_refused(shape):
    """The kernels give no tangent: a dual number is refused with and without a gradient, never answered without its tangent."""
    import torch.autograd.forward_ad as fwd
    x = torch.randn(shape, device="cuda")
    target = top_logits(x, 2)
    with fwd.dual_level():
        for form in (x, x.clone().requires_grad_()):
            dual = fwd.make_dual(form, torch.ones_like(x))
            for f in top_logits(dual, 2):
                assert fwd.unpack_dual(f).tangent is None
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    distill_loss_topk(dual, target)
        assert torch.isfinite(distill_loss_topk(x, target))         # no dual: answered
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda y: distill_loss_topk(y, target), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("shape,k", [((5, 80), 1), ((5, 300), 2), ((9, 4), 1), ((5, 40000), 1), ((5, 140000), 1), ((2, 4, 3, 5), 1), ((2, 40, 128, 64), 1)])
def test_nan_at_the_only_kept_classes(shape, k):
    """softmax of a row with a NaN is NaN everywhere: so are its loss and its whole gradient, wherever the NaN stands."""
    C = shape[1]
    g = torch.Generator().manual_seed(C)
    z = torch.randn(shape, generator=g)
    z[1].view(C, -1)[C // 2:C // 2 + k, 0] = math.nan
    indices = (C // 2 + torch.arange(k, dtype=torch.int32)).view((1, k) + (1,) * (len(shape) - 2)).expand((shape[0], k) + shape[2:]).contiguous()
    for lse in (None, torch.full(shape[:1] + shape[2:], math.log(2.0 * k))):
        target = TopLogits(torch.zeros(indices.shape), indices, lse)
        host, x = z.clone().requires_grad_(), z.cuda().requires_grad_()
        want, got = (distill_loss_topk(t, TopLogits(*(None if f is None else f.to(t.device) for f in target)), reduction="none") for t in (host, x))
        want.sum().backward()
        got.sum().backward()
        bad = torch.zeros(shape, dtype=torch.bool)
        bad[1].view(C, -1)[:, 0] = True
        assert torch.equal(host.grad.isnan(), bad) and torch.equal(x.grad.isnan().cpu(), bad)
        assert torch.equal(want.isnan(), got.isnan().cpu()) and int(want.isnan().sum()) == 1
        y = z.cuda().requires_grad_()
        distill_loss_topk(y, TopLogits(*(None if f is None else f.cuda() for f in target)), reduction="sum").backward()
        assert torch.equal(y.grad.isnan().cpu(), bad)


def test_nan_among_the_values():
    nan_among_the_values("cuda")


@pytest.mark.parametrize("shape,k", [((40, 300), 5), ((3, 4, 9, 16), 2), ((2, 140000), 3), ((1, 40, 128, 128), 2)])
@pytest.mark.parametrize("captured", [False, True])
def test_a_backward_pass_replayed_without_its_forward_pass(shape, k, captured):
    """Captured by itself (the forward pass eager, or in a graph of its own) and replayed with other upstream gradients: nothing of one replay
    is left for the next.  The node is called directly, on the capturing stream."""
    g = torch.Generator(device="cuda").manual_seed(3)
    target = top_logits(torch.randn(shape, generator=g, device="cuda"), k, temperature=2.0)
    x = torch.randn(shape, generator=g, device="cuda").requires_grad_()
    up = torch.ones((), device="cuda")
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(forward):
            loss = distill_loss_topk(x, target, temperature=2.0)
    else:
        loss = distill_loss_topk(x, target, temperature=2.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(backward):
        grad = loss.grad_fn.apply(up)[0]
    for turn, scale in enumerate((2.0, 1.0, 0.5, 1.0, 1.0, -3.0)):
        if captured and turn % 2 == 0:
            with torch.no_grad():
                x.copy_(torch.randn(shape, generator=g, device="cuda"))
            forward.replay()
        up.fill_(scale)
        backward.replay()
        torch.cuda.synchronize()
        y = x.detach().clone().requires_grad_()
        want = distill_loss_topk(y, target, temperature=2.0)
        assert torch.equal(loss.detach(), want.detach())
        assert torch.equal(grad, torch.autograd.grad(want, y, torch.full((), scale, device="cuda"))[0])


def test_graphed_callable():
    """torch.cuda.make_graphed_callables: forward and backward pass in graphs of their own, inside an eager program."""
    z, values, indices, lse = problem(30, 90, 4, T=2.0)
    target = TopLogits(values.cuda(), indices.cuda(), lse.cuda())
    run = torch.cuda.make_graphed_callables(lambda x: distill_loss_topk(x, target, temperature=2.0), (z.cuda().requires_grad_(),))
    for seed, scale in ((1, 1.0), (2, 3.0), (3, 1.0)):
        x = torch.randn(30, 90, generator=torch.Generator().manual_seed(seed)).cuda().requires_grad_()
        y = x.detach().clone().requires_grad_()
        (run(x) * scale).backward()
        (distill_loss_topk(y, target, temperature=2.0) * scale).backward()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, y.grad)


@pytest.mark.parametrize("scale", [1.0, 2.0])
@pytest.mark.parametrize("shape,k", [((512, 4096), 5), ((4, 8, 256, 256), 2)])
def test_saved_memory_can_be_offloaded_and_recomputed(shape, k, scale):
    """Nothing as large as the logits stays on the device between the passes, where saved tensors are kept on the host or computed again."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator(device="cuda").manual_seed(3)
    target = top_logits(torch.randn(shape, generator=g, device="cuda"), k, temperature=2.0)
    z = torch.randn(shape, generator=g, device="cuda")
    x = z.clone().requires_grad_()
    want, = torch.autograd.grad(scale * distill_loss_topk(x, target, temperature=2.0), x)

    def offloaded(y):
        with torch.autograd.graph.save_on_cpu():
            return distill_loss_topk(y, target, temperature=2.0)

    def again(y):
        return checkpoint(lambda t: distill_loss_topk(t, target, temperature=2.0), y, use_reentrant=False)
    for form in (offloaded, again):
        y = z.clone().requires_grad_()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = form(y)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before < z.numel() * z.element_size() // 4
        (scale * loss).backward()
        assert torch.equal(y.grad, want)


def test_the_gradient_belongs_to_the_caller():
    """Changing it in place is no change to what a second backward pass needs."""
    z, values, indices, lse = problem(20, 70, 4, T=2.0)
    x = z.cuda().requires_grad_()
    loss = distill_loss_topk(x, TopLogits(values.cuda(), indices.cuda(), lse.cuda()), temperature=2.0)
    want, = torch.autograd.grad(loss, x, retain_graph=True)
    kept = want.clone()
    want.mul_(0.25)
    for _ in range(2):
        got, = torch.autograd.grad(loss, x, retain_graph=True)
        assert torch.equal(got, kept)
        got.zero_()
    loss.backward(retain_graph=True)
    x.grad.mul_(2.0)
    x.grad = None
    loss.backward()
    assert torch.equal(x.grad, kept)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("P", [6143, 6144])
@pytest.mark.parametrize("V", [511, 513, 1024, 1025])
def test_top_of_rows_by_a_wave_or_a_workgroup(P, V, dtype):
    """Both sides of the borders between them, in rows, classes and kept logits; rows that begin anywhere."""
    g = torch.Generator().manual_seed(V)
    z = torch.randn(P, V + 1, generator=g).to(dtype)
    z[::7] = z[::7].mul(4).round()                               # ties
    for form in (z[:, :-1].contiguous(), z[:, 1:]):
        x = form.cuda() if form.is_contiguous() else z.cuda()[:, 1:]
        for k in (24, 25, 40, 41):
            got = top_logits(x, k)
            if k == 24:
                order = torch.sort(form.float(), dim=1, descending=True, stable=True).indices[:, :41]
                values = form.gather(1, order)
            assert torch.equal(got.indices.cpu().long(), order[:, :k]) and torch.equal(got.values.cpu(), values[:, :k])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,C,side,k", [(1, 150, 128, 8), (1, 150, 128, 2), (1, 256, 128, 3), (4500, 40, 2, 3), (1100, 40, 4, 3)])
def test_planes_in_place_and_copied(N, C, side, k, dtype, monkeypatch):
    """Sizes on both sides of the rule give what the definition says, whichever way they are read."""
    g = torch.Generator().manual_seed(C)
    t, z = (2 * torch.randn(N, C, side, side, generator=g) for _ in range(2))
    t, z = t.to(dtype), z.to(dtype)
    order = torch.sort(t.float(), dim=1, descending=True, stable=True).indices[:, :k]
    rows = lambda x: x.cpu().movedim(1, -1).reshape(N * side * side, -1)                     # noqa: E731
    some = torch.randint(0, N * side * side, (20,), generator=g)
    for positions in (0, None, 1 << 30):
        if positions is not None:
            monkeypatch.setattr("segk.distill.PLANE_POSITIONS", positions)
        got = top_logits(t.cuda(), k, temperature=2.0)
        assert torch.equal(got.indices.cpu().long(), order) and torch.equal(got.values.cpu(), t.gather(1, order))
        x = z.cuda().requires_grad_()
        each = distill_loss_topk(x, got, temperature=2.0, reduction="none")
        grad, = torch.autograd.grad(each.sum(), x)
        loss, want, _, lerr, gerr = loss_and_gradient(rows(z)[some], rows(got.values)[some], rows(got.indices)[some], got.lse.cpu().reshape(-1)[some], 2.0)
        assert bool(((each.detach().cpu().reshape(-1)[some].double() - loss).abs() <= lerr + 2.0 ** -23 * loss).all())
        assert bool(((rows(grad)[some].double() - want).abs() <= gerr + (half_step(dtype) + 2.0 ** -21) * want.abs()).all())
        monkeypatch.undo()


def test_a_weight_that_wants_a_derivative_is_refused():
    x = torch.randn(6, 40, device="cuda", requires_grad=True)
    target = top_logits(x, 2)
    for grad in (True, False):
        for weight in (torch.tensor(2.0, requires_grad=True), torch.tensor(2.0, device="cuda", requires_grad=True)):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="weight"):
                distill_loss_topk(x, target, weight=weight)
            assert torch.equal(distill_loss_topk(x, target, weight=weight.detach()), distill_loss_topk(x, target, weight=2.0))


def test_empty_batches():
    for shape in ((0, 9), (0, 4, 3, 3), (2, 4, 0, 3)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        target = top_logits(x, 2)
        assert target.values.shape == shape[:1] + (2,) + shape[2:] and target.lse.shape == shape[:1] + shape[2:] and target.lse.is_cuda
        for reduction in ("mean", "sum", "none"):
            for t in (target, target._replace(lse=None)):
                loss = distill_loss_topk(x, t, reduction=reduction)
                loss.sum().backward()
                assert float(loss.detach().sum()) == 0 and x.grad.shape == shape and loss.dtype == F32 and loss.is_cuda
