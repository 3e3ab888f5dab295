"""Distillation from top logits on host tensors: definitions, refusals, the training loop; and the refusals of the C entry points,
which need no GPU."""
import math

import pytest
import torch

from distill_oracle import loss_and_gradient, top
from loss.distill import TopLogits, distill_loss_topk, top_logits


def problem(P, V, k, seed=0, dtype=torch.float32, ignored=0.0, T=1.0):
    g = torch.Generator().manual_seed(seed)
    t = (2.5 * torch.randn(P, V, generator=g)).to(dtype)
    z = (0.5 * t.float() + 1.5 * torch.randn(P, V, generator=g)).to(dtype)
    values, indices = top(t, k)
    lse = torch.logsumexp(t.float() / T, 1)
    if ignored:
        indices[torch.rand(P, generator=g) < ignored] = -1
    return z, TopLogits(values, indices, lse)


@pytest.mark.parametrize("V,k", [(1, 1), (2, 1), (2, 2), (7, 3), (80, 8), (300, 64)])
@pytest.mark.parametrize("rest", [False, True])
def test_host_loss_is_the_definition(V, k, rest):
    z, target = problem(9, V, k, seed=V, ignored=0.3, T=2.0)
    target = target if rest else target._replace(lse=None)
    loss, grad, counted, _, _ = loss_and_gradient(z, *target, 2.0, 0.7)
    for reduction, want, scale in (("none", loss, 1.0), ("sum", loss.sum(), 1.0), ("mean", loss.sum() / max(1, int(counted.sum())), 1.0 / max(1, int(counted.sum())))):
        x = z.double().requires_grad_()
        got = distill_loss_topk(x, target, temperature=2.0, reduction=reduction, weight=0.7)
        # double precision throughout, but for the logsumexp that the target holds in fp32 on both sides
        torch.testing.assert_close(got.double(), want, rtol=1e-9, atol=1e-9)
        got.sum().backward()
        torch.testing.assert_close(x.grad, grad * scale, rtol=1e-9, atol=1e-9)


def test_gradient_of_the_definition_against_differences():
    z, target = problem(4, 11, 3, seed=3, T=1.5)
    _, grad, _, _, _ = loss_and_gradient(z, *target, 1.5)
    g = torch.Generator().manual_seed(5)
    for _ in range(4):
        d = torch.randn(z.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = (loss_and_gradient(z.double() + s * h * d, *target, 1.5)[0].sum() for s in (1, -1))
        # central difference: error h^2 / 6 times a third derivative of order 1, and 1e-16 / h
        assert abs(float((up - down) / (2 * h)) - float((grad * d).sum())) < 1e-8


def test_host_top_logits_order_and_ties():
    z = torch.tensor([[1.0, 3.0, 3.0, -math.inf, 0.0, -0.0, math.nan, math.inf], [0.0] * 8])
    values, indices, lse = top_logits(z, 6)
    assert indices.tolist() == [[6, 7, 1, 2, 0, 4], [0, 1, 2, 3, 4, 5]] and indices.dtype == torch.int32
    assert abs(float(lse[1]) - math.log(8)) < 1e-6 and math.isnan(float(lse[0]))
    assert math.isnan(float(top_logits(torch.tensor([[1.0, math.inf]]), 1).lse)) and float(top_logits(torch.full((1, 3), -math.inf), 1).lse) == -math.inf
    z = torch.randn(2, 5, 3, 4)
    values, indices, lse = top_logits(z, 2, dim=1)
    v, i = top(z.permute(0, 2, 3, 1).reshape(-1, 5), 2)
    assert torch.equal(values.permute(0, 2, 3, 1).reshape(-1, 2), v) and torch.equal(indices.permute(0, 2, 3, 1).reshape(-1, 2), i)
    assert top_logits(torch.randn(0, 5), 2).values.shape == (0, 2)


def test_positions_without_entries_and_empty_batches():
    z, target = problem(5, 6, 2)
    none = target._replace(indices=torch.full_like(target.indices, -1))
    x = z.clone().requires_grad_()
    loss = distill_loss_topk(x, none)
    loss.backward()
    assert float(loss) == 0 and not x.grad.any()
    x = torch.full((1, 6), math.nan, requires_grad=True)           # not read where nothing was kept
    distill_loss_topk(x, TopLogits(torch.zeros(1, 2), torch.tensor([[6, -1]]))).backward()
    assert not x.grad.any()
    e = torch.zeros(0, 6, requires_grad=True)
    loss = distill_loss_topk(e, TopLogits(torch.zeros(0, 2), torch.zeros(0, 2, dtype=torch.int64)))
    loss.backward()
    assert float(loss) == 0 and e.grad.shape == (0, 6)


def test_refusals():
    z, target = problem(4, 9, 3)
    with pytest.raises(ValueError, match="temperature"):
        distill_loss_topk(z, target, temperature=0.0)
    for t in (math.inf, math.nan, -1.0, 1e-20, 1e20, "2"):
        with pytest.raises(ValueError, match="temperature"):
            top_logits(z, 2, temperature=t)
    with pytest.raises(ValueError, match="Reduction parameter unknown."):
        distill_loss_topk(z, target, reduction="batch")
    with pytest.raises(IndexError):
        distill_loss_topk(z, target, dim=2)
    for k in (0, 10, -1):
        with pytest.raises(ValueError, match="between 1 and"):
            top_logits(z, k)
    with pytest.raises(ValueError, match="between 1 and min\\(64"):
        top_logits(torch.zeros(1, 100), 65)
    with pytest.raises(ValueError, match="values and indices"):
        distill_loss_topk(z, TopLogits(target.values[:3], target.indices[:3]))
    with pytest.raises(ValueError, match="values and indices"):
        distill_loss_topk(z, TopLogits(target.values, target.indices[:, :2]))
    with pytest.raises(ValueError, match="kept entries"):
        distill_loss_topk(z, TopLogits(torch.zeros(4, 10), torch.zeros(4, 10, dtype=torch.int32)))
    with pytest.raises(TypeError, match="int32 or int64"):
        distill_loss_topk(z, target._replace(indices=target.indices.to(torch.int16)))
    with pytest.raises(TypeError, match="values"):
        distill_loss_topk(z, target._replace(values=target.indices))
    with pytest.raises(ValueError, match="lse"):
        distill_loss_topk(z, target._replace(lse=torch.zeros(3)))
    with pytest.raises(ValueError, match="detach"):
        distill_loss_topk(z, target._replace(values=target.values.clone().requires_grad_()))
    with pytest.raises(TypeError, match="floating"):
        top_logits(torch.zeros(3, 4, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="same device"):
        distill_loss_topk(z, TopLogits(target.values.to("meta"), target.indices, None))


def test_forward_mode_derivatives():
    """Kept by the loss on the CPU; a target is data in this mode too."""
    import torch.autograd.forward_ad as fwd
    z, target = problem(5, 30, 4, T=2.0)
    tangent = torch.randn(z.shape, generator=torch.Generator().manual_seed(9))
    _, grad, _, _, _ = loss_and_gradient(z, *target, 2.0)
    with fwd.dual_level():
        dual = fwd.make_dual(z.double(), tangent.double())
        got = fwd.unpack_dual(distill_loss_topk(dual, target, temperature=2.0, reduction="sum")).tangent
        assert abs(float(got) - float((grad * tangent.double()).sum())) < 1e-9
        for f in top_logits(fwd.make_dual(z, tangent), 3):
            assert fwd.unpack_dual(f).tangent is None
        with pytest.raises(ValueError, match="detach"):
            distill_loss_topk(z, target._replace(values=fwd.make_dual(target.values, torch.ones_like(target.values))))
        with pytest.raises(ValueError, match="detach"):
            distill_loss_topk(z, target._replace(lse=fwd.make_dual(target.lse, torch.ones_like(target.lse))))


def test_c_entry_points_refuse_bad_arguments_without_a_gpu():
    from segk import _lib
    F32, BF16 = _lib.SEGK_F32, _lib.SEGK_BF16
    top_call = lambda **k: _lib.call("segk_top_logits", *{**dict(z=4096, dt=F32, o=4, c=80, i=1, ld=80, k=8, t=1.0, v=4096, x=4096, l=4096, d=0, s=None), **k}.values())  # noqa: E731
    for kw, text in ((dict(z=None), "null"), (dict(dt=7), "dtype"), (dict(o=0), "shape"), (dict(c=0), "shape"), (dict(c=1 << 30), "shape"), (dict(ld=79), "ld"),
                     (dict(k=0), "k must"), (dict(k=65), "k must"), (dict(k=9, c=8, ld=8), "k must"), (dict(t=0.0), "temperature"), (dict(t=math.inf), "temperature"),
                     (dict(t=math.nan), "temperature"), (dict(z=4097), "aligned"), (dict(v=None), "null"), (dict(v=4100), "16-byte"), (dict(i=4, ld=320, k=9), "innermost"), (dict(i=4, c=257, ld=1028), "innermost"),
                     (dict(o=1 << 20, i=1 << 12, c=4, ld=4 << 12), "positions"), (dict(t=1e-20), "temperature"),
                     (dict(t=1e20), "temperature")):
        with pytest.raises(_lib.SegkError, match=text):
            top_call(**kw)
    base = dict(z=4096, dt=BF16, o=4, c=80, i=1, ld=80, v=4096, vdt=F32, x=4096, xb=4, lse=None, k=8, t=1.0, w=1.0, f=1, up=None, loss=4096, each=None, dz=4096,
                ldd=80, ws=4096, wsb=1 << 20, d=0, s=None)
    for kw, text in ((dict(x=None), "null"), (dict(vdt=9), "dtype"), (dict(xb=2), "bytes"), (dict(loss=None, dz=None), "no output"), (dict(f=3, up=16), "mean"),
                     (dict(f=2), "upstream"), (dict(f=4), "upstream"), (dict(f=4, up=16), "only the gradient"), (dict(ldd=79), "dlogits"), (dict(wsb=64), "SEGK_EWORKSPACE"),
                     (dict(ws=4098), "workspace must"), (dict(t=-1.0), "temperature"), (dict(k=81, c=80), "k must")):
        with pytest.raises(_lib.SegkError, match=text):
            _lib.call("segk_distill", *{**base, **kw}.values())
    assert _lib.query("segk_distill_workspace", 0, 4, 4) == 0 and _lib.query("segk_distill_workspace", 8, 80, 1) >= 4 * 8


class _Stored(torch.utils.data.Dataset):
    """Images with a teacher's top logits in place of label maps."""

    def __init__(self, n, C, side, k):
        g = torch.Generator().manual_seed(1)
        self.x = torch.randn(n, 3, side, side, generator=g)
        self.t = top_logits(2 * torch.randn(n, C, side, side, generator=g), k, temperature=2.0)

    def __len__(self):
        return self.x.shape[0]

    def __getitem__(self, i):
        return self.x[i], TopLogits(*(f[i] for f in self.t))


def test_training_loop_takes_the_loss_and_its_targets():
    """train() of the plain loop moves the target to the device and adds up loss(outputs, target): top logits go through it unchanged."""
    from train_helper.naive_train import train
    net = torch.nn.Conv2d(3, 4, 3, padding=1)
    before = net.weight.detach().clone()
    loader = torch.utils.data.DataLoader(_Stored(4, 4, 8, 2), batch_size=2)
    seen = []

    def loss(pred, target):
        assert isinstance(target, TopLogits) and target.values.shape == (2, 2, 8, 8)
        seen.append(distill_loss_topk(pred, target, temperature=2.0))
        return seen[-1]
    avg = train(loader, net, [loss], 0, 1, torch.device("cpu"), 2)
    assert len(seen) == 2 and abs(avg - sum(float(s) for s in seen) / 2) < 1e-6 and not torch.equal(before, net.weight)


@pytest.mark.parametrize("T", [8.0, 20.0, 64.0, 256.0, 4096.0])
@pytest.mark.parametrize("rest", [False, True])
def test_host_loss_at_high_temperatures(T, rest):
    """The terms of a row are of the order 1 / T and cancel to 1 / T^2: in fp32 nothing of the loss would be left."""
    z, target = problem(32, 300, 8, seed=2, T=T)
    target = target if rest else target._replace(lse=None)
    loss, grad, _, _, _ = loss_and_gradient(z, *target, T)
    x = z.clone().requires_grad_()
    got = distill_loss_topk(x, target, temperature=T, reduction="none")
    # 64-bit terms, log q of up to 8, times T^2, on both sides; one rounding to fp32
    assert got.dtype == torch.float32 and bool(((got.double() - loss).abs() <= 2.0 ** -24 * loss.abs() + T * T * 2.0 ** -47).all())
    got.sum().backward()
    assert bool(((x.grad.double() - grad).abs() <= 2.0 ** -24 * grad.abs() + T * 2.0 ** -47).all())


def nan_among_the_values(device):
    """A teacher's NaN without a logsumexp: softmax over the kept entries is NaN, and so are loss and gradient; entries that do not exist
    may hold anything, and a row of nothing but -inf counts as 0."""
    for shape in ((5, 9), (5, 80), (5, 40000), (5, 140000), (5, 4, 2, 3), (5, 40, 64, 64)):
        C, behind = shape[1], shape[2:]
        for k in (1, 3):
            for dtype in (torch.float32, torch.bfloat16):
                values = torch.zeros((5, k) + behind, dtype=dtype)
                indices = torch.arange(k).view((1, k) + (1,) * len(behind)).repeat((5, 1) + behind)
                values[1, 0], values[2], values[3, k - 1] = math.nan, math.nan, math.nan
                indices[3, k - 1] = -1
                values[4] = -math.inf
                x = torch.zeros(shape, device=device, requires_grad=True)
                loss = distill_loss_topk(x, TopLogits(values.to(device), indices.to(device)), reduction="none")
                loss.sum().backward()
                rows, grads = loss.detach().view(5, -1), x.grad.view(5, -1)
                assert rows[1:3].isnan().all() and grads[1:3].isnan().all()
                assert torch.isfinite(rows[[0, 3, 4]]).all() and torch.isfinite(grads[[0, 3, 4]]).all() and not rows[4].any() and not grads[4].any()
                assert float(distill_loss_topk(x.detach(), TopLogits(values.to(device), indices.to(device)), reduction="sum").isnan())


def test_nan_among_the_values():
    nan_among_the_values("cpu")


def test_which_planes_are_read_in_place():
    """Every side of the rule, at sizes on which it was measured; whatever it says, the kernels' own limits hold."""
    from segk.distill import _in_place
    yes = [(32, 1, 2, 4, 8), (32, 5, 4, 2, 32), (33, 1, 16384, 4, 8), (80, 1, 16384, 4, 2), (80, 16, 1024, 2, 0), (150, 1, 16384, 4, 1), (256, 1, 36864, 4, 0), (256, 1, 65536, 2, 8),
           (150, 1, 36864, 4, 8), (80, 4096, 16, 4, 0), (300, 9, 1, 4, 64)]
    no = [(33, 1, 16383, 4, 1), (80, 1, 65536, 4, 9), (257, 1, 1 << 20, 4, 1), (150, 1, 16384, 4, 8), (256, 1, 16384, 4, 0), (256, 1, 36864, 2, 0), (80, 16384, 4, 4, 0)]
    assert all(_in_place(*c) for c in yes) and not any(_in_place(*c) for c in no)
    for C in (2, 32, 33, 256, 257, 5000):
        for outer in (1, 1000, 1 << 20):
            for inner in (2, 16, 1 << 10):
                for selected in (0, 1, 8, 9, 64):
                    assert not _in_place(C, outer, inner, 4, selected) or C <= (256 if selected <= 8 else 32)
