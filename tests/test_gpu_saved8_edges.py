"""The 8-bit saved activations and the layer over them where they can go wrong beside their sizes."""
import pytest
import torch
from test_gpu_saved8 import inputs

from sgnn_amd import nn as snn

pytestmark = pytest.mark.gpu


def test_products_of_two_numbers(gpu_device):
    """An fp32 product takes six of the nine products of two numbers' three parts; what it leaves out is at
    most 2^-22 of the whole.  Numbers 1 + 2^-7 - m 2^-23, for which every sum on the way is exact (all are
    multiples of 2^-23 below 2), so that nothing else is off; the result is no further than that."""
    m = torch.tensor([1, 2, 5, 31, 64, 127, 128])
    v = (1 + 2.0 ** -7 - m.double() * 2.0 ** -23).float()
    assert torch.equal(v.double(), 1 + 2.0 ** -7 - m.double() * 2.0 ** -23)
    want = v.double()[:, None] * v.double()[None]
    x, w = v[:, None].to(gpu_device), v[:, None].to(gpu_device)
    y = snn.linear_saved_int8(x, w).double().cpu()
    assert bool(((y - want).abs() <= 2.0 ** -22 * want).all())
    x.requires_grad_()
    eye = torch.zeros(7, 7, device=gpu_device)
    eye[:, 3] = v.to(gpu_device)                     # dx = grad . weight, one product each
    snn.linear_saved_int8(x, w).backward(eye)
    want = v.double() * v.double()[3]
    assert bool(((x.grad[:, 0].double().cpu() - want).abs() <= 2.0 ** -22 * want).all())


@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
@pytest.mark.parametrize("n,F,H", [(300, 100, 24), (4000, 602, 100), (70000, 64, 40), (9000, 256, 200)])
def test_fp32_layer_is_as_exact_as_torch(gpu_device, n, F, H, slope):
    """Output and input gradient in fp32 are as far from 64 bits as torch's products: four times at most
    (sums over six products for one of theirs: sqrt(6) times the roundings) and a rounding."""
    x = inputs(n, F, torch.float32, gpu_device, seed=n, spread=0.5)
    g = torch.Generator().manual_seed(H)
    w = (torch.randn(H, F, generator=g) / F ** 0.5).to(gpu_device)
    grad = torch.randn(n, H, generator=g).to(gpu_device)
    xs = x.clone().requires_grad_()
    y = snn.linear_saved_int8(xs, w, slope=slope)
    y.backward(grad)
    s = torch.tensor(slope, dtype=torch.float32).double().item()

    def layer(t):
        a = x.to(t)
        factor = torch.where(a > 0, torch.ones_like(a), torch.full_like(a, s))
        return (a * factor) @ w.to(t).t(), (grad.to(t) @ w.to(t)) * factor
    for got, plain, want in zip((y.detach(), xs.grad), layer(torch.float32), layer(torch.float64)):
        off, usual = ((a.double() - want).norm() / want.norm() for a in (got, plain))
        assert off <= 4 * usual + 2.0 ** -23


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(gpu_device, grad):
    """A forward-mode derivative is refused whether or not an operand requires a gradient, never lost."""
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.randn(5, 8, device=gpu_device), torch.randn(3, 8, device=gpu_device, requires_grad=grad)
    for dual in (0, 1):
        with forward_ad.dual_level():
            args = [x, w]
            args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
            with pytest.raises(RuntimeError, match="forward"):
                snn.linear_saved_int8(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                snn.linear_saved_int8(*args)
    assert snn.linear_saved_int8(x, w.detach()).grad_fn is None


@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
def test_input_grad_is_a_tensor_of_its_own(gpu_device, slope):
    """Writing to the result leaves the gradient that it was made of alone, whatever the slope."""
    saved = snn.save_int8(inputs(20, 40, torch.float32, gpu_device, seed=1), slope)
    wide = torch.randn(20, 50, device=gpu_device)
    for grad in (torch.randn(20, 40, device=gpu_device), wide[:, 3:43], wide[:1, :40].expand(20, 40)):
        before = grad.clone()
        dx = saved.input_grad(grad)
        assert slope != 1.0 or torch.equal(dx, grad)
        dx.add_(1.0)
        assert torch.equal(grad, before)


@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
@pytest.mark.parametrize("n,F,H", [(300, 100, 24), (5000, 602, 100), (66000, 64, 40), (9000, 256, 200)])
def test_fp32_weight_gradient_is_as_exact_as_torch(gpu_device, n, F, H, slope):
    """The weight gradient formed from the codes is as far from 64 bits as torch's product of the values they
    stand for: four times at most (three products a pair: sqrt(3) times the roundings) and a rounding.
    With 16 bits of the gradient it would be off by 2^-17 at least."""
    saved = snn.save_int8(inputs(n, F, torch.float32, gpu_device, seed=n, spread=0.5), slope)
    grad = torch.randn(n, H, generator=torch.Generator().manual_seed(H)).to(gpu_device)
    value = saved.restore()
    want = grad.double().t() @ value.double()
    off, usual = ((a.double() - want).norm() / want.norm() for a in (saved.weight_grad(grad), grad.t() @ value))
    assert off <= 4 * usual + 2.0 ** -23


@pytest.mark.parametrize("slope", [0.0, 0.2, 0.9, 1.0])
@pytest.mark.parametrize("n,F,H", [(3, 7, 33), (130, 31, 64), (400, 90, 24), (66000, 40, 20), (9001, 70, 200), (500, 300, 16)])
def test_bf16_activations_in_the_product(gpu_device, n, F, H, slope):
    """Activations that the slope moves are no bf16 numbers any more; they enter the product with 16 bits (two
    bf16 numbers: half a step of half a step, 2^-16).  The output is off by that, by its sum of up to two
    products a feature in 32 bits (2^-23 an addition) and by its own rounding, half a step of 2^-8."""
    x = inputs(n, F, torch.bfloat16, gpu_device, seed=n, spread=0.5)
    w = (torch.randn(H, F, generator=torch.Generator().manual_seed(H)) / F ** 0.5).to(gpu_device, torch.bfloat16)
    xd, wd = x.double(), w.double()
    act = torch.where(xd > 0, xd, torch.tensor(slope, dtype=torch.float32).double().item() * xd)
    want = act @ wd.t()
    off = (2.0 ** -16 + (2 * F + 8) * 2.0 ** -23) * (act.abs() @ wd.abs().t())
    y = snn.linear_saved_int8(x, w, slope=slope).double()
    assert bool(((y - want).abs() <= off + 2.0 ** -8 * (want.abs() + off) + 2.0 ** -134).all())


@pytest.mark.parametrize("slope", [0.0, 0.2, 1.0])
def test_infinite_bf16_activations(gpu_device, slope):
    """In bf16 an infinity stays one on the way to the output, and what is beside it is what it was."""
    x = inputs(70, 40, torch.bfloat16, gpu_device, seed=2)
    w = (torch.randn(30, 40, generator=torch.Generator().manual_seed(1)) / 6 + 0.01).to(gpu_device, torch.bfloat16)
    before = snn.linear_saved_int8(x, w, slope=slope)
    x[5, 3], x[60, 39] = float("inf"), -float("inf")
    y = snn.linear_saved_int8(x, w, slope=slope)
    assert torch.equal(y[5].float(), float("inf") * torch.sign(w[:, 3].float()))
    if slope:
        assert torch.equal(y[60].float(), -float("inf") * torch.sign(w[:, 39].float()))
    beside = [r for r in range(70) if r not in (5, 60)]
    assert torch.equal(y[beside], before[beside])


@pytest.mark.parametrize("slope", [0.2, 1.0])
def test_activations_of_more_than_2_to_the_31_elements(gpu_device, slope):
    """2.2 million rows of 1000 features in bf16: codes, values, outputs and gradients of the rows at the end
    and around element 2^31 are those of these rows alone."""
    n, F, H = 2_200_000, 1000, 8
    x = torch.randn(n, F, device=gpu_device, dtype=torch.bfloat16)
    w = torch.randn(H, F, device=gpu_device).bfloat16() / 32
    grad = torch.randn(n, H, device=gpu_device).bfloat16()
    parts = [slice(2 ** 31 // F - 40, 2 ** 31 // F + 40), slice(n - 70, n)]
    saved = snn.save_int8(x, slope)
    value = saved.restore()
    act = saved.input_grad(x)
    xs = x.requires_grad_()
    y = snn.linear_saved_int8(xs, w, slope=slope)
    (dx,) = torch.autograd.grad(y, xs, grad)
    for at in parts:
        own = x[at].detach().clone()
        alone = snn.save_int8(own, slope)
        assert torch.equal(saved.codes[at], alone.codes) and torch.equal(saved.steps[at], alone.steps)
        assert torch.equal(value[at], alone.restore()) and torch.equal(act[at], alone.input_grad(own))
        own.requires_grad_()
        z = snn.linear_saved_int8(own, w, slope=slope)
        # few rows share the features between wavefronts, so their sums have another order: (2 F + 8)
        # additions of 2^-23 on either side and two roundings of half a step
        near = 2 * (2 * F + 8) * 2.0 ** -23 * 2 * (own.detach().float().abs() @ w.float().abs().t()) + 2.0 ** -7 * z.abs()
        assert bool(((y[at] - z).abs() <= near).all())
        assert torch.equal(dx[at], torch.autograd.grad(z, own, grad[at])[0])
    only = torch.zeros_like(grad)
    for at in parts:
        only[at] = grad[at]
    want = sum(grad[at].double().t() @ value[at].double() for at in parts)
    size = sum(grad[at].double().abs().t() @ value[at].double().abs() for at in parts)
    got = saved.weight_grad(only).double()
    assert bool(((got - want).abs() <= (3 * 150 + 1032) * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("slope", [1.5, 7.0])
def test_slopes_beyond_one(gpu_device, dtype, slope):
    """Output and input gradient with a slope that enlarges: sums in 32 bits of up to six products a term,
    the sum's error times the slope, one rounding (half a step of 2^-24 or 2^-8) of the result; bf16
    activations with 16 bits."""
    n, F, H = 700, 90, 40
    x = inputs(n, F, dtype, gpu_device, seed=5, spread=0.5).requires_grad_()
    g = torch.Generator().manual_seed(6)
    w = (torch.randn(H, F, generator=g) / 9).to(gpu_device, dtype)
    grad = torch.randn(n, H, generator=g).to(gpu_device, dtype)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    y = snn.linear_saved_int8(x, w, slope=slope)
    y.backward(grad)
    xd, wd, gd = x.detach().double(), w.double(), grad.double()
    factor = torch.where(xd > 0, torch.ones_like(xd), torch.full_like(xd, slope))
    act = factor * xd
    off = (2.0 ** -16 * (half > 2.0 ** -20) + 2.0 ** -24 + (6 * F + 20) * 2.0 ** -23) * (act.abs() @ wd.abs().t())
    want = act @ wd.t()
    assert bool(((y.detach().double() - want).abs() <= off + half * (want.abs() + off)).all())
    want = (gd @ wd) * factor
    off = (6 * H + 21) * 2.0 ** -23 * (gd.abs() @ wd.abs()) * factor
    assert bool(((x.grad.double() - want).abs() <= off + half * (want.abs() + off)).all())
