"""Activations kept in 8 bits (``sgnn_amd.saved8``): codes and steps bit for bit against a 64-bit
restatement of their definition, the gradients formed from them against 64-bit products.

Tolerances.  Codes, steps and restored values are exact.  A weight gradient is a sum of exact
products in 32 bits: with n rows and three planes per 32-bit gradient it has at most 3 n + 8
additions (the chunks' included), each off by at most 2^-23 of the running sum (2^-24 for a
rounding, twice that where the matrix unit cuts off), whose magnitude is at most
``|grad|.T @ |value|``.  A bf16 result adds half a step, 2^-8 of its value; below 2^-126 steps
stop shrinking and half of one is 2^-134 (bf16: 2^-126 times 2^-7, halved) or 2^-150 (fp32)."""
import numpy as np
import pytest
import torch

from sgnn_amd import nn as snn
from sgnn_amd.saved8 import SavedInt8

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134}        # half a step of the subnormal numbers


def reference(x, slope):
    """codes, biased steps and values from the definition (numpy, 64 bits)."""
    x32 = x.float().cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        a32 = np.where(x32 > 0, x32, np.float32(slope) * x32).astype(np.float32)
    if slope == 0.0:
        a32 = np.where(x32 > 0, x32, np.where(np.isnan(x32), x32, np.float32(0)))
    n, F = a32.shape
    G = -(-F // 32)
    wide = np.zeros((n, G * 32))
    wide[:, :F] = a32
    positive = np.zeros((n, G * 32), bool)
    positive[:, :F] = x32 > 0
    b = wide.reshape(n, G, 32)
    pos = positive.reshape(n, G, 32)
    bad = ~np.isfinite(b).all(2)
    clean = np.where(bad[:, :, None], 0.0, b)
    peak = np.abs(clean).max(2)
    s = np.full((n, G), -125)
    todo = np.ones((n, G), bool)
    for k in range(-125, 122):                       # the smallest exponent that holds the group
        step = 2.0 ** k
        holds = (np.rint(peak / step) <= 127) if slope == 1.0 else (peak <= 128 * step)
        if k == 121:                                 # the last step: what it does not hold is cut off
            holds[:] = True
        s[todo & holds] = k
        todo &= ~holds
    assert not todo.any()
    step = (2.0 ** s)[:, :, None]
    if slope == 1.0:
        q = np.rint(clean / step).clip(-127, 127)
        value = q * step
    else:
        q = np.ceil(clean / step) - 1
        q = np.where(pos, q.clip(0, 127), q.clip(-128, -1))
        value = (q + 0.5) * step
        if slope == 0.0:
            value = np.where(q < 0, 0.0, value)
    value = np.where(bad[:, :, None], np.nan, value)
    biased = np.where(bad, 255, s + 127)
    return q.reshape(n, -1)[:, :F], biased, value.reshape(n, -1)[:, :F], bad


def inputs(n, F, dtype, device, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, F, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
    x[torch.rand(n, F, generator=g) < 0.2] = 0.0
    return x.to(device=device, dtype=dtype)


def check_saved(x, slope):
    q, biased, value, bad = reference(x, slope)
    saved = snn.save_int8(x, slope=slope)
    F = x.shape[1]
    assert np.array_equal(saved.steps.cpu().numpy().astype(int), biased)
    good = np.repeat(~bad, 32, axis=1)[:, :F]
    got = saved.codes.cpu().numpy().astype(int)[:, :F]
    assert np.array_equal(got[good], q.astype(int)[good])
    if slope != 1.0:
        assert np.array_equal(got < 0, ~(x.float().cpu().numpy() > 0))
    for t in (torch.float32, torch.bfloat16):
        assert np.array_equal(saved.restore(t).double().cpu().numpy(), value, equal_nan=True)
    return saved


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
@pytest.mark.parametrize("n,F", [(1, 1), (3, 31), (5, 32), (7, 33), (300, 100), (64, 602), (2, 5000), (1000, 8)])
def test_codes(gpu_device, dtype, slope, n, F):
    check_saved(inputs(n, F, DTYPES[dtype], gpu_device, seed=n + F), slope)


@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
def test_codes_at_the_borders(gpu_device, slope):
    """Powers of two, the rounding borders 127.5 and 128, zeros of both signs, the smallest and
    largest numbers, subnormals."""
    rows = []
    for top in (127.0, 127.49999, 127.5, 127.50001, 128.0, 128.00002, 255.0, 1.0, 2.0 ** -100, 2.0 ** 100):
        rows.append([top] + [top * k / 128 for k in range(-15, 16)])
    rows.append([0.0, -0.0] * 16)
    rows.append([3.4028234e38, -3.4028234e38] + [1e38, 1e-38] * 15)
    rows.append([2.0 ** -126, 2.0 ** -127, 2.0 ** -149, -(2.0 ** -149)] + [2.0 ** -k for k in range(120, 148)])
    rows.append([1.0] + [2.0 ** -149, -(2.0 ** -149)] * 15 + [0.0])
    rows.append([-1.0 - k for k in range(32)])
    check_saved(torch.tensor(rows, dtype=torch.float32, device=gpu_device), slope)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
def test_groups_with_values_that_are_no_numbers(gpu_device, dtype, slope):
    x = inputs(6, 100, DTYPES[dtype], gpu_device, seed=3)
    x[0, 3], x[1, 40], x[2, 99], x[3, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    saved = check_saved(x, slope)
    grad = torch.ones(6, 4, dtype=DTYPES[dtype], device=gpu_device)
    dw = saved.weight_grad(grad).float().cpu().numpy()
    bad = np.isnan(reference(x, slope)[2]).any(0)
    assert np.array_equal(np.isnan(dw), np.broadcast_to(bad, dw.shape))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_offsets(gpu_device, dtype):
    """Rows at odd strides and odd offsets, a transposed view, an expanded row: the same codes as
    their contiguous copies."""
    base = inputs(50, 131, DTYPES[dtype], gpu_device, seed=5)
    for view in (base[:, 1:100], base[::2, 3:], base.t()[:77], base[:1].expand(50, 131), base[7:8]):
        for slope in (0.0, 1.0):
            a, b = snn.save_int8(view, slope), snn.save_int8(view.contiguous(), slope)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.steps, b.steps)
    saved = snn.save_int8(base, 0.2)
    wide = inputs(50, 300, DTYPES[dtype], gpu_device, seed=6)
    for grad in (wide[:, 1:34], wide.t()[:50, :40], wide[:1, :9].expand(50, 9), wide[:, :64]):
        assert torch.equal(saved.weight_grad(grad), saved.weight_grad(grad.contiguous()))
    for grad in (wide[:, 1:132], wide[:1, :131].expand(50, 131)):
        assert torch.equal(saved.input_grad(grad), saved.input_grad(grad.contiguous()))


def check_weight_grad(saved, grad):
    value = saved.restore(torch.float32).double()
    g = grad.double()
    want = g.t() @ value
    size = g.abs().t() @ value.abs()
    got = saved.weight_grad(grad)
    assert got.dtype == grad.dtype and got.shape == want.shape
    n = grad.shape[0]
    bound = (3 * n + 8) * 2.0 ** -23 * size * (1 + 2 * HALF_STEP[grad.dtype]) + HALF_STEP[grad.dtype] * want.abs()
    assert bool(((got.double() - want).abs() <= bound + LEAST[grad.dtype]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
@pytest.mark.parametrize("n,F,H", [(1, 1, 1), (2, 33, 5), (31, 32, 32), (32, 256, 33), (33, 257, 64), (100, 602, 65),
                                   (777, 40, 130), (5000, 100, 128), (4096, 300, 16), (20000, 64, 300),
                                   (300, 2100, 1100), (3000, 700, 1000), (2000, 1300, 900)])
def test_weight_grad(gpu_device, dtype, slope, n, F, H):
    x = inputs(n, F, DTYPES[dtype], gpu_device, seed=n, spread=0.5)
    grad = torch.randn(n, H, generator=torch.Generator().manual_seed(H)).to(gpu_device, DTYPES[dtype])
    check_weight_grad(snn.save_int8(x, slope), grad)


def test_weight_grad_takes_either_type(gpu_device):
    x = inputs(500, 70, torch.bfloat16, gpu_device, seed=1)
    saved = snn.save_int8(x, 0.0)
    for dtype in DTYPES.values():
        check_weight_grad(saved, torch.randn(500, 20, device=gpu_device).to(dtype))


def test_weight_grad_repeats_bit_for_bit(gpu_device):
    saved = snn.save_int8(inputs(30000, 96, torch.float32, gpu_device, seed=2), 0.2)
    grad = torch.randn(30000, 48, device=gpu_device)
    first = saved.weight_grad(grad)
    for _ in range(3):
        assert torch.equal(first, saved.weight_grad(grad))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_that_are_no_numbers(gpu_device, dtype):
    """A NaN or infinite gradient reaches its own unit's row of dW and no other."""
    x = inputs(200, 40, DTYPES[dtype], gpu_device, seed=4).abs() + 1
    saved = snn.save_int8(x, 0.0)
    grad = torch.randn(200, 6, device=gpu_device).to(DTYPES[dtype])
    grad[5, 1], grad[100, 4] = float("nan"), float("inf")
    dw = saved.weight_grad(grad).float()
    assert bool(torch.isnan(dw[1]).all()) and bool(torch.isfinite(dw[[0, 2, 3, 5]]).all())
    assert bool((~torch.isfinite(dw[4])).all())
    dx = saved.input_grad(torch.full((200, 40), float("inf"), device=gpu_device))
    assert bool(torch.isinf(dx).all())
    off = snn.save_int8(-x, 0.0).input_grad(torch.full((200, 40), float("nan"), device=gpu_device))
    assert bool((off == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 0.2, 1.0])
def test_input_grad(gpu_device, dtype, slope):
    x = inputs(129, 70, DTYPES[dtype], gpu_device, seed=8)
    grad = torch.randn(129, 70, device=gpu_device).to(DTYPES[dtype])
    want = torch.where(x > 0, grad.double(), float(np.float32(slope)) * grad.double())
    got = snn.save_int8(x, slope).input_grad(grad)
    assert got.dtype == grad.dtype
    assert bool(((got.double() - want).abs() <= HALF_STEP[grad.dtype] * want.abs()).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
def test_linear_layer(gpu_device, dtype, slope):
    """Output and input gradient are the full activation's, the weight's is that of the codes."""
    t = DTYPES[dtype]
    x = inputs(400, 90, t, gpu_device, seed=11, spread=0.5).requires_grad_()
    w = (torch.randn(24, 90, device=gpu_device) / 9).to(t).requires_grad_()
    grad = torch.randn(400, 24, device=gpu_device).to(t)
    y = snn.linear_saved_int8(x, w, slope=slope)
    y.backward(grad)
    check_layer(x, w, grad, y, slope)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("slope", [0.0, 1.0, 0.2])
@pytest.mark.parametrize("n,F,H", [(1, 1, 1), (3, 7, 33), (130, 31, 64), (129, 33, 65), (200, 65, 128), (64, 602, 130),
                                   (257, 96, 200), (500, 300, 16), (66000, 40, 20), (65537, 33, 70),
                                   (20000, 100, 20), (17000, 130, 70), (9001, 70, 200), (4000, 200, 130)])
def test_linear_layer_sizes(gpu_device, dtype, slope, n, F, H):
    t = DTYPES[dtype]
    g = torch.Generator().manual_seed(n + F + H)
    x = inputs(n, F, t, gpu_device, seed=n, spread=0.5).requires_grad_()
    w = (torch.randn(H, F, generator=g) / F ** 0.5).to(gpu_device, t).requires_grad_()
    grad = torch.randn(n, H, generator=g).to(gpu_device, t)
    y = snn.linear_saved_int8(x, w, slope=slope)
    y.backward(grad)
    check_layer(x, w, grad, y, slope)


def check_layer(x, w, grad, y, slope):
    t = x.dtype
    F, H = x.shape[1], w.shape[0]
    xd, wd, gd = x.detach().double(), w.detach().double(), grad.double()
    s = float(np.float32(slope))
    act = torch.where(xd > 0, xd, s * xd)
    half = HALF_STEP[t]
    # a rounded activation, a 32-bit sum of up to six products a feature and a rounded result
    bound = (half + (6 * F + 20) * 2.0 ** -23) * (act.abs() @ wd.abs().t()) + half * (act @ wd.t()).abs() + LEAST[t]
    assert bool(((y.detach().double() - act @ wd.t()).abs() <= bound).all())
    dact = gd @ wd
    want = torch.where(xd > 0, dact, s * dact)
    # the same over the units, times the slope and rounded
    bound = (6 * H + 20) * 2.0 ** -23 * (gd.abs() @ wd.abs()) + 1.01 * half * dact.abs() + LEAST[t]
    assert bool(((x.grad.double() - want).abs() <= bound).all())
    assert torch.equal(w.grad, snn.save_int8(x.detach(), slope).weight_grad(grad))
    with torch.no_grad():
        assert torch.equal(snn.linear_saved_int8(x, w, slope=slope), y)
        frozen = snn.linear_saved_int8(x.detach(), w.detach(), slope=slope)
    assert torch.equal(frozen, y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_layer_layouts(gpu_device, dtype):
    """Strided, transposed, offset and expanded operands in the middle of NaN: the results of their copies."""
    t = DTYPES[dtype]
    n, F, H = 150, 45, 37
    xs, ws, gs = (torch.full((r, c), float("nan"), device=gpu_device, dtype=t) for r, c in ((160, 64), (50, 60), (160, 50)))
    x, w, g = xs[3:153, 5:50], ws[2:39, 7:52], gs[1:151, 3:40]
    x.copy_(inputs(n, F, t, gpu_device, seed=1, spread=0.5))
    w.copy_(torch.randn(H, F, device=gpu_device) / 7)
    g.copy_(torch.randn(n, H, device=gpu_device))

    def run(x, w, g):
        xi, wi = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = snn.linear_saved_int8(xi, wi, slope=0.2)
        return (y.detach(), *torch.autograd.grad(y, (xi, wi), g))
    want = run(x.contiguous(), w.contiguous(), g.contiguous())
    for args in ((x, w, g), (x.t().contiguous().t(), w.t().contiguous().t(), g.t().contiguous().t())):
        for a, b in zip(run(*args), want):
            assert torch.equal(a, b)
    one = g[:1].expand(n, H)
    for a, b in zip(run(x, w, one), run(x.contiguous(), w.contiguous(), one.contiguous())):
        assert torch.equal(a, b)


def test_linear_layer_gradient_against_differences(gpu_device):
    """Values that the codes hold exactly (whole numbers with a peak of 127 in every group): the
    gradient is that of the function, checked by central differences in 64 bits."""
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-127, 128, (20, 64), generator=g).float()
    x[:, 0], x[:, 32] = 127.0, -127.0
    w, c = torch.randn(5, 64, generator=g), torch.randn(20, 5, generator=g)
    xg, wg = x.to(gpu_device).requires_grad_(), w.to(gpu_device).requires_grad_()
    ((snn.linear_saved_int8(xg, wg) ** 2) * c.to(gpu_device)).sum().backward()

    def f(a, b):
        return ((a @ b.t()) ** 2 * c.double()).sum().item()
    xd, wd, h = x.double(), w.double(), 1e-4
    for at in ((0, 3), (4, 63), (2, 32)):
        up, down = wd.clone(), wd.clone()
        up[at] += h
        down[at] -= h
        want = (f(xd, up) - f(xd, down)) / (2 * h)
        assert abs(wg.grad[at].item() - want) <= 1e-4 * max(1.0, wg.grad.abs().max().item())
    for at in ((0, 3), (19, 63)):
        up, down = xd.clone(), xd.clone()
        up[at] += h
        down[at] -= h
        want = (f(up, wd) - f(down, wd)) / (2 * h)
        assert abs(xg.grad[at].item() - want) <= 1e-4 * max(1.0, xg.grad.abs().max().item())


def test_layer_keeps_only_the_codes(gpu_device):
    n, F = 100_000, 256
    x = torch.randn(n, F, device=gpu_device)
    w = torch.randn(8, F, device=gpu_device, requires_grad=True)
    before = torch.cuda.memory_allocated(gpu_device)
    hidden = x * 1.0
    y = snn.linear_saved_int8(hidden, w, slope=0.0)
    del hidden
    kept = torch.cuda.memory_allocated(gpu_device) - before - y.numel() * 4
    # codes, steps and y (subtracted at its size): the allocator hands out a block it has whole when
    # less than 1 MiB of it would be left, so each may count for up to 1 MiB more.  x would be 97 MiB.
    assert kept <= n * F + n * F // 32 + 4096 + 3 * 2 ** 20
    y.sum().backward()


def test_empty_and_frozen(gpu_device):
    x = torch.empty(0, 40, device=gpu_device, requires_grad=True)
    w = torch.randn(3, 40, device=gpu_device, requires_grad=True)
    y = snn.linear_saved_int8(x, w, slope=0.0)
    y.sum().backward()
    assert y.shape == (0, 3) and x.grad.shape == (0, 40) and bool((w.grad == 0).all())
    x = torch.randn(30, 40, device=gpu_device)
    y = snn.linear_saved_int8(x, w, slope=0.2)
    w.grad = None
    y.sum().backward()
    assert w.grad is not None
    z = torch.randn(30, 40, device=gpu_device, requires_grad=True)
    snn.linear_saved_int8(z, w.detach(), slope=0.2).sum().backward()
    assert z.grad is not None


def test_captured_layer(gpu_device):
    """Forward and backward recorded into a graph and replayed on new data, with eager work between."""
    x = torch.randn(600, 70, device=gpu_device)
    w = torch.randn(40, 70, device=gpu_device)
    grad = torch.randn(600, 40, device=gpu_device)

    def step(x, w, grad):
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = snn.linear_saved_int8(xs, ws, slope=0.2)
        return (y.detach(), *torch.autograd.grad(y, (xs, ws), grad))
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        step(x, w, grad)
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, grad)
    for k in range(4):
        x.copy_(torch.randn(600, 70, device=gpu_device) * (k + 1))
        grad.copy_(torch.randn(600, 40, device=gpu_device))
        want = step(x, w, grad)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_another_stream(gpu_device):
    x = torch.randn(3000, 100, device=gpu_device)
    grad = torch.randn(3000, 12, device=gpu_device)
    want = snn.save_int8(x, 0.2).weight_grad(grad)
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        got = snn.save_int8(x, 0.2).weight_grad(grad)
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    assert torch.equal(got, want)


def test_refusals_on_the_gpu(gpu_device):
    x = torch.randn(10, 40, device=gpu_device)
    saved = snn.save_int8(x, 0.0)
    for bad in (torch.randn(9, 3, device=gpu_device), torch.randn(10, device=gpu_device)):
        with pytest.raises(ValueError):
            saved.weight_grad(bad)
    with pytest.raises(ValueError):
        saved.input_grad(torch.randn(10, 41, device=gpu_device))
    with pytest.raises(TypeError):
        saved.weight_grad(torch.randn(10, 3, device=gpu_device, dtype=torch.float16))
    with pytest.raises(ValueError):
        SavedInt8(saved.codes[:, :40], saved.steps, (10, 40), 0.0, torch.float32)
    with pytest.raises(ValueError):
        SavedInt8(saved.codes, saved.steps, (10, 70), 0.0, torch.float32)
    with pytest.raises(TypeError):
        saved.restore(torch.float16)
    with pytest.raises(ValueError):
        snn.linear_saved_int8(x, torch.randn(3, 41, device=gpu_device))
    with pytest.raises(TypeError):
        snn.linear_saved_int8(x, torch.randn(3, 40, device=gpu_device, dtype=torch.bfloat16))
    for slope in (-0.1, float("nan"), float("inf"), 1e-50, 1.0 + 1e-12):
        with pytest.raises(ValueError):
            snn.save_int8(x, slope)


def _ring(n, device):
    at = torch.arange(n, device=device)
    return torch.stack([torch.cat([at, (at + 1) % n]), torch.cat([(at + 1) % n, at])])


def test_convolutions_with_checkpoints(gpu_device):
    """The same outputs and input gradients as without, weight gradients within the codes' error
    (half a step, 1/128 of the group's largest value at most, times |grad| summed)."""
    n, edges = 500, _ring(500, gpu_device)
    x = torch.randn(n, 48, device=gpu_device)
    for build in (lambda c: snn.GCNConv(48, 20, checkpoint=c, input_slope=0.0),
                  lambda c: snn.GCNConv(48, 20, checkpoint=c, input_slope=0.1),
                  lambda c: snn.SGConv(48, 20, K=2, checkpoint=c),
                  lambda c: snn.SGConv(48, 20, K=2, checkpoint=c, reorder=False)):
        torch.manual_seed(0)
        full = build(None).to(gpu_device)
        torch.manual_seed(0)
        kept = build("int8").to(gpu_device)
        c = torch.randn(n, 20, device=gpu_device)
        outs = []
        for m in (full, kept):
            xi = x.clone().requires_grad_()
            y = m(xi, edges)
            (y * c).sum().backward()
            outs.append((y.detach(), xi.grad))
        assert torch.allclose(outs[0][0], outs[1][0], rtol=0, atol=1e-5)
        assert torch.allclose(outs[0][1], outs[1][1], rtol=0, atol=1e-5)
        # |A_hat^T c| <= |c| summed over a row's two neighbours and itself, at most 3 max |c|
        bound = n * (x.abs().max() / 128) * 3 * c.abs().max()
        assert bool(((full.lin.weight.grad - kept.lin.weight.grad).abs() <= bound).all())
        assert (full.lin.weight.grad - kept.lin.weight.grad).norm() <= 0.05 * full.lin.weight.grad.norm()


def test_convolutions_refuse():
    with pytest.raises(ValueError):
        snn.GCNConv(4, 4, checkpoint="int4")
    with pytest.raises(ValueError):
        snn.SGConv(4, 4, cached=True, checkpoint="int8")
    with pytest.raises(ValueError):
        snn.GCNConv(4, 4, input_slope=-1.0)
