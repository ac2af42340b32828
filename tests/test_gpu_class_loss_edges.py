"""``class_cross_entropy`` where it can go wrong beside its sizes: what the label's element of dz keeps,
weights whose rows lie far apart, rows without a class, small and large heads through every kernel.

Tolerances are those of ``test_gpu_class_loss``, but where a test says otherwise."""
import pytest
import torch
from test_gpu_class_loss import DTYPES, HALF_STEP, U, check, close, make, reference  # noqa: F401

from sgnn_amd import nn as snn

pytestmark = pytest.mark.gpu


def gradients(x, w, labels, idx=None, g=None):
    """Both gradients of the mean (or of the rows' losses weighted by g)."""
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    if g is None:
        snn.class_cross_entropy(xs, ws, labels, idx=idx).backward()
    else:
        (snn.class_cross_entropy(xs, ws, labels, idx=idx, reduction="none") * g).sum().backward()
    return xs.grad, ws.grad


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("stored", ["by class", "by feature"])
@pytest.mark.parametrize("B,D,V", [(300, 64, 100), (300, 100, 2000), (513, 192, 700), (300, 256, 300), (1500, 256, 5000),
                                   (300, 300, 90), (2500, 320, 3000), (33, 257, 1000), (12000, 264, 12001)])
def test_label_elements_in_the_weight_gradient(gpu_device, B, D, V, stored, by_row):
    """bf16.  A class's gradient is mostly the label's elements of dz; they reach it with 16 bits (two bf16
    numbers: half a step of half a step, 2^-16) or more, the other elements of dz with 8 (2^-8), and the
    result is rounded once.  Bounds as in ``reference``, with 2^-16 in the place of 2^-8 for those
    elements.  Logits in which the label stands out but is not certain, so that p - 1 is no bf16 number."""
    x, w, labels = make(B, D, V, torch.bfloat16, gpu_device, seed=B + V)
    labels[5] = -1
    x = (x.float() + 2.5 * w.float()[labels.clamp_min(0)]).bfloat16()
    g = torch.linspace(-1.0, 2.0, B, device=gpu_device) if by_row else None
    live = labels >= 0
    weight = torch.where(live, g.double() if by_row else torch.ones(B, device=gpu_device).double() / int(live.sum()),
                         torch.zeros(B, device=gpu_device).double())[:, None]
    xd, wd = x.double() * live[:, None], w.double()
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    ez = ((6 * D + 20) * U * size).amax(1, keepdim=True)
    p = torch.softmax(z, 1)
    delta = 2 * ez + 4 * U * (1 + z.amax(1, keepdim=True) - z) + (V / 4 + 1100) * U
    at = labels.clamp_min(0)[:, None]
    one = torch.zeros_like(p).scatter_(1, at, 1.0)
    dz = (p - one) * weight
    keep = torch.full_like(p, 2.0 ** -8).scatter_(1, at, 2.0 ** -16)
    edz = p * weight.abs() * torch.expm1(delta) + 4 * U * (p + one) * weight.abs() + keep * dz.abs()
    want = dz.t() @ xd
    bound = edz.t() @ xd.abs() + (6 * B + 600) * U * ((dz.abs() + edz).t() @ xd.abs())
    bound = bound + HALF_STEP[torch.bfloat16] * (want.abs() + bound) + 1e-38
    if stored == "by feature":
        w = w.t().contiguous().t()
    _, dw = gradients(x, w, labels, g=g)
    close(dw, want, bound, "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [5, 40])
@pytest.mark.parametrize("D,V,stride", [(64, 96, 36_000_000), (256, 70, 1 << 26), (128, 96, 34_087_040),
                                        (192, 96, 34_087_048), (320, 70, 36_000_000)])
def test_classes_far_apart(gpu_device, dtype, B, D, V, stride):
    """Rows of the weight so far apart that a step's offsets pass 32 bits: bit for bit the results of a
    copy with its rows together.  (What lies between the rows is never touched.)"""
    t = DTYPES[dtype]
    x, w, labels = make(B, D, V, t, gpu_device, seed=D)
    far = torch.empty_strided((V, D), (stride, 1), dtype=t, device=gpu_device)
    far.copy_(w)
    want, got = check(x, w, labels), check(x, far, labels)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("B,D,V", [(5, 40, 3000), (30, 300, 700), (128, 64, 128), (200, 100, 900), (513, 602, 1000),
                                   (300, 256, 5000), (12000, 40, 12001)])
def test_fp32_is_as_exact_as_torch(gpu_device, B, D, V):
    """Losses and gradients of fp32 operands are as far from the definition in 64 bits as those of torch's
    operators in fp32.  The sums here run over six products where those run over one: with roundings of
    either sign that is sqrt(6) = 2.5 times as far, 4 is allowed, and a rounding (2^-23) beside it.  With
    16 bits of each operand (half of the six products) it would be 2^-17 at least, 30 times the roundings
    of sums of these lengths."""
    x, w, labels = make(B, D, V, torch.float32, gpu_device, seed=B)
    dx, dw = gradients(x, w, labels)
    rows = snn.class_cross_entropy(x, w, labels, reduction="none")
    answers = []
    for t in (torch.float32, torch.float64):
        a, b = x.to(t).requires_grad_(), w.to(t).requires_grad_()
        losses = torch.nn.functional.cross_entropy(a @ b.t(), labels, reduction="none")
        answers.append((losses.detach(), *torch.autograd.grad(losses.mean(), (a, b))))
    for got, plain, want, what in zip((rows, dx, dw), *answers, ("row losses", "dx", "dweight")):
        assert relative(got, want) <= 4 * relative(plain, want) + 2.0 ** -23, what


@pytest.mark.parametrize("unit", [False, True])
@pytest.mark.parametrize("B,D,V", [(64, 128, 4096), (300, 33, 5001), (64, 128, 4095)])
def test_stacked_head_with_rows_without_a_class(gpu_device, B, D, V, unit):
    """The label head of the stacked training treats labels and indices out of range alike on either side of
    the class count from which it runs over the classes in pieces: they add nothing to the loss, count in
    the mean, and dz = softmax / B.  Loss and gradients against that in 64 bits, with the bounds of
    ``reference`` for rows of weight 1 / B (whose own dz is p / B alone: a share of the same bound)."""
    from sgnn_amd.stacked import _head_cross_entropy
    x, w, labels = make(B, D, V, torch.float32, gpu_device, seed=B, nodes=B + 9)
    labels[:5] = torch.tensor([-1, V, -100, 2 ** 40, V - 1], device=gpu_device)
    idx = torch.arange(B, device=gpu_device)
    idx[7], idx[8] = -1, B + 9
    E, Wt = x.clone().requires_grad_(), w.t().contiguous().requires_grad_()
    loss = _head_cross_entropy(E, Wt, labels, idx, unit=unit)
    loss.backward()
    dead = torch.tensor([0, 1, 2, 3, 7, 8], device=gpu_device)
    known = labels.clone()
    known[:4] = 0
    inside = idx.clone()
    inside[7:9] = 0
    ref = reference(x, w, known, inside)             # every row with a class
    p = torch.softmax(x.double() @ w.double().t(), 1)
    dz = p.clone()
    alive = torch.ones(B, dtype=torch.bool, device=gpu_device)
    alive[dead] = False
    dz[torch.arange(B, device=gpu_device)[alive], labels[idx[alive]]] -= 1
    dz /= B
    close(loss.detach(), ref["loss"][alive].sum() / B, ref["loss_bound"].mean() + 1e-30, "mean loss")
    close(E.grad, dz @ w.double(), ref["dx_bound"], "dE")
    close(Wt.grad.t(), dz.t() @ x.double(), ref["dw_bound"], "dWt")


@pytest.mark.parametrize("B,D,V", [(5, 40, 300), (30, 64, 700), (200, 48, 500)])
def test_rows_without_a_class_that_count(gpu_device, B, D, V):
    """The same through every kernel of fp32 operands, bit for bit the results of the rows' losses for rows
    with a class; and the call is refused in bf16, where no caller needs it."""
    from sgnn_amd._lib import SgnnHipError
    from sgnn_amd.class_loss import _ClassXent
    x, w, labels = make(B, D, V, torch.float32, gpu_device, seed=D)
    labels[1], labels[3] = -1, V
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    rows = _ClassXent.apply(xs, ws, labels, None, False, True)
    assert torch.equal(rows.detach(), snn.class_cross_entropy(x, w, labels, reduction="none"))
    rows.sum().backward()
    p = torch.softmax(x.double() @ w.double().t(), 1)
    for r in range(B):
        if r not in (1, 3):
            p[r, labels[r]] -= 1
    known = labels.clone()
    known[1] = known[3] = 0
    ref = reference(x, w, known, g=torch.ones(B, device=gpu_device))
    close(xs.grad, p @ w.double(), ref["dx_bound"], "dx")
    close(ws.grad, p.t() @ x.double(), ref["dw_bound"], "dweight")
    with pytest.raises(SgnnHipError):
        _ClassXent.apply(x.bfloat16(), w.bfloat16(), labels, None, True, True)


def test_stacked_head_refuses_nothing_it_took(gpu_device):
    """Heads of thousands of classes with more features than the class loss takes, and labels or indices
    longer than the batch (the first of them count): the loss of the stock product, as with fewer classes."""
    from sgnn_amd.stacked import _cross_entropy, _head_cross_entropy
    g = torch.Generator(gpu_device).manual_seed(0)
    E = torch.randn(4, 65600, device=gpu_device, generator=g, requires_grad=True)
    Wt = torch.randn(65600, 4100, device=gpu_device, generator=g) / 256
    labels = torch.tensor([3, 4099, 0, 17, 5, 6], device=gpu_device)
    loss = _head_cross_entropy(E, Wt, labels, None)
    want = _cross_entropy(E.matmul(Wt), labels, None)
    assert torch.equal(loss, want)
    assert torch.equal(torch.autograd.grad(loss, E)[0], torch.autograd.grad(want, E)[0])
    E, Wt = E[:, :40].detach(), Wt[:40].contiguous()
    want = _cross_entropy(E.matmul(Wt), labels[:4], None)
    assert torch.allclose(_head_cross_entropy(E, Wt, labels, None), want, rtol=1e-5, atol=0)
    idx = torch.tensor([5, 4, 1, 0, 2, 2, 3], device=gpu_device)
    want = _cross_entropy(E.matmul(Wt), labels, idx[:4])
    assert torch.allclose(_head_cross_entropy(E, Wt, labels, idx), want, rtol=1e-5, atol=0)


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("B,D,V", [(7, 40, 90), (200, 48, 150), (130, 64, 300), (200, 100, 2000), (70, 192, 100),
                                   (300, 256, 300), (100, 300, 200)])
def test_masked_classes_and_rows_without_a_class(gpu_device, B, D, V, by_row):
    """bf16.  Classes masked by an infinite weight (p is 0 in every row that counts) beside rows without a
    class, the last among them: the weight's gradient is that of the other classes, 0 in the masked ones."""
    x, w, labels = make(B, D, V, torch.bfloat16, gpu_device, seed=B)
    x[:, 0] = x[:, 0].abs() + 1
    keep = V - 10
    labels %= keep
    labels[2], labels[B // 2], labels[B - 1] = -1, V, -1
    masked = w.clone()
    masked[keep:, 0] = -float("inf")
    g = torch.linspace(0.5, 1.5, B, device=gpu_device) if by_row else None
    _, dw = gradients(x, masked, labels, g=g)
    labels[B // 2] = -1
    ref = reference(x, w[:keep], labels, g=g)
    close(dw[:keep], ref["dw"], ref["dw_bound"], "dweight")
    assert bool((dw[keep:] == 0).all())


# up to 32 rows (bf16: 16), rows in registers (bf16 up to 256 features), tiles, tiles in several pieces
EVERY_WAY = [(5, 40, 300), (16, 100, 500), (30, 300, 400), (150, 64, 400), (150, 300, 400), (12000, 264, 12001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stored", ["by class", "by feature"])
@pytest.mark.parametrize("B,D,V", EVERY_WAY)
def test_row_gradients_every_way(gpu_device, dtype, B, D, V, stored):
    """A gradient of its own for every row, some of them 0 or negative, through every kernel."""
    x, w, labels = make(B, D, V, DTYPES[dtype], gpu_device, seed=B + 1)
    labels[B // 3] = -1
    g = torch.randn(B, generator=torch.Generator().manual_seed(B)).to(gpu_device)
    g[B // 2] = 0.0
    if stored == "by feature":
        w = w.t().contiguous().t()
    dx, dw = gradients(x, w, labels, g=g)
    ref = reference(x, w, labels, g=g)
    close(dx, ref["dx"], ref["dx_bound"], "dx")
    close(dw, ref["dw"], ref["dw_bound"], "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stored", ["by class", "by feature"])
@pytest.mark.parametrize("B,D,V", EVERY_WAY)
def test_rows_without_a_class_every_way(gpu_device, dtype, B, D, V, stored):
    """Labels and indices out of range whose rows hold NaN and infinities, a repeated index, the last row
    among them: losses and gradients are those of the other rows."""
    x, w, labels = make(B, D, V, DTYPES[dtype], gpu_device, seed=B + 2, nodes=B + 4)
    labels[:2] = torch.tensor([-1, V], device=gpu_device)
    idx = torch.arange(B, device=gpu_device) + 2
    idx[1], idx[3], idx[B - 1] = 0, -1, B + 4
    idx[2] = idx[4]
    if B > 5:
        idx[B // 2] = 1
    dead = [1, 3, B - 1] + ([B // 2] if B > 5 else [])
    for k, r in enumerate(dead):
        x[r] = (float("nan"), float("inf"), -float("inf"))[k % 3]
    if stored == "by feature":
        w = w.t().contiguous().t()
    dx, dw, loss = check(x, w, labels, idx)
    assert bool((dx[dead] == 0).all()) and bool(torch.isfinite(dw).all()) and bool(torch.isfinite(loss))


@pytest.mark.parametrize("dtype,B", [("bf16", 4), ("bf16", 70), ("f32", 4), ("f32", 70)])
def test_weights_of_more_than_2_to_the_31_elements(gpu_device, dtype, B):
    """8.5 million classes of 256 features.  All but 300 of them, at both ends and around element 2^31, are
    masked by a large negative weight on a feature that is 1 (p is 0, exactly): losses and gradients are
    those of the 300."""
    t = DTYPES[dtype]
    V, D = 8_500_000, 256
    at = torch.cat([torch.arange(100), torch.arange(100) + 2 ** 31 // D - 50, torch.arange(100) + V - 100]).to(gpu_device)
    x, w, labels = make(B, D, 300, t, gpu_device, seed=B)
    x[:, 0], w[:, 0] = 1.0, 0.0
    big = torch.zeros(V, D, dtype=t, device=gpu_device)
    big[:, 0] = -2.0 ** 20
    big[at] = w
    labels[0] = 299
    ref = reference(x, w, labels)
    dx, dw = gradients(x, big, at[labels])
    # a masked class adds an exact 0, so the sums' roundings are those of 300 classes and of joining up to 768
    # workgroups' shares: within the (V / 4 + 1100) u of the bound for V = 300
    rows = snn.class_cross_entropy(x, big, at[labels], reduction="none")
    close(rows, ref["loss"], ref["loss_bound"], "row losses")
    close(dx, ref["dx"], ref["dx_bound"], "dx")
    close(dw[at], ref["dw"], ref["dw_bound"], "dweight")
    dw[at] = 0
    assert not bool(dw.any())
