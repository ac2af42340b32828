"""``class_cross_entropy`` against the definition in 64 bits.

Tolerances, from the arithmetic.  u = 2^-23 bounds an addition or a product in 32 bits (2^-24 for
a rounding, twice that where the matrix unit cuts off).
* a logit is a sum of at most 6 D + 16 products (six for each pair of 32-bit numbers; the three
  left out are below 3 * 2^-24 of the pair): off by ez = (6 D + 20) u |x| |w|^T;
* relative to the row's maximum its exponential is off by 2 ez plus 4 u (1 + z_max - z) for the
  subtraction, the scaling and the function, and a row's sum of them by another (V / 4 + 1100) u
  (a lane adds every fourth class at most, then the lanes, wavefronts and up to 512 splits); so p
  is off by a factor e^(+-delta) and the loss by delta plus 4 u (|max| + |z_y| + log V);
* dz is p g - g [v = y], rounded to bf16 (half a step, 2^-8) or to three planes (u);
* a gradient is a sum of at most 6 K + 600 products of those, rounded once to its type."""
import math

import pytest
import torch

from sgnn_amd import nn as snn

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -23


def make(B, D, V, dtype, device, seed=0, scale=1.5, nodes=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, D, generator=g)
    w = torch.randn(V, D, generator=g) * (scale / math.sqrt(D))
    labels = torch.randint(0, V, (nodes or B,), generator=g)
    return x.to(device, dtype), w.to(device, dtype), labels.to(device)


def reference(x, w, labels, idx=None, g=None):
    """Row losses, gradients for row weights g (the mean's if None), and the bounds above."""
    dtype = x.dtype
    xd, wd = x.double(), w.double()
    B, D = xd.shape
    V = wd.shape[0]
    if idx is None:
        y = labels
    else:
        inside = (idx >= 0) & (idx < labels.numel())
        y = torch.where(inside, labels[idx.clamp(0, labels.numel() - 1)], torch.full_like(idx, -1))
    live = (y >= 0) & (y < V)
    xd = torch.where(live[:, None], xd, torch.zeros_like(xd))
    at = torch.where(live, y, torch.zeros_like(y))[:, None]
    z = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    ez = (6 * D + 20) * U * size
    top = z.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    delta = 2 * ez.amax(1, keepdim=True) + 4 * U * (1 + top - z) + (V / 4 + 1100) * U
    loss = torch.where(live, (lse - z.gather(1, at)).squeeze(1), torch.zeros(B, dtype=torch.float64, device=x.device))
    loss_bound = 2 * ez.amax(1) + (V / 4 + 1100 + 4) * U + 4 * U * (top.abs().squeeze(1) + z.gather(1, at).abs().squeeze(1)
                                                                    + math.log(V + 1)) + 4 * U * loss.abs()
    count = int(live.sum())
    if g is None:
        g = torch.full((B,), 1.0 / max(count, 1), dtype=torch.float64, device=x.device)
    g = torch.where(live, g.double(), torch.zeros_like(g.double()))[:, None]
    p = torch.exp(z - lse) * g.abs()
    one = torch.zeros_like(z).scatter_(1, at, 1.0) * g
    dz = torch.exp(z - lse) * g - one
    plane = HALF_STEP[dtype] if dtype == torch.bfloat16 else U
    edz = p * torch.expm1(delta) + 4 * U * (p + one.abs()) + plane * dz.abs()
    adz = dz.abs() + edz
    dx, dw = dz @ wd, dz.t() @ xd
    edx = edz @ wd.abs() + (6 * V + 600) * U * (adz @ wd.abs())
    edw = edz.t() @ xd.abs() + (6 * B + 600) * U * (adz.t() @ xd.abs())
    half = HALF_STEP[dtype]
    return dict(loss=loss, loss_bound=loss_bound, count=count, dx=dx, dw=dw,
                dx_bound=edx + half * (dx.abs() + edx) + 1e-38, dw_bound=edw + half * (dw.abs() + edw) + 1e-38)


def close(got, want, bound, what):
    bad = (got.double() - want).abs() - bound
    assert bool((bad <= 0).all()), f"{what}: {float(bad.max())} beyond the bound {float(bound.max())}"


def check(x, w, labels, idx=None):
    ref = reference(x, w, labels, idx)
    xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = snn.class_cross_entropy(xs, ws, labels, idx=idx)
    assert loss.dtype == torch.float32 and loss.shape == ()
    loss.backward()
    count = max(ref["count"], 1)
    close(loss.detach(), ref["loss"].sum() / count, ref["loss_bound"].sum() / count + 1e-30, "mean loss")
    assert xs.grad.dtype == x.dtype and ws.grad.dtype == w.dtype
    close(xs.grad, ref["dx"], ref["dx_bound"], "dx")
    close(ws.grad, ref["dw"], ref["dw_bound"], "dweight")
    rows = snn.class_cross_entropy(x, w, labels, idx=idx, reduction="none")
    close(rows, ref["loss"], ref["loss_bound"], "row losses")
    return xs.grad, ws.grad, loss.detach()


SIZES = [(1, 1, 1), (1, 16, 65), (2, 8, 3), (3, 64, 128), (128, 64, 127), (129, 65, 129), (257, 100, 300), (512, 128, 1000),
         (40, 602, 777), (130, 768, 70), (300, 33, 5000), (1000, 256, 2000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,V", SIZES)
def test_loss_and_gradients(gpu_device, dtype, B, D, V):
    check(*make(B, D, V, DTYPES[dtype], gpu_device, seed=B + D + V))


@pytest.mark.parametrize("dtype", DTYPES)
def test_several_pieces(gpu_device, dtype):
    """More classes than one piece of the backward pass holds, the last piece ragged."""
    B, D, V = (12000, 264, 23001) if dtype == "bf16" else (12000, 40, 12001)
    check(*make(B, D, V, DTYPES[dtype], gpu_device, seed=1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [1, 2, 5, 8, 16, 17, 33])
@pytest.mark.parametrize("D,V", [(256, 3001), (101, 999)])
def test_few_rows(gpu_device, dtype, B, D, V):
    check(*make(B, D, V, DTYPES[dtype], gpu_device, seed=B))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [20, 100])
@pytest.mark.parametrize("D", [8, 32, 33, 64, 96, 160, 224, 256, 288, 320])
def test_nothing_beside_the_operands_is_read(gpu_device, dtype, B, D):
    """Operands in the middle of NaN, at every alignment of rows that takes a path of its own."""
    t = DTYPES[dtype]
    x, w, labels = make(B, D, 256, t, gpu_device, seed=D)
    around = []
    for m in (x, w):
        nan = torch.full((m.numel() + 2048,), float("nan"), device=gpu_device, dtype=t)
        nan[1024:1024 + m.numel()] = m.flatten()
        around.append(nan[1024:1024 + m.numel()].view(m.shape))
    check(around[0], around[1], labels)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_class(gpu_device, dtype):
    """Labels of -1, of V and far out, indices out of range, repeated indices; the padded rows hold NaN."""
    x, w, labels = make(200, 48, 150, DTYPES[dtype], gpu_device, seed=2, nodes=90)
    labels[:6] = torch.tensor([-1, 150, -100, 2 ** 40, -2 ** 40, 149], device=gpu_device)
    idx = torch.randint(0, 90, (200,), device=gpu_device, generator=torch.Generator(gpu_device).manual_seed(3))
    idx[:8] = torch.tensor([0, 1, 2, 3, 4, 5, -1, 90], device=gpu_device)
    idx[100:110] = 17
    dead = torch.cat([torch.arange(5), torch.tensor([6, 7])]).to(gpu_device)
    x[dead] = float("nan")
    x[dead[1]] = float("inf")
    dx, dw, loss = check(x, w, labels, idx)
    assert bool((dx[dead] == 0).all()) and bool(torch.isfinite(dw).all()) and bool(torch.isfinite(loss))


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_row_counts(gpu_device, dtype):
    x, w, labels = make(30, 20, 100, DTYPES[dtype], gpu_device)
    dx, dw, loss = check(x, w, torch.full_like(labels, -1))
    assert loss.item() == 0 and bool((dx == 0).all()) and bool((dw == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu_device, dtype):
    """Transposed, strided, offset and expanded operands: bit for bit the results of their copies."""
    t = DTYPES[dtype]
    x, w, labels = make(140, 70, 333, t, gpu_device, seed=4)
    base = check(x, w, labels)
    wide = torch.zeros(140, 75, device=gpu_device, dtype=t)
    wide[:, 3:73] = x
    tall = torch.zeros(335, 77, device=gpu_device, dtype=t)
    tall[1:334, 5:75] = w
    columns = torch.zeros(72, 340, device=gpu_device, dtype=t)
    columns[1:71, 3:336] = w.t()
    for xv in (x, wide[:, 3:73], x.t().contiguous().t()):
        for wv in (w, tall[1:334, 5:75], w.t().contiguous().t(), columns[1:71, 3:336].t()):
            for a, b in zip(check(xv, wv, labels), base):
                assert torch.equal(a, b)
    one = x[:1].expand(140, 70)
    for a, b in zip(check(one, w, labels), check(one.contiguous(), w, labels)):
        assert torch.equal(a, b)
    head = torch.nn.Parameter(w.t().contiguous())                 # the label head's own layout, D x V
    snn.class_cross_entropy(x, head.t(), labels).backward()
    assert head.grad.is_contiguous() and torch.equal(head.grad, base[1].t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_row_gradients_and_scaled_means(gpu_device, dtype):
    t = DTYPES[dtype]
    x, w, labels = make(150, 64, 400, t, gpu_device, seed=5)
    labels[7] = -1
    g = torch.randn(150, device=gpu_device)
    g[3] = 0.0
    ref = reference(x, w, labels, g=g)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    (snn.class_cross_entropy(xs, ws, labels, reduction="none") * g).sum().backward()
    close(xs.grad, ref["dx"], ref["dx_bound"], "dx")
    close(ws.grad, ref["dw"], ref["dw_bound"], "dweight")
    ref = reference(x, w, labels, g=torch.full((150,), -3.0 / 149, device=gpu_device, dtype=torch.float64))
    xs.grad = ws.grad = None
    (snn.class_cross_entropy(xs, ws, labels) * -3.0).backward()
    close(xs.grad, ref["dx"], ref["dx_bound"], "dx")
    close(ws.grad, ref["dw"], ref["dw_bound"], "dweight")
    # an expanded gradient, and one operand frozen
    xs.grad = None
    snn.class_cross_entropy(xs, w, labels, reduction="none").sum().backward()
    ref = reference(x, w, labels, g=torch.ones(150, device=gpu_device))
    close(xs.grad, ref["dx"], ref["dx_bound"], "dx")
    ws.grad = None
    snn.class_cross_entropy(x, ws, labels).backward()
    close(ws.grad, reference(x, w, labels)["dw"], reference(x, w, labels)["dw_bound"], "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
def test_peaked_and_far_logits(gpu_device, dtype):
    """A model that is sure, right or wrong; logits of some hundreds; equal logits; classes masked by
    the type's lowest value; scales down to the subnormals."""
    t = DTYPES[dtype]
    x, w, labels = make(100, 32, 300, t, gpu_device, seed=6)
    check(x * 20, w * 8, labels)
    check(x, torch.zeros_like(w), labels)
    check(torch.zeros_like(x), w, labels)
    check(x * 2.0 ** -70, w * 2.0 ** 60, labels)
    sure = w[labels] * 30
    check(sure, w, labels)
    check(-sure, w, labels)
    masked_x, masked_w = x.clone(), w.clone()
    masked_x[:, 0] = 1.0
    masked_w[:, 0] = 0.0
    masked_w[200:, 0] = torch.finfo(t).min
    keep = labels % 200
    rows = snn.class_cross_entropy(masked_x, masked_w, keep, reduction="none")
    want = reference(masked_x, masked_w[:200], keep)
    close(rows, want["loss"], want["loss_bound"], "masked classes")


def test_operands_of_wide_range(gpu_device):
    """A row, a class or a feature far larger than the rest: exact to 32 bits in the small rows, too."""
    x, w, labels = make(150, 40, 260, torch.float32, gpu_device, seed=13)
    for scale in (2.0 ** 20, 2.0 ** 40, 2.0 ** -30):
        far = x.clone()
        far[3] *= scale
        check_range(far, w, labels)
        far = w.clone()
        far[7] *= scale
        check_range(x * 0.01, far, labels)
    far, other = x.clone(), w.clone()
    far[:, 5] *= 2.0 ** 30
    other[:, 5] *= 2.0 ** -30
    check_range(far, other, labels)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [9, 120])
def test_logits_beyond_all_reason(gpu_device, dtype, B):
    """Logits of thousands to 10^15 in some rows: p of those is 1 for the largest logit and 0 for the
    others, exactly; the rows beside them come out as ever."""
    t = DTYPES[dtype]
    x, w, labels = make(B, 24, 200, t, gpu_device, seed=14)
    for power in (14, 24, 50):
        far = x.clone()
        far[2], far[5] = far[2] * 2.0 ** power, far[5] * 2.0 ** power
        z = far.double() @ w.double().t()
        ref = reference(x, w, labels)
        rows = snn.class_cross_entropy(far, w, labels, reduction="none").double()
        for r in (2, 5):
            want = z[r].max() - z[r, labels[r]]
            assert abs(rows[r] - want) <= 1e-5 * z[r].abs().max() + 1e-5
        beside = [r for r in range(B) if r not in (2, 5)]
        close(rows[beside], ref["loss"][beside], ref["loss_bound"][beside], "rows beside")
        xs = far.clone().requires_grad_()
        g = torch.full((B,), 1.0 / B, device=gpu_device)
        (snn.class_cross_entropy(xs, w, labels, reduction="none") * g).sum().backward()
        close(xs.grad[beside], ref["dx"][beside], ref["dx_bound"][beside], "dx beside")
        for r in (2, 5):
            gap = z[r].sort().values
            if gap[-1] - gap[-2] > 40:                       # clear of the rounding: p is 0 or 1
                want = (w[z[r].argmax()].double() - w[labels[r]].double()) / B
                assert bool(((xs.grad[r].double() - want).abs() <= 2.0 ** -7 * w.double().abs().amax() / B).all())


def check_range(x, w, labels):
    ref = reference(x, w, labels)
    rows = snn.class_cross_entropy(x, w, labels, reduction="none")
    finite = torch.isfinite(ref["loss_bound"])
    close(rows[finite], ref["loss"][finite], ref["loss_bound"][finite], "row losses")
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    snn.class_cross_entropy(xs, ws, labels).backward()
    assert bool(torch.isfinite(xs.grad).all()) and bool(torch.isfinite(ws.grad).all())
    keep = torch.isfinite(ref["dx_bound"]) & torch.isfinite(ref["dx"])
    close(xs.grad[keep], ref["dx"][keep], ref["dx_bound"][keep], "dx")


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers(gpu_device, dtype):
    """A NaN in a counted row, or in a class, is seen: in that row's loss and the mean, not in other rows."""
    t = DTYPES[dtype]
    x, w, labels = make(60, 40, 200, t, gpu_device, seed=7)
    x[11, 3] = float("nan")
    rows = snn.class_cross_entropy(x, w, labels, reduction="none")
    assert bool(torch.isnan(rows[11])) and int(torch.isnan(rows).sum()) == 1
    assert bool(torch.isnan(snn.class_cross_entropy(x, w, labels)))
    x, w, labels = make(60, 40, 200, t, gpu_device, seed=7)
    w[17, 5] = float("nan")
    assert bool(torch.isnan(snn.class_cross_entropy(x, w, labels, reduction="none")).all())


def test_gradient_against_differences(gpu_device):
    x, w, labels = make(20, 12, 90, torch.float32, gpu_device, seed=8)
    labels[4] = -1
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    snn.class_cross_entropy(xs, ws, labels).backward()

    def f(a, b):
        return torch.nn.functional.cross_entropy(a @ b.t(), labels, ignore_index=-1).item()
    xd, wd, h = x.double(), w.double(), 1e-5
    for at in ((0, 0), (4, 3), (19, 11)):
        e = torch.zeros_like(xd)
        e[at] = h
        assert abs(xs.grad[at].item() - (f(xd + e, wd) - f(xd - e, wd)) / (2 * h)) <= 1e-6
    for at in ((0, 0), (int(labels[0]), 5), (89, 11)):
        e = torch.zeros_like(wd)
        e[at] = h
        assert abs(ws.grad[at].item() - (f(xd, wd + e) - f(xd, wd - e)) / (2 * h)) <= 1e-6


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_bit_for_bit(gpu_device, dtype):
    x, w, labels = make(700, 96, 5000, DTYPES[dtype], gpu_device, seed=9)
    first = None
    for _ in range(3):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = snn.class_cross_entropy(xs, ws, labels)
        loss.backward()
        got = (loss.detach(), xs.grad, ws.grad)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", [(300, 900), (4, 2000)])
def test_captured_step(gpu_device, dtype, B, V):
    """Forward and backward recorded into a graph, replayed on new data with eager work between."""
    t = DTYPES[dtype]
    x, w, labels = make(B, 64, V, t, gpu_device, seed=10)

    def step():
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = snn.class_cross_entropy(xs, ws, labels)
        return (loss.detach(), *torch.autograd.grad(loss, (xs, ws)))
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(gpu_device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(torch.randn(B, 64, device=gpu_device))
        labels.copy_(torch.randint(-1, V, (B,), device=gpu_device))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_graphs_and_two_streams(gpu_device):
    """Two captured steps replayed in turn and eager calls on two streams at once do not share scratch."""
    sets = [make(200, 48, 700, torch.float32, gpu_device, seed=s) for s in (11, 12)]

    def step(x, w, labels):
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = snn.class_cross_entropy(xs, ws, labels)
        return (loss.detach(), *torch.autograd.grad(loss, (xs, ws)))
    want = [step(*s) for s in sets]
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    streams = [torch.cuda.Stream(gpu_device) for _ in sets]
    got = [None, None]
    for k, st in enumerate(streams):
        st.wait_stream(torch.cuda.current_stream(gpu_device))
        with torch.cuda.stream(st):
            for _ in range(5):
                got[k] = step(*sets[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_memory_does_not_grow_with_rows_times_classes(gpu_device):
    B, D, V = 8192, 64, 60000
    x, w, labels = make(B, D, V, torch.bfloat16, gpu_device)
    x.requires_grad_()
    w.requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(gpu_device)
    before = torch.cuda.memory_allocated(gpu_device)
    snn.class_cross_entropy(x, w, labels).backward()
    assert torch.cuda.max_memory_allocated(gpu_device) - before < B * V * 2 / 3


def test_no_rows(gpu_device):
    x = torch.empty(0, 8, device=gpu_device, requires_grad=True)
    w = torch.randn(70, 8, device=gpu_device, requires_grad=True)
    labels = torch.empty(0, dtype=torch.int64, device=gpu_device)
    loss = snn.class_cross_entropy(x, w, labels)
    loss.backward()
    assert loss.item() == 0 and bool((w.grad == 0).all()) and x.grad.shape == (0, 8)
    assert snn.class_cross_entropy(x, w, labels, reduction="none").shape == (0,)


def test_refusals(gpu_device):
    x, w, labels = make(10, 8, 70, torch.float32, gpu_device)
    call = snn.class_cross_entropy
    for args, error in (((x, w.bfloat16(), labels), TypeError), ((x.half(), w.half(), labels), TypeError),
                        ((x, w, labels.int()), TypeError), ((x, w, labels[:5]), ValueError),
                        ((x, w[:, :7], labels), ValueError), ((x[0], w, labels), ValueError),
                        ((x, w[:0], labels), ValueError), ((x, w, labels.cpu()), ValueError),
                        ((x.cpu(), w.cpu(), labels.cpu()), ValueError), ((x, w, labels[None]), TypeError)):
        with pytest.raises(error):
            call(*args)
    with pytest.raises(ValueError):
        call(x, w, labels, reduction="sum")
    with pytest.raises(ValueError):
        call(x, w, labels, idx=torch.zeros(9, dtype=torch.int64, device=gpu_device))
    with pytest.raises(TypeError):
        call(x, w, labels, idx=torch.zeros(10, device=gpu_device))
    with pytest.raises(ValueError):
        call(x, w, labels[:0], idx=torch.zeros(10, dtype=torch.int64, device=gpu_device))


def test_head_over_a_checkpointed_stack(gpu_device):
    """The operators together as a training step uses them: two graph convolutions that keep their
    inputs in 8 bits under a wide label head, against the same step with everything kept."""
    n, V = 800, 500
    g = torch.Generator().manual_seed(0)
    edges = torch.randint(0, n, (2, 3000), generator=g).to(gpu_device)
    x = torch.randn(n, 96, generator=g).to(gpu_device)
    labels = torch.randint(0, V, (n,), generator=g).to(gpu_device)
    idx = torch.randperm(n, generator=g)[:400].to(gpu_device)
    results = []
    for keep in (None, "int8"):
        torch.manual_seed(1)
        first = snn.GCNConv(96, 64, checkpoint=keep).to(gpu_device)
        second = snn.GCNConv(64, 48, checkpoint=keep, input_slope=0.0).to(gpu_device)
        head = torch.nn.Parameter(torch.randn(V, 48, generator=torch.Generator().manual_seed(2)).to(gpu_device) / 7)
        h = second(first(x, edges), edges)[idx]
        if keep:
            loss = snn.class_cross_entropy(h, head, labels, idx=idx)
        else:
            loss = torch.nn.functional.cross_entropy(h @ head.t(), labels[idx])
        loss.backward()
        results.append((loss.detach(), head.grad, second.lin.weight.grad, first.lin.weight.grad, first.bias.grad))
    full, kept = results
    # the loss and what lies above the codes: 32-bit arithmetic in another order; the weights'
    # gradients: half a step in 127 of a group's peak, averaged over the rows
    for a, b in zip(full[:2] + full[4:], kept[:2] + kept[4:]):
        assert (a - b).norm() <= 1e-4 * a.norm()
    for a, b in zip(full[2:4], kept[2:4]):
        assert (a - b).norm() <= 0.03 * a.norm()


@pytest.mark.parametrize("indexed", [False, True])
@pytest.mark.parametrize("B,D,V", [(64, 128, 4096), (300, 33, 5001)])
def test_label_head_of_a_stacked_layer(gpu_device, B, D, V, indexed):
    """The label head of the stacked training with thousands of classes runs through the same loss."""
    from sgnn_amd.stacked import _head_cross_entropy
    x, w, labels = make(B, D, V, torch.float32, gpu_device, seed=B, nodes=3 * B if indexed else B)
    idx = torch.randperm(3 * B, generator=torch.Generator().manual_seed(3)).to(gpu_device)[:B] if indexed else None
    ref = reference(x, w, labels, idx)
    E, Wt = x.requires_grad_(), w.t().contiguous().requires_grad_()
    loss = _head_cross_entropy(E, Wt, labels, idx, unit=True)
    assert "ClassXent" in loss.grad_fn.name()
    loss.backward()
    assert Wt.grad.is_contiguous()
    close(loss.detach(), ref["loss"].mean(), ref["loss_bound"].mean() + 1e-30, "mean loss")
    close(E.grad, ref["dx"], ref["dx_bound"], "dE")
    close(Wt.grad, ref["dw"].t(), ref["dw_bound"].t(), "dWt")


def test_stacked_layer_with_thousands_of_classes(gpu_device):
    """Its captured training steps give what the same steps give one by one, bit for bit."""
    from sgnn_amd.norm_adj import NormAdj
    from sgnn_amd.stacked import EmbeddingLayer, LayerParam, get_activation
    n, F, V = 500, 40, 4500
    g = torch.Generator().manual_seed(0)
    edges = torch.randint(0, n, (2, 3000), generator=g).numpy()
    adj = NormAdj.from_coo(edges[0], edges[1], None, n, gpu_device)
    X = torch.randn(n, F, generator=g).to(gpu_device)
    labels = torch.randint(0, V, (n,), generator=g).to(gpu_device)
    results = []
    for graph in (True, False):
        torch.manual_seed(5)
        p = LayerParam(16, inner_act=get_activation("leaky_relu=0.2"), act=get_activation("linear"), max_iter=12,
                       batch_size=64, learning_rate=0.01, lam=1e-4)
        layer = EmbeddingLayer(adj, labels, torch.ones(n, dtype=torch.bool, device=gpu_device), F, 16, V, p, gpu_device)
        before = layer.Wt.detach().clone()
        layer.use_graph = graph
        layer.run(X)
        assert layer.use_graph is graph                              # the capture did not fall back
        assert not torch.equal(before, layer.Wt)
        results.append((layer.W.detach().clone(), layer.Wt.detach().clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,V", [(5, 40, 3000), (30, 300, 700), (200, 100, 900), (300, 300, 5000)])
def test_one_gradient_alone(gpu_device, dtype, B, D, V):
    """Either operand's gradient by itself is the one that comes with the other's, bit for bit."""
    x, w, labels = make(B, D, V, DTYPES[dtype], gpu_device, seed=B)
    both = x.clone().requires_grad_(), w.clone().requires_grad_()
    snn.class_cross_entropy(*both, labels).backward()
    only_x, only_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    snn.class_cross_entropy(only_x, w, labels).backward()
    snn.class_cross_entropy(x, only_w, labels).backward()
    assert torch.equal(only_x.grad, both[0].grad) and torch.equal(only_w.grad, both[1].grad)
    turned = w.t().contiguous().requires_grad_()         # stored by feature: the same values, the gradient likewise
    snn.class_cross_entropy(x, turned.t(), labels).backward()
    assert turned.grad.is_contiguous()
    close(turned.grad.t(), both[1].grad.double(), reference(x, w, labels)["dw_bound"] * 2, "dweight by feature")
