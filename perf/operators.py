"""Workloads of the wide-head loss and of the 8-bit saved activations.

Two operators of full-graph and mini-batch training whose cost is memory:

* ``xent``: softmax cross-entropy of ``x @ weight.T`` over many classes, computed in pieces of
  the classes so that the logits are never kept: the mean with the gradients of ``x`` and
  ``weight`` (``train``), or row by row for evaluation and serving (``rows``);
* ``save`` / ``wgrad`` / ``layer``: a layer's input kept in 8 bits for its backward pass: written
  and read back, the weight gradient formed from the codes, and a whole linear layer that keeps
  nothing else of its input.

A saved activation ``a = x if x > 0 else slope * x`` is held in groups of 32 consecutive
features of a row that share a power-of-two step ``2^s``:

* ``slope == 1`` (no activation): the code is ``rint(a / 2^s)`` and stands for ``code * 2^s``,
  ``s`` the smallest exponent whose codes stay within +-127;
* any other slope: the code is ``ceil(a / 2^s) - 1`` and stands for ``(code + 1/2) * 2^s``, ``s``
  the smallest exponent with ``|a| <= 128 * 2^s`` in the group, so a code is negative exactly
  where ``x > 0`` is false; with ``slope == 0`` negative codes stand for 0.

``own`` chooses between plain torch operations in 32 bits and the package's operators.
"""
import math

import torch

own = False

GROUP = 32
MIN_STEP = -125
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # an optimiser iteration of a decoupled layer: batch of 512 nodes, an embedding of 128, a
        # label set beyond the 64 classes of the small head; latency counts
        dict(name="xent_batch_f32", op="xent", mode="train", dtype="f32", B=512, D=128, V=1000, none=0.0),
        # a wide feature row straight into the head (602 features), odd class count, all in fp32
        dict(name="xent_wide_f32", op="xent", mode="train", dtype="f32", B=2048, D=602, V=10007, none=0.0),
        # large-batch training on many classes in bf16
        dict(name="xent_train_bf16", op="xent", mode="train", dtype="bf16", B=4096, D=256, V=50000, none=0.0),
        # ragged sizes; a tenth of the rows carry no label (a padded or partly labelled batch)
        dict(name="xent_ragged_bf16", op="xent", mode="train", dtype="bf16", B=1777, D=100, V=30011, none=0.1),
        # evaluation: the loss of each of many nodes, every node of a graph of 169343 being a class
        dict(name="xent_eval_bf16", op="xent", mode="rows", dtype="bf16", B=16384, D=128, V=169343, none=0.0),
        # serving: the log-probability of one node's label; the weight is read once
        dict(name="xent_row_f32", op="xent", mode="rows", dtype="f32", B=1, D=256, V=100003, none=0.0),
        # a hidden layer of the Reddit-sized graph, after a ReLU
        dict(name="save_relu_f32", op="save", dtype="f32", n=232965, F=256, slope=0.0),
        # a mid-sized citation graph's features in bf16, width not a multiple of the group
        dict(name="save_plain_bf16", op="save", dtype="bf16", n=19717, F=500, slope=1.0),
        # weight gradient of the first layer on the Reddit-sized graph (602 features, 128 units)
        dict(name="wgrad_reddit_f32", op="wgrad", dtype="f32", n=232965, F=602, H=128, slope=1.0),
        # weight gradient of a hidden layer in bf16, after a ReLU
        dict(name="wgrad_hidden_bf16", op="wgrad", dtype="bf16", n=169343, F=256, H=256, slope=0.0),
        # a citation graph's first layer, forward and backward: many features, few nodes and units
        dict(name="layer_cites_f32", op="layer", dtype="f32", n=2708, F=1433, H=16, slope=1.0),
        # a hidden layer of the Reddit-sized graph behind a leaky ReLU, forward and backward
        dict(name="layer_hidden_f32", op="layer", dtype="f32", n=232965, F=256, H=64, slope=0.2),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ranges; sizes are spread over their logarithm."""
    op = rng.choice(["xent", "xent", "xent", "save", "wgrad", "layer"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "xent":
        mode = rng.choice(["train", "train", "rows"])
        budget = 2e10 if dtype == "f32" else 5e10            # multiply-adds of one product
        while True:
            case = dict(op=op, mode=mode, dtype=dtype, B=_log_int(rng, 1, 16384), D=_log_int(rng, 16, 768),
                        V=_log_int(rng, 65, 170000), none=rng.choice([0.0, 0.0, 0.1]))
            if case["B"] * case["D"] * case["V"] <= budget and case["B"] * case["V"] <= 1e9:
                return case
    slope = rng.choice([0.0, 1.0, 0.2])
    while True:
        case = dict(op=op, dtype=dtype, n=_log_int(rng, 64, 232965), F=_log_int(rng, 8, 1433), slope=slope)
        if op != "save":
            case["H"] = _log_int(rng, 4, 256)
        cells = case["n"] * case["F"]
        if cells <= 6e7 and cells * case.get("H", 1) <= 5e9:
            return case


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "xent":
        B, D, V = case["B"], case["D"], case["V"]
        ids = 8 * B * (2 if case["mode"] == "train" else 1)
        operands = size * (B * D + V * D)
        if case["mode"] == "train":                          # logits and two gradient products
            return {"bytes": 2 * operands + ids + 4, "flops": 6 * B * D * V}
        return {"bytes": operands + ids + 4 * B, "flops": 2 * B * D * V}
    n, F = case["n"], case["F"]
    cells, groups = n * F, n * -(-F // GROUP)
    if case["op"] == "save":                                 # write the codes, then read them back
        return {"bytes": 2 * (size * cells + cells + groups), "flops": 4 * cells}
    H = case["H"]
    if case["op"] == "wgrad":
        return {"bytes": cells + groups + size * (n * H + F * H), "flops": 2 * cells * H}
    # x and weight in, codes out and in again, y out, its gradient in, both gradients out
    return {"bytes": size * (2 * cells + 2 * F * H + 2 * n * H) + 2 * (cells + groups), "flops": 6 * cells * H}


# ------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "xent":
        B, D, V = case["B"], case["D"], case["V"]
        w = randn(V, D) * (1.5 / math.sqrt(D))
        nodes = 2 * B + 7
        labels = torch.randint(0, V, (nodes,), generator=g, device="cuda")
        if case["none"]:
            labels[torch.rand(nodes, generator=g, device="cuda") < case["none"]] = -1
        idx = torch.randperm(nodes, generator=g, device="cuda")[:B].contiguous()
        if case["mode"] != "train":                          # evaluation reads its rows in order
            labels, idx = labels[idx].contiguous(), None
        y = labels if idx is None else labels[idx]
        x = randn(B, D) + 0.7 * w[y.clamp_min(0)]            # a model that has learned something
        return dict(x=x.to(dtype), weight=w.to(dtype), labels=labels, idx=idx)
    n, F = case["n"], case["F"]
    x = randn(n, F) * torch.exp(0.7 * randn(n, 1))           # rows of unlike magnitude
    if case["slope"] == 1.0:
        x = x * (torch.rand(n, F, generator=g, device="cuda") < 0.6)     # input features hold zeros
    out = dict(x=x.to(dtype))
    if case["op"] != "save":
        out["grad"] = (randn(n, case["H"]) * (1.0 / n)).to(dtype)
    if case["op"] == "layer":
        out["weight"] = (randn(case["H"], F) * (1.0 / math.sqrt(F))).to(dtype)
    return out


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        if case["op"] == "wgrad":
            from sgnn_amd import nn
            state["saved"] = nn.save_int8(state.pop("x"), slope=case["slope"])
        elif case["op"] == "layer" or (case["op"] == "xent" and case["mode"] == "train"):
            for k in ("x", "weight"):
                state[k].requires_grad_()
    elif case["op"] == "wgrad":
        state["codes"], state["steps"] = _encode(_act(state.pop("x").float(), case["slope"]), case["slope"])
    return state


# -------------------------------------------------------------------------------- plain form
def _act(x, slope):
    return torch.where(x > 0, x, slope * x)


def _grouped(a):
    n, F = a.shape
    groups = -(-F // GROUP)
    if groups * GROUP != F:
        a = torch.cat([a, a.new_zeros(n, groups * GROUP - F)], 1)
    return a.view(n, groups, GROUP)


def _power(s):
    """2^s in 32 bits for whole s in [-126, 127], exactly (a library power may be a rounding off)."""
    return ((s.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(a, slope):
    """int8 codes [n, F] and int32 step exponents [n, groups]."""
    n, F = a.shape
    b = _grouped(a)
    m = b.abs().amax(2)
    fraction, exponent = torch.frexp(m)                      # m = fraction * 2^exponent, fraction in [1/2, 1)
    if slope == 1.0:
        # 127.5 / 128 of the next power of two would round to 128: one exponent more
        s = exponent - 7 + (fraction >= 127.5 / 128).int()
    else:
        s = exponent - 7 - (fraction == 0.5).int()           # a power of two fits its own exponent
    s = torch.where(m > 0, s, torch.full_like(s, MIN_STEP)).clamp_min(MIN_STEP)
    scaled = b * _power(-s).unsqueeze(2)
    if slope == 1.0:
        q = torch.round(scaled)
    else:
        q = torch.ceil(scaled) - 1
        q = torch.where(b > 0, q.clamp(0, 127), q.clamp(-128, -1))
    return q.to(torch.int8).view(n, -1)[:, :F].contiguous(), s


def _decode(codes, steps, slope):
    n, F = codes.shape
    q = _grouped(codes.float())
    if slope != 1.0:
        q = q + 0.5
        if slope == 0.0:
            q = q.clamp_min(0.0)
    return (q * _power(steps).unsqueeze(2)).view(n, -1)[:, :F]


def _plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "xent":
        x, w, idx = state["x"].float(), state["weight"].float(), state["idx"]
        y = state["labels"] if idx is None else state["labels"][idx]
        B, V = x.shape[0], w.shape[0]
        counted = (y >= 0) & (y < V)
        row = torch.arange(B, device=x.device)
        at = torch.where(counted, y, torch.zeros_like(y))
        z = x @ w.t()
        top = z.amax(1, keepdim=True)
        picked = z[row, at]
        p = torch.exp(z - top)
        total = p.sum(1, keepdim=True)
        loss = (top + torch.log(total)).squeeze(1) - picked
        loss = torch.where(counted, loss, torch.zeros_like(loss))
        if case["mode"] == "rows":
            return loss
        live = counted.sum().clamp_min(1)
        share = counted.float().unsqueeze(1) / live
        p *= share / total
        p[row, at] -= share.squeeze(1)
        return loss.sum() / live, (p @ w).to(dtype), (p.t() @ x).to(dtype)
    slope = case["slope"]
    if case["op"] == "wgrad":
        return (state["grad"].float().t() @ _decode(state["codes"], state["steps"], slope)).to(dtype)
    x = state["x"].float()
    a = _act(x, slope)
    codes, steps = _encode(a, slope)
    if case["op"] == "save":
        return _decode(codes, steps, slope).to(dtype)
    w, grad = state["weight"].float(), state["grad"].float()
    dx = grad @ w
    if slope != 1.0:
        dx = torch.where(codes >= 0, dx, slope * dx)
    return (a @ w.t()).to(dtype), dx.to(dtype), (grad.t() @ _decode(codes, steps, slope)).to(dtype)


# ----------------------------------------------------------------------------- the operators
def _own(state):
    from sgnn_amd import nn
    case = state["case"]
    if case["op"] == "xent":
        x, w = state["x"], state["weight"]
        loss = nn.class_cross_entropy(x, w, state["labels"], idx=state["idx"],
                                      reduction="none" if case["mode"] == "rows" else "mean")
        if case["mode"] == "rows":
            return loss
        dx, dw = torch.autograd.grad(loss, (x, w))
        return loss.detach(), dx, dw
    if case["op"] == "wgrad":
        return state["saved"].weight_grad(state["grad"])
    if case["op"] == "save":
        return nn.save_int8(state["x"], slope=case["slope"]).restore()
    y = nn.linear_saved_int8(state["x"], state["weight"], slope=case["slope"])
    dx, dw = torch.autograd.grad(y, (state["x"], state["weight"]), state["grad"])
    return y.detach(), dx, dw


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- the definition, 64 bits
def _exact_power(s):
    return torch.bitwise_left_shift(s.long() + 1023, 52).view(torch.float64)


def _exact_codes(a, slope):
    """Codes and steps from the definition: the smallest step whose codes hold the group."""
    n, F = a.shape
    groups = (F + GROUP - 1) // GROUP
    wide = torch.zeros(n, groups * GROUP, dtype=torch.float64, device=a.device)
    wide[:, :F] = a
    wide = wide.reshape(n, groups, GROUP)
    peak = wide.abs().max(dim=2, keepdim=True).values
    s = torch.full_like(peak, float(MIN_STEP))
    guess = torch.floor(torch.log2(peak.clamp_min(2.0 ** -140))) - 9      # at least one below the answer
    for k in range(5, -1, -1):                               # the last write is the smallest that holds
        step = _exact_power(guess + k)
        holds = torch.round(peak / step) <= 127 if slope == 1.0 else peak <= 128 * step
        s = torch.where(holds & (guess + k >= MIN_STEP), guess + k, s)
    step = _exact_power(s)
    if slope == 1.0:
        q = torch.round(wide / step)
        value = q * step
    else:
        q = torch.ceil(wide / step) - 1
        q = torch.where(wide > 0, q.clamp(min=0, max=127), q.clamp(min=-128, max=-1))
        value = (q + 0.5) * step
        if slope == 0.0:
            value = torch.where(q < 0, torch.zeros_like(value), value)
    return value.reshape(n, -1)[:, :F]


def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["op"] == "xent":
        x, w = inputs["x"].double(), inputs["weight"].double()
        y = inputs["labels"] if inputs["idx"] is None else inputs["labels"].index_select(0, inputs["idx"])
        B, V = x.shape[0], w.shape[0]
        known = y.ge(0).logical_and(y.lt(V))
        count = max(int(known.sum()), 1)
        losses, dx = [], []
        dw = torch.zeros_like(w)
        piece = max(1, min(B, int(2e8 // V)))
        for lo in range(0, B, piece):
            hi = min(B, lo + piece)
            z = x[lo:hi].matmul(w.T)
            logp = torch.log_softmax(z, dim=1)
            k = known[lo:hi]
            pick = y[lo:hi].clamp(0, V - 1).unsqueeze(1)
            losses.append(-logp.gather(1, pick).squeeze(1) * k)
            if case["mode"] == "train":
                dz = logp.exp_()
                dz.scatter_add_(1, pick, torch.full_like(pick, -1.0, dtype=torch.float64))
                dz *= (k.double() / count).unsqueeze(1)
                dx.append(dz.matmul(w))
                dw += dz.T.matmul(x[lo:hi])
        losses = torch.cat(losses)
        if case["mode"] == "rows":
            return losses
        return losses.sum() / count, torch.cat(dx), dw
    slope = case["slope"]
    x = inputs["x"]
    # the activation is taken in 32 bits by definition: the codes are those of the rounded value
    a = torch.where(x.float() > 0, x.float(), x.float() * slope).double()
    value = _exact_codes(a, slope)
    if case["op"] == "save":
        return value
    grad = inputs["grad"].double()
    dw = grad.T.matmul(value)
    if case["op"] == "wgrad":
        return dw
    w = inputs["weight"].double()
    dx = grad.matmul(w)
    if slope != 1.0:
        dx = dx * torch.where(x.double() > 0, 1.0, slope)
    return a.matmul(w.T), dx, dw
