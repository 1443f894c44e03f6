"""The operators of layers whose weights and activations are 8-bit integers: what is measured of them.

A row of numbers is held as int8 values q and one fp32 scale s: s = amax / 127, q = 127 x / amax rounded to the nearest whole number, ties to even.  Weights
[features, inputs] have a scale per feature, activations [tokens, inputs] one per token, and a product of the two is whole numbers until both scales meet it.
Three operators, each in a plain form of elementary torch operations and as the framework's call:

* ``rows``     the rows of a matrix as int8 values and scales: a checkpoint's weights once, activations in every layer;
* ``linear``   a layer: its activations' rows in 8 bits, the product with the weights, both scales; with a residual, or as silu(gate) · up of neighbouring features;
* ``experts``  the layers of a mixture of experts: the tokens of every expert, ordered by expert, against that expert's weights.

``run`` takes the plain form unless ``own`` is set.
"""
import math

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # activations of one decoding token, and of a large batch of prompts; a float32 matrix of an odd width
        dict(name="rows 1 x 4096", op="rows", rows=1, k=4096, dtype="bfloat16"),
        dict(name="rows 8192 x 14336", op="rows", rows=8192, k=14336, dtype="bfloat16"),
        dict(name="rows 4097 x 1001 fp32", op="rows", rows=4097, k=1001, dtype="float32"),
        # the attention output of one token of a model of 4096 columns: the smallest layer call
        dict(name="linear 1 x 4096 x 4096", op="linear", rows=1, n=4096, k=4096, form="plain", dtype="bfloat16"),
        # the way back from the hidden columns for six requests that decode together
        dict(name="linear 6 x 4096 x 14336", op="linear", rows=6, n=4096, k=14336, form="residual", dtype="bfloat16"),
        # gate and up of a batch of 48 requests
        dict(name="linear 48 x 28672 x 4096", op="linear", rows=48, n=28672, k=4096, form="gated", dtype="bfloat16"),
        # queries, keys and values of a short prompt of odd length
        dict(name="linear 333 x 6144 x 4096", op="linear", rows=333, n=6144, k=4096, form="plain", dtype="bfloat16"),
        # gate and up of a batch of long prompts: the largest
        dict(name="linear 8192 x 28672 x 4096", op="linear", rows=8192, n=28672, k=4096, form="gated", dtype="bfloat16"),
        # one token that chose four of 32 experts
        dict(name="experts 1 x 4 of 32", op="experts", tokens=1, top=4, experts=32, n=2048, k=2048, form="gated", dtype="bfloat16"),
        # a decoding batch, on the way back from the hidden columns
        dict(name="experts 64 x 4 of 32, back", op="experts", tokens=64, top=4, experts=32, n=2048, k=1024, form="plain", dtype="bfloat16"),
        # a prompt over experts of an odd size, some chosen often and some hardly
        dict(name="experts 1000 x 3 of 24", op="experts", tokens=1000, top=3, experts=24, n=2736, k=1112, form="gated", dtype="bfloat16"),
        # a large batch of prompts
        dict(name="experts 8192 x 4 of 32", op="experts", tokens=8192, top=4, experts=32, n=2048, k=2048, form="gated", dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "linear", "linear", "linear", "experts", "experts"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float16", "float32"])
    if op == "rows":
        k = _log(rng, 16, 28672)
        return dict(op="rows", rows=_log(rng, 1, min(65536, 8192 * 14336 // k)), k=k, dtype=dtype)
    form = rng.choice(["plain", "plain", "residual", "gated"])
    k = _log(rng, 64, 14336)
    step = rng.choice([1, 8, 64])                                             # any number of inputs, and those of ordinary layers
    k = max(1, k // step) * step
    if op == "linear":
        n = max(2, _log(rng, 64, 28672) // 2 * 2) if form == "gated" else _log(rng, 64, 28672)
        return dict(op="linear", rows=_log(rng, 1, min(8192, 8192 * 28672 * 4096 // (n * k))), n=n, k=k, form=form, dtype=dtype)
    form = "gated" if form == "gated" else "plain"
    experts = _log(rng, 2, 128)
    top = rng.randrange(1, min(8, experts) + 1)
    k = min(k, 4096)
    n = max(16, _log(rng, 64, 4096) // 2 * 2)
    return dict(op="experts", tokens=_log(rng, 1, max(1, min(8192, 8192 * 4 * 2048 * 2048 // (top * n * k)))), top=top, experts=experts, n=n, k=k, form=form, dtype=dtype)


# --------------------------------------------------------------------------- inputs
def _in_8_bits(x):
    """(q, s) of the rows of x: the quotient in 64 bits, since a value next to the middle of two whole numbers goes one way or the other."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    q = (x * 127.0 / torch.where(amax == 0, torch.ones_like(amax), amax)).round()
    return q, (amax.float() / 127.0).squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, case["dtype"])

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    def activations(m, k):
        # a few channels are much larger than the rest, as behind a norm with learned gains
        return (randn(m, k) * torch.exp(0.7 * randn(k))).to(dt)

    def weights(n, k):
        q, s = _in_8_bits(randn(n, k, dtype=torch.bfloat16) * (k ** -0.5))
        return q.to(torch.int8), s

    if case["op"] == "rows":
        return dict(case, x=activations(case["rows"], case["k"]))
    n, k = case["n"], case["k"]
    if case["op"] == "linear":
        s = dict(case, x=activations(case["rows"], k))
        s["values"], s["scales"] = weights(n, k)
        s["residual"] = randn(case["rows"], n).to(dt) if case["form"] == "residual" else None
        return s
    T, E, top = case["tokens"], case["experts"], case["top"]
    s = dict(case, x=activations(T, k))
    v, sc = weights(E * n, k)
    s["values"], s["scales"] = v.view(E, n, k), sc.view(E, n)
    # every token chooses `top` experts, some of which are liked more than others; its rows, ordered by expert
    choice = (randn(T, E) + randn(E)).topk(top, -1).indices.reshape(-1)
    order = torch.sort(choice, stable=True)
    s["source"] = (order.indices // top).to(torch.int32)
    count = torch.bincount(choice, minlength=E)
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), count.cumsum(0)]).to(torch.int32)
    s["expert"] = order.values                                                # of every row
    s["most"] = int(count.max())
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"rows": _plain_rows, "linear": _plain_linear, "experts": _plain_experts}[state["op"]](state)


def _own(s):
    from jax_llama_b200.ops import int8 as I
    from jax_llama_b200.ops import kernels as K
    if s["op"] == "rows":
        return I.quantize_rows(s["x"])
    if "weight" not in s:                                                     # as a model holds its layers
        s["weight"] = I.Int8Weight(s["values"], s["scales"])
    mode = {"plain": K.PLAIN, "residual": K.RESIDUAL, "gated": K.SWIGLU}[s["form"]]
    if s["op"] == "linear":
        return I.linear_int8(s["x"], s["weight"], residual=s["residual"], mode=mode, resident=True)
    return I.expert_linear_int8(s["x"], s["weight"], s["offsets"], rows=s["source"], mode=mode)


def _plain_rows(s):
    q, scale = _in_8_bits(s["x"])
    return q.to(torch.int8), scale


def _finish(y, s):
    if s["form"] == "gated":
        gate, up = y[..., 0::2], y[..., 1::2]
        y = gate / (1.0 + torch.exp(-gate)) * up
    elif s["form"] == "residual":
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_linear(s):
    q, scale = _in_8_bits(s["x"])
    y = (q.float() @ s["values"].float().t()) * scale[:, None] * s["scales"]
    return _finish(y, s)


def _plain_experts(s):
    """The rows of every expert in a batch of products of the most that one expert has."""
    q, scale = _in_8_bits(s["x"])
    source, expert = s["source"].long(), s["expert"]
    at = torch.arange(source.numel(), device=DEV) - s["offsets"].long()[expert]
    rows = torch.zeros(s["experts"], s["most"], s["k"], device=DEV)
    rows[expert, at] = q.float()[source]
    y = torch.bmm(rows, s["values"].float().transpose(1, 2))[expert, at]
    return _finish(y * scale[source, None] * s["scales"][expert], s)


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    largest = x.abs().max(-1).values
    held = torch.round(127.0 * x / largest[:, None])
    if case["op"] == "rows":
        return held.to(torch.int8), largest / 127.0
    held = torch.where(largest[:, None] > 0, held, torch.zeros_like(held))
    step, w, w_step = largest / 127.0, s["values"], s["scales"].double()
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", held, w.double()) * torch.outer(step, w_step)
    else:
        y = torch.empty(s["source"].numel(), case["n"], dtype=torch.float64, device=DEV)
        ends = s["offsets"].tolist()
        for e in range(case["experts"]):
            rows = s["source"][ends[e]:ends[e + 1]].long()
            y[ends[e]:ends[e + 1]] = (held[rows] @ w[e].double().T) * torch.outer(step[rows], w_step[e])
    if case["form"] == "gated":
        return torch.sigmoid(y[:, ::2]) * y[:, ::2] * y[:, 1::2]
    return y + s["residual"].double() if case["form"] == "residual" else y


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    k = case["k"]
    if case["op"] == "rows":
        return {"bytes": case["rows"] * (k * (size + 1) + 4), "flops": 2.0 * case["rows"] * k}
    n, form = case["n"], case["form"]
    out = n // 2 if form == "gated" else n
    if case["op"] == "linear":
        m = case["rows"]
        return {"bytes": n * (k + 4) + m * size * (k + out + (n if form == "residual" else 0)), "flops": 2.0 * m * n * k}
    rows, some = case["tokens"] * case["top"], min(case["experts"], case["tokens"] * case["top"])
    return {"bytes": some * n * (k + 4) + case["tokens"] * k * size + rows * (4 + out * size), "flops": 2.0 * rows * n * k}
