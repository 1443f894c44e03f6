"""What layers and engines with 8-bit weights hand to their products, stage by stage against 64 bits: every result row of every product, from the numbers that the stage was given and the
matrices that the model was built from.  A wrong scale, row, order, expert or norm in between is off by far more than the roundings that are allowed here."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200 import LLaMAConfig                                          # noqa: E402
from jax_llama_b200.models import reference as ref                              # noqa: E402
from jax_llama_b200.models.engine import B200Engine                             # noqa: E402
from jax_llama_b200.models.feedforward import GLU_ALPHA, MoeFeedForward         # noqa: E402
from jax_llama_b200.models.llama import tree_to                                 # noqa: E402
from jax_llama_b200.ops import int8 as I                                        # noqa: E402
from jax_llama_b200.ops import kernels as K                                     # noqa: E402
from jax_llama_b200.ops import seq_kernels as SK                                # noqa: E402

from tests import int8_oracle as O                                              # noqa: E402
from tests.test_gpu_int8_experts import SPECS, tensors                          # noqa: E402

U = O.U


def within(got, off, want):
    err = (got.double() - want).abs()
    worst = err / off.clamp(min=1e-300)
    assert bool((err <= off).all()), f"off by {worst.max().item():.3g} of the bound, row {int(worst.amax(-1).argmax())}"


# --------------------------------------------------------------------------- a mixture's layer
def clamped(y, F, limit, dtype):
    """g σ(alpha g) (u + 1) of gate and up numbers that are off by three roundings each: the sigmoid by |alpha g| times five of them and six of its own, three products, the sum."""
    g, u = y[:, :F], y[:, F:]
    dg = du = 3.1 * U
    live = (u.abs() < limit).double()
    g2, u2 = g.clamp(max=limit), u.clamp(-limit, limit)
    s = torch.sigmoid(GLU_ALPHA * g2)
    t = g2 * s * (u2 + 1)
    off = t.abs() * (dg + 5.1 * U * (GLU_ALPHA * g2).abs() + 10 * U) + (g2 * s).abs() * (du * u2.abs() * live + 1.1 * U * (u2 + 1).abs())
    return off + O.half_step(dtype) * (t.abs() + off) + O.smallest(dtype), t


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 2, 5, 40, 700])
def test_a_mixture(name, dtype, M, monkeypatch):
    spec, W = SPECS[name], 96
    w = tensors(spec, W, dtype, seed=M)
    layer = MoeFeedForward(spec, w, weights="int8")
    rest = MoeFeedForward(spec, {k: torch.zeros_like(v) if k[0] == "e" and k.split(".")[1] in ("up", "down", "gate") else v for k, v in w.items()})      # shared and identity experts
    h = torch.randn(M, W, device="cuda", generator=torch.Generator(device="cuda").manual_seed(M)).to(dtype)
    hidden, results, routes, orders = [], [], [], []

    def recorded(fn, into):
        def call(*args, **kw):
            out = fn(*args, **kw)
            into.append(out)
            return out
        return call

    few = M * spec.top <= I.MAX_CHOICES
    which = "choice_linear_int8" if few else "expert_linear_int8"
    real = getattr(I, which)

    def product(x, weight, *args, **kw):
        out = real(x, weight, *args, **kw)
        (hidden if weight is layer.up8 else results).append((x.clone(), out))
        return out

    monkeypatch.setattr(I, which, product)
    monkeypatch.setattr(I, "expert_order", recorded(I.expert_order, orders))
    monkeypatch.setattr(SK, "moe_route", recorded(SK.moe_route, routes))
    got = layer.run(h)
    assert (len(hidden), len(results), len(routes), len(orders)) == (1, 1, 1, 0 if few else 1)
    idx, wt = routes[0]
    pos = torch.arange(M * spec.top, device="cuda") if few else orders[0][0].long()
    t_all, y_all = results[0]
    expert, token = idx.view(-1).long(), torch.arange(M, device="cuda").repeat_interleave(spec.top)
    total, size = torch.zeros(M, W, dtype=torch.float64, device="cuda"), torch.zeros(M, W, dtype=torch.float64, device="cuda")
    share = wt.double().view(-1)
    assert torch.equal(hidden[0][0], h) and (few or len(set(pos[expert >= 0].tolist())) == int((expert >= 0).sum()))
    for e in range(spec.experts):
        at = (expert == e).nonzero().view(-1)
        if not len(at):
            continue
        up = torch.cat([w[f"e{e}.gate"], w[f"e{e}.up"]]) if spec.gated else w[f"e{e}.up"]
        y = O.products(*O.rows(h[token[at]]), *O.rows(up))
        if spec.act == "relu2":
            bound = O.bound_relu2(y, dtype)
        elif spec.act == "silu":
            bound = O.bound_gated(torch.stack([y[:, :spec.ff], y[:, spec.ff:]], 2).flatten(1), dtype)
        else:
            bound = clamped(y, spec.ff, spec.limit, dtype)
        t = t_all[pos[at]]
        within(t, *bound)
        y = O.products(*O.rows(t), *O.rows(w[f"e{e}.down"]))
        within(y_all[pos[at]], *O.bound(y, torch.float32))
        part = share[at, None] * y_all[pos[at]].double()
        total.index_add_(0, token[at], part)
        size.index_add_(0, token[at], part.abs())
    other = rest.run(h).double()
    # the weighted sum and what it is added to: a rounding for every product and addition
    within(got, (spec.top + 5) * 1.1 * U * (size + other.abs()) + 2.0 ** -140, total + other)


# --------------------------------------------------------------------------- the LLaMA engine
CFGS = {
    "gqa128": LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_sequence_length=256,
                          initializer_range=0.05),
    "tied64": LLaMAConfig(vocab_size=777, hidden_size=320, intermediate_size=600, num_hidden_layers=2, num_attention_heads=5, num_key_value_heads=5, max_sequence_length=128,
                          initializer_range=0.05, tie_word_embeddings=True),
}


def rows_behind_a_norm(x, g, eps):
    """Values and scales in 64 bits, where values may be a neighbour, and how far a scale may be off (as derived in test_gpu_int8_norm.py)."""
    xd = x.double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + eps).sqrt() * g.double()
    amax = h.abs().amax(-1, keepdim=True)
    t = 127.0 * h / amax
    return t.round(), amax[:, 0] / 127.0, ((t - t.floor() - 0.5).abs() < 127.0 * 40 * U).double()


@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("B,S", [(1, 1), (1, 5), (2, 7), (1, 40), (3, 100)])
def test_the_engine(name, B, S, monkeypatch):
    cfg = CFGS[name]
    tree = tree_to(ref.init_params(cfg, seed=1), dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    for l in tree["transformer"]["h"].values():               # norms that do something
        for n in ("attention_norm", "ffn_norm"):
            l[n]["kernel"] = (1.0 + 0.3 * torch.randn(l[n]["kernel"].shape, generator=g)).to(torch.bfloat16)
    tree["transformer"]["ln_f"]["kernel"] = (1.0 + 0.3 * torch.randn(tree["transformer"]["ln_f"]["kernel"].shape, generator=g)).to(torch.bfloat16)
    tree = tree_to(tree, device="cuda")
    eng = B200Engine.from_tree(cfg, tree, weights="int8")
    calls, real = [], K.linear

    def linear(x, w, *, residual=None, **kw):
        x0, r0 = x.clone(), None if residual is None else residual.clone()
        out = real(x, w, residual=residual, **kw)
        calls.append((x0, w, r0, kw, out.clone()))
        return out

    monkeypatch.setattr(K, "linear", linear)
    ids = torch.randint(0, cfg.vocab_size, (B, S), generator=torch.Generator().manual_seed(B)).cuda()
    logits = eng.forward(ids).logits
    assert len(calls) == 4 * cfg.num_hidden_layers + 1
    stream = tree["transformer"]["wte"]["embedding"][ids.view(-1)]
    eps = cfg.rms_norm_eps

    def check(call, matrix, x=None, norm=None, residual=None, gated=False, dtype=torch.bfloat16):
        x0, _, r0, kw, out = call
        if x is not None:
            assert torch.equal(x0.view(x.shape), x)
        x0 = x0.view(-1, matrix.shape[1])
        assert (r0 is None) == (residual is None) and (residual is None or torch.equal(r0.view(residual.shape), residual))
        wq, ws = O.rows(matrix)
        if norm is None:
            q, s = O.rows(x0)
            y = O.products(q, s, wq, ws)
            extra = None
        else:
            q, s, near = rows_behind_a_norm(x0, norm, eps)
            y = O.products(q, s, wq, ws)
            # (a value that is the neighbour counts with the scale as it came out, and is rounded with the rest: 19 + 4 of U more)
            extra = (near @ wq.abs().t()) * s[:, None] * ws.double() * (1 + 23 * U) + 19 * U * y.abs()
        bound = O.bound_gated(y, dtype, extra=extra) if gated else O.bound(y, dtype, residual=None if residual is None else residual.view(y.shape), extra=extra)
        within(out.view(bound[1].shape), *bound)
        return out

    for i in range(cfg.num_hidden_layers):
        l = tree["transformer"]["h"][str(i)]
        a, f = l["attention"], l["feed_forward"]
        qkv, wo, w13, w2 = calls[4 * i:4 * i + 4]
        check(qkv, torch.cat([a[n]["kernel"].t() for n in ("wq", "wk", "wv")]), x=stream, norm=l["attention_norm"]["kernel"])
        stream = check(wo, a["wo"]["kernel"].t(), residual=stream)
        both = torch.stack([f["w1"]["kernel"].t(), f["w3"]["kernel"].t()], 1).flatten(0, 1)
        h = check(w13, both, x=stream, norm=l["ffn_norm"]["kernel"], gated=True)
        stream = check(w2, f["w2"]["kernel"].t(), x=h, residual=stream)
    head = tree["transformer"]["wte"]["embedding"] if cfg.tie_word_embeddings else tree["lm_head"]["kernel"].t()
    out = check(calls[-1], head, x=stream, norm=tree["transformer"]["ln_f"]["kernel"], dtype=torch.float32)
    assert torch.equal(logits.view(out.shape), out)


def test_gates_far_below_zero():
    """silu(y) is 0 where exp(-y) passes 2^126, from about y = -87.3 on, and what it is above."""
    values = torch.tensor([[127], [127]], dtype=torch.int8, device="cuda")
    for g, u in ((-80.0, 3.0), (-87.0, 1.0), (-88.0, 1.0), (-1000.0, 5.0)):
        w = I.Int8Weight(values, torch.tensor([g, u], device="cuda") / 127.0)
        for M in (1, 20, 300):
            y = I.linear_int8(torch.full((M, 1), 1.0, device="cuda"), w, mode=K.SWIGLU)
            if g < -87.5:
                assert not y.any()
            else:
                want = g * torch.sigmoid(torch.tensor(g, dtype=torch.float64)).item() * u
                assert bool(((y.double() / want - 1).abs() < 1e-4).all())          # (|g| times three roundings of g in the exponent: 87 * 3 * 2^-24 = 1.6e-5, twice the exponential's, the rest)
