"""Mixtures of experts whose matrices are held in 8 bits, in the layers and the engine of the hybrid families."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200.config import MoeMlpSpec                                     # noqa: E402
from jax_llama_b200.models.feedforward import MoeFeedForward                     # noqa: E402
from jax_llama_b200.models.hybrid_engine import HybridEngine, random_tensors     # noqa: E402
from jax_llama_b200.models.nikonex import NikonexForCausalLM                     # noqa: E402
from jax_llama_b200.ops import int8 as I                                         # noqa: E402

from tests import test_gpu_nikonex as N                                          # noqa: E402

SPECS = {
    "relu2, shared": MoeMlpSpec(experts=8, top=2, ff=64, groups=4, keep=2, shared_ff=40),
    "silu": MoeMlpSpec(experts=6, top=3, ff=48, act="silu", gated=True, score="softmax"),
    "silu, odd sizes": MoeMlpSpec(experts=5, top=2, ff=41, act="silu", gated=True, shared_ff=24, shared_gate=False),
    "clamped": MoeMlpSpec(experts=4, top=2, ff=64, act="glu_clamped", gated=True, limit=7.0, shared_limit=7.0, score="softmax"),
    "silu, identity": MoeMlpSpec(experts=6, top=3, ff=64, act="silu", gated=True, identity=3, choice_bias=True, score="softmax"),
}


def tensors(spec, W, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {k: (torch.randn(s, generator=g, device="cuda") * (s[-1] ** -0.5 if len(s) > 1 else 0.1)).to(dtype) for k, s in MoeFeedForward.shapes(spec, W).items()}


def numbers(w, spec):
    """The same layer with the numbers that the experts' 8-bit weights stand for."""
    return {k: I.Int8Weight.of(v).float().to(v.dtype) if k[0] == "e" and k.split(".")[1] in ("up", "down", "gate") else v for k, v in w.items()}


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 5, 40, 700])
def test_layer(name, dtype, M):
    """Against the layer with the same numbers in the engine's type: the same router, so the same choices.  What is left is rounding rows of activations to 8 bits, twice: half a step,
    amax / 254, per element, of a row's norm at most (amax / rms) / 254: 2 % with amax / rms = 5 for the inputs (squared by relu2: 4 %), 3.2 % for hidden rows of up to 64
    (amax / rms <= 8); bfloat16 adds half a percent per product: below 9 % together."""
    spec, W = SPECS[name], 96
    w = tensors(spec, W, dtype)
    layer, plain = MoeFeedForward(spec, w, weights="int8"), MoeFeedForward(spec, numbers(w, spec))
    h = torch.randn(M, W, device="cuda", generator=torch.Generator(device="cuda").manual_seed(M)).to(dtype)
    got, want = layer.run(h), plain.run(h)
    assert got.dtype is torch.float32 and got.shape == want.shape
    assert ((got - want).norm() / want.norm()).item() < 0.09
    assert torch.equal(layer.run(h), got)
    size = sum(t.numel() * t.element_size() for t in layer.weights()), sum(t.numel() * t.element_size() for t in plain.weights())
    assert size[0] < size[1]


def test_rows_do_not_depend_on_the_batch():
    """Products of whole numbers: a token's experts give the same bits whatever runs beside it."""
    spec = SPECS["silu"]
    layer = MoeFeedForward(spec, tensors(spec, 96, torch.float32), weights="int8")
    h = torch.randn(300, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    idx = torch.stack([torch.randperm(6, generator=torch.Generator().manual_seed(m))[:3] for m in range(300)]).to(torch.int32).cuda()
    y, pos = layer._experts_int8(h, idx)
    for M in (1, 7, 90):
        z, p = layer._experts_int8(h[:M], idx[:M].contiguous())
        assert torch.equal(z[p.long()], y[pos.view(300, 3)[:M].reshape(-1).long()])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_engine(dtype):
    cfg = N.config(N.MIXED)
    params = random_tensors(cfg, "cuda", 3)
    eng = HybridEngine(cfg, params, dtype=dtype, expert_weights="int8")
    eager = HybridEngine(cfg, params, dtype=dtype, expert_weights="int8", use_cuda_graph=False)
    full = HybridEngine(cfg, params, dtype=dtype)
    assert eng.weight_bytes_per_step(4) < full.weight_bytes_per_step(4)
    ids = torch.randint(0, cfg.vocab_size, (3, 21), generator=torch.Generator().manual_seed(1)).cuda()
    a, b = (e.generate(ids, max_length=40, do_sample=False) for e in (eng, eager))
    assert a.shape == (3, 40) and torch.equal(a, b)
    model = NikonexForCausalLM(cfg, dtype=dtype, expert_weights="int8")
    model.params = params
    assert torch.equal(model(ids).logits, eng.forward(ids).logits)


def test_refusals():
    cfg = N.config([N.lat(), N.ret()])
    with pytest.raises(ValueError, match="no mixture"):
        HybridEngine(cfg, random_tensors(cfg, "cuda", 0), expert_weights="int8")
    with pytest.raises(ValueError, match="expert_weights"):
        HybridEngine(N.config(N.MIXED), {}, expert_weights="int4")
