"""The LLaMA engine with 8-bit weights."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200 import LLaMAConfig, LLaMAForCausalLM                    # noqa: E402
from jax_llama_b200.models import reference as ref                          # noqa: E402
from jax_llama_b200.models.engine import B200Engine                         # noqa: E402
from jax_llama_b200.models.llama import tree_to                             # noqa: E402
from jax_llama_b200.ops.int8 import Int8Weight                              # noqa: E402

CFGS = {
    "gqa128": LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_sequence_length=256,
                          initializer_range=0.05),
    "tied64": LLaMAConfig(vocab_size=777, hidden_size=320, intermediate_size=600, num_hidden_layers=2, num_attention_heads=5, num_key_value_heads=5, max_sequence_length=128,
                          initializer_range=0.05, tie_word_embeddings=True),
}


def make(name):
    cfg = CFGS[name]
    tree = tree_to(ref.init_params(cfg, seed=1), dtype=torch.bfloat16)
    return cfg, tree, B200Engine.from_tree(cfg, tree_to(tree, device="cuda"), weights="int8")


@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("B,S", [(1, 1), (2, 7), (1, 40), (3, 120)])
def test_logits_against_the_numbers_that_the_weights_stand_for(name, B, S):
    """fp32 model with the dequantised weights.  What is left is the activations' rounding to 8 bits: per element at most half a step, amax / 254, so of a row's norm at most
    (amax / rms) / 254, 2 % with amax / rms = 5 (rows of 320 to 1024 normal numbers have 3 to 4.5).  Four products a layer meet the stream, behind them the head: nine in all,
    18 % if every one of them pointed the same way."""
    cfg, tree, eng = make(name)
    assert all(isinstance(w, Int8Weight) for l in eng.layers for w in (l.wqkv, l.wo, l.w13, l.w2)) and isinstance(eng.lm_head, Int8Weight)
    numbers = tree_to(eng.to_tree(), device="cpu", dtype=torch.float32)
    ids = torch.randint(0, cfg.vocab_size, (B, S), generator=torch.Generator().manual_seed(B))
    if cfg.tie_word_embeddings:              # (the head is the table in 8 bits, the table itself stays)
        numbers["lm_head"] = {"kernel": eng.lm_head.float().t().contiguous().cpu()}
        want = ref.forward(numbers, type(cfg)(**{**cfg.to_dict(), "tie_word_embeddings": False}), ids).logits
    else:
        want = ref.forward(numbers, cfg, ids).logits
    got = eng.forward(ids.cuda()).logits.float().cpu()
    assert got.shape == want.shape
    assert ((got - want).norm() / want.norm()).item() < 0.18


@pytest.mark.parametrize("name", list(CFGS))
def test_weights_come_back_within_half_a_step(name):
    cfg, tree, eng = make(name)
    back = eng.to_tree()["transformer"]["h"]["1"]
    want = tree["transformer"]["h"]["1"]
    for part, key in (("attention", "wq"), ("attention", "wo"), ("feed_forward", "w1"), ("feed_forward", "w2"), ("feed_forward", "w3")):
        a, b = back[part][key]["kernel"].double().cpu(), want[part][key]["kernel"].double()
        step = b.abs().amax(0, keepdim=True) / 127              # [in, out]: a scale per output
        assert bool(((a - b).abs() <= step * (0.5 + 1e-4) + b.abs() * 2.0 ** -8 + step * 2.0 ** -8).all())
    full = B200Engine.from_tree(cfg, tree_to(tree, device="cuda"))
    assert 0.45 < eng.weight_bytes_per_step() / full.weight_bytes_per_step() < 0.55


@pytest.mark.parametrize("B", [1, 3, 8, 20])
def test_generation_with_and_without_a_graph(B):
    cfg, tree, eng = make("gqa128")
    plain = B200Engine.from_tree(cfg, tree_to(tree, device="cuda"), weights="int8", use_cuda_graph=False)
    ids = torch.randint(3, cfg.vocab_size, (B, 9), generator=torch.Generator().manual_seed(B)).cuda()
    a = eng.generate(ids, max_length=40, do_sample=False, eos_token_id=-1, pad_token_id=0)
    b = plain.generate(ids, max_length=40, do_sample=False, eos_token_id=-1, pad_token_id=0)
    assert a.shape == (B, 40) and torch.equal(a, b)
    assert torch.equal(eng.generate(ids, max_length=40, do_sample=False, eos_token_id=-1, pad_token_id=0), a)


def test_through_the_model_class_and_a_stream():
    cfg, tree, eng = make("gqa128")
    params = tree_to(tree, device="cuda")
    model = LLaMAForCausalLM(cfg, _do_init=False, weights="int8")
    ids = torch.randint(3, cfg.vocab_size, (2, 11), generator=torch.Generator().manual_seed(5)).cuda()
    assert torch.equal(model(ids, params=params).logits, eng.forward(ids).logits)
    assert model._engine_for(params).weights == "int8"
    want = eng.generate(ids, max_length=20, do_sample=False, eos_token_id=-1, pad_token_id=0)
    st = eng.begin_stream(ids, max_length=20, do_sample=False, eos_token_id=-1, pad_token_id=0)
    for _ in range(8):
        st.step()
    assert torch.equal(st.sequences()[:, :20], want[:, :20])
    st.close()
