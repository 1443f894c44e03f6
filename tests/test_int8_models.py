"""8-bit weights of the LLaMA model class and the engine: what is held, and what is refused.  (On the CPU; the engine itself: test_gpu_int8_models.py.)"""
import os
import subprocess
import sys
import types

import pytest
import torch

from jax_llama_b200 import LLaMAConfig, LLaMAForCausalLM, LLaMAModel
from jax_llama_b200.models import reference as ref
from jax_llama_b200.models.engine import B200Engine, LayerWeights
from jax_llama_b200.ops.int8 import Int8Weight

CFG = dict(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, max_sequence_length=32)


@pytest.fixture
def built(monkeypatch):
    """What from_tree and random_init hand to the engine."""
    seen = {}

    def init(self, config, embedding, layers, final_norm, lm_head, **kw):
        seen.update(embedding=embedding, layers=layers, lm_head=lm_head, **kw)

    monkeypatch.setattr(B200Engine, "__init__", init)
    return seen


def _all_int8(layers):
    return all(isinstance(getattr(l, n), Int8Weight) for l in layers for n in LayerWeights.MATRICES)


def test_a_layer_in_8_bits_leaves_the_layer_as_it_was():
    w = torch.randn(8, 16).to(torch.bfloat16)
    layer = LayerWeights(torch.ones(16), w, w, torch.ones(16), w, w)
    low = layer.in_8_bits()
    assert all(getattr(layer, n) is w for n in LayerWeights.MATRICES) and _all_int8([low]) and low.attn_norm is layer.attn_norm
    assert all(getattr(low.in_8_bits(), n) is getattr(low, n) for n in LayerWeights.MATRICES)
    assert torch.equal(low.wo.values, Int8Weight.of(w).values)


def test_layers_are_in_8_bits_as_they_are_built(built):
    """(One in bf16 at a time: the whole model never is.)"""
    cfg = LLaMAConfig(**CFG)
    tree = ref.init_params(cfg, seed=0)
    B200Engine.from_tree(cfg, tree, weights="int8", device="cpu")
    assert len(built["layers"]) == 2 and _all_int8(built["layers"])
    low = built["layers"]
    B200Engine.from_tree(cfg, tree)
    full = built["layers"]
    assert all(torch.is_tensor(getattr(l, n)) for l in full for n in LayerWeights.MATRICES)
    assert all(torch.equal(getattr(a, n).values, Int8Weight.of(getattr(b, n)).values) for a, b in zip(low, full) for n in LayerWeights.MATRICES)
    B200Engine.random_init(cfg, "cpu", weights="int8")
    assert _all_int8(built["layers"])


def test_refusals_of_the_engine_ahead_of_any_work(built):
    cfg = LLaMAConfig(**CFG)
    for make in (lambda **kw: B200Engine.from_tree(cfg, {}, **kw), lambda **kw: B200Engine.random_init(cfg, "cpu", **kw)):
        with pytest.raises(ValueError, match="int4"):
            make(weights="int4")
        with pytest.raises(NotImplementedError):
            make(weights="int8", tp=2)


def test_layers_in_8_bits_are_no_bf16_engine():
    cfg = LLaMAConfig(**CFG)
    w = torch.randn(8, 16).to(torch.bfloat16)
    layer = LayerWeights(torch.ones(16), w, w, torch.ones(16), w, w)
    with pytest.raises(ValueError, match="bf16"):
        B200Engine(cfg, w, [layer, layer.in_8_bits()], torch.ones(16), w)
    with pytest.raises(ValueError, match="bf16"):
        B200Engine(cfg, w, [layer], torch.ones(16), Int8Weight.of(w))


def test_parameters_on_the_cpu_are_refused():
    """The reference backend has the full weights: it is not what a model of 8-bit weights answers with."""
    cfg = LLaMAConfig(**CFG)
    ids = torch.randint(0, 64, (1, 5))
    for make in (lambda: LLaMAForCausalLM(cfg, weights="int8"), lambda: LLaMAModel(cfg, weights="int8")):
        model = make()
        with pytest.raises(ValueError, match="CUDA"):
            model(ids)
    model = LLaMAForCausalLM(cfg, weights="int8")
    with pytest.raises(ValueError, match="CUDA"):
        model.generate(ids, max_length=8)
    with pytest.raises(ValueError, match="CUDA"):
        model.init_cache(1, 8, model.params)
    assert LLaMAForCausalLM(cfg, weights="bf16")(ids).logits.shape == (1, 5, 64)


def test_what_only_the_full_weights_give_is_refused():
    model = LLaMAForCausalLM(LLaMAConfig(**CFG), _do_init=False, weights="int8")
    here = {"engine": types.SimpleNamespace(device=torch.device("cuda"), weights="int8")}
    for kw in (dict(output_attentions=True), dict(output_hidden_states=True)):
        with pytest.raises(NotImplementedError, match="int8"):
            model._use_engine(here, kw.get("output_attentions", False), kw.get("output_hidden_states", False))
    assert model._use_engine(here, False, False)


def test_values_and_engines_that_do_not_fit():
    cfg = LLaMAConfig(**CFG)
    with pytest.raises(ValueError, match="int4"):
        LLaMAForCausalLM(cfg, weights="int4")
    low, full = ({"engine": types.SimpleNamespace(device=torch.device("cuda"), weights=w)} for w in ("int8", "bf16"))
    for weights, bad, good in (("int8", full, low), ("bf16", low, full)):
        model = LLaMAForCausalLM(cfg, _do_init=False, weights=weights)
        with pytest.raises(ValueError, match="weights"):
            model._engine_for(bad)
        assert model._engine_for(good) is good["engine"]
    plain = LLaMAForCausalLM(cfg, _do_init=False)
    assert plain._engine_for(low) is low["engine"] and plain._engine_for(full) is full["engine"]


def test_the_example_on_the_cpu_has_no_8_bit_weights(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "example.py"), "--ckpt_dir", str(tmp_path), "--tokenizer_path", "none", "--device", "cpu", "--weights", "int8"],
                       capture_output=True, text=True, timeout=300, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert r.returncode != 0 and "needs a CUDA device" in r.stderr
