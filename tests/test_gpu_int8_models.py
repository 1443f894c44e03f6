"""LLaMA engines with 8-bit weights: what they take of their caller's tensors and of the GPU's memory."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200 import LLaMAConfig, LLaMAForCausalLM                    # noqa: E402
from jax_llama_b200.convert_weights import write_meta_checkpoint            # noqa: E402
from jax_llama_b200.models import reference as ref                          # noqa: E402
from jax_llama_b200.models.engine import B200Engine                       # noqa: E402
from jax_llama_b200.models.llama import tree_to                             # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_sequence_length=256,
                  initializer_range=0.05)
DEEP = LLaMAConfig(vocab_size=1000, hidden_size=1024, intermediate_size=4096, num_hidden_layers=24, num_attention_heads=8, num_key_value_heads=8, max_sequence_length=64)


def generate(eng, B=2):
    ids = torch.randint(3, CFG.vocab_size, (B, 9), generator=torch.Generator().manual_seed(B)).cuda()
    return eng.generate(ids, max_length=24, do_sample=False, eos_token_id=-1, pad_token_id=0)


def test_engines_of_the_same_layers():
    """A bf16 engine, two in 8 bits from its layers: none changes what another one holds."""
    tree = tree_to(tree_to(ref.init_params(CFG, seed=1), dtype=torch.bfloat16), device="cuda")
    full = B200Engine.from_tree(CFG, tree)
    want, before = generate(full), [(l, l.wqkv, l.w2) for l in full.layers]
    a, b = (B200Engine(CFG, full.embedding, full.layers, full.final_norm, full.lm_head, weights="int8") for _ in range(2))
    assert all(l.wqkv is q and l.w2 is d and torch.is_tensor(q) for l, q, d in before)
    assert torch.equal(generate(full), want)
    low = generate(B200Engine.from_tree(CFG, tree, weights="int8"))
    assert torch.equal(generate(a), low) and torch.equal(generate(b), low)
    assert torch.equal(generate(B200Engine(CFG, full.embedding, a.layers, full.final_norm, a.lm_head, weights="int8")), low)
    with pytest.raises(ValueError):
        B200Engine(CFG, full.embedding, a.layers, full.final_norm, full.lm_head)


def _matrices(cfg):
    h, hd = cfg.hidden_size, cfg.head_dim
    return h * (cfg.num_attention_heads + 2 * cfg.num_key_value_heads) * hd + h * cfg.num_attention_heads * hd + 3 * h * cfg.intermediate_size


@pytest.mark.parametrize("how", ["host tree", "random"])
def test_memory_while_an_engine_is_built(how):
    """8-bit layers and one layer's working forms: fp32, bf16 and 64-bit numbers of the largest of its matrices (24 bytes a weight are ample), nothing that grows with the number of layers beyond a byte and scales."""
    tree = ref.init_params(DEEP, seed=0, dtype=torch.bfloat16) if how == "host tree" else None
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    eng = B200Engine.from_tree(DEEP, tree, device="cuda", weights="int8") if how == "host tree" else B200Engine.random_init(DEEP, "cuda", weights="int8")
    torch.cuda.synchronize()
    peak, layer, L = torch.cuda.max_memory_allocated() - start, _matrices(DEEP), DEEP.num_hidden_layers
    assert eng.weight_bytes_per_step() > L * layer
    assert peak < 1.01 * L * layer + 24 * layer + (64 << 20)
    assert peak < 2 * L * layer                                # (what the layers in bf16 alone would take)


def test_an_engine_as_the_parameters():
    """The model class on an engine that was built from a tree in host memory: no bf16 tree on the GPU."""
    tree = tree_to(ref.init_params(CFG, seed=1), dtype=torch.bfloat16)
    eng = B200Engine.from_tree(CFG, tree, device="cuda", weights="int8")
    model = LLaMAForCausalLM(CFG, _do_init=False, weights="int8")
    ids = torch.randint(3, CFG.vocab_size, (2, 11), generator=torch.Generator().manual_seed(5))
    want = LLaMAForCausalLM(CFG, _do_init=False, weights="int8")(ids, params=tree_to(tree, device="cuda")).logits
    assert torch.equal(model(ids, params={"engine": eng}).logits, want)


def test_the_example_in_8_bits(tmp_path, spm_model):
    spm = pytest.importorskip("sentencepiece")
    vocab = spm.SentencePieceProcessor(model_file=spm_model).vocab_size()
    cfg = LLaMAConfig(vocab_size=vocab, hidden_size=256, intermediate_size=768, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_sequence_length=64)
    write_meta_checkpoint(ref.init_params(cfg, seed=0), cfg, str(tmp_path / "ckpt"), mp=1, dtype=torch.float32, multiple_of=256)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "example.py"), "--ckpt_dir", str(tmp_path / "ckpt"), "--tokenizer_path", spm_model, "--weights", "int8", "--max_gen_len", "4",
                        "--temperature", "0", "--prompt", "hello world"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1500:]
    assert r.stdout.count("==================================") == 1 and "hello world" in r.stdout.lower()
