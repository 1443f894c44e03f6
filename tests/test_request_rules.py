"""What a request may ask beyond sampling, on the CPU path: rules on its tokens, several answers, a common prefix."""
import math

import pytest
import torch

from jax_llama_b200 import LLaMA, LLaMA2Tokenizer, LLaMAConfig, LLaMAForCausalLM, LogitRules, allowed_mask
from jax_llama_b200.models.reference import join_prefix
from jax_llama_b200.ops import kernels as K
from jax_llama_b200.ops.rules import BoundRules

from . import prefix_oracle as oracle


@pytest.fixture(scope="module")
def model():
    cfg = LLaMAConfig(vocab_size=300, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_sequence_length=128, initializer_range=0.2)
    return LLaMAForCausalLM(cfg, seed=0)


def prompts(rows, n, seed):
    return torch.randint(3, 300, (rows, n), generator=torch.Generator().manual_seed(seed))


def test_bind_lays_out_rows_and_answers():
    b = LogitRules(repetition_penalty=[1.0, 1.5], presence_penalty=0.25, logit_bias=[{3: 1.0}, {4: -math.inf, 2: 2.0, 7: 0.5}], allowed_tokens=[[0, 31, 32], None]).bind(
        2, 40, "cpu", repeat=2)
    assert b.repetition.tolist() == [1.0, 1.0, 1.5, 1.5] and b.frequency.tolist() == [0.0] * 4 and b.presence.tolist() == [0.25] * 4
    assert b.bias_ids.tolist() == [[3, -1, -1, -1]] * 2 + [[2, 4, 7, -1]] * 2 and b.bias_values[2, :3].tolist() == [2.0, -math.inf, 0.5]
    assert b.allowed.shape == (4, 2) and b.allowed[0].tolist() == [-2 ** 31 + 1, 1] and b.allowed[2].tolist() == [-1, 255]
    one = LogitRules(logit_bias={1: 2.0}, allowed_tokens=[5]).bind(3, 40, "cpu")
    assert one.repetition is None and one.bias_ids.shape == (1, 1) and one.allowed.shape == (1, 2)
    assert not LogitRules().active and LogitRules(frequency_penalty=0.1).active and LogitRules(allowed_tokens=[]).active
    same = LogitRules(logit_bias={9: 1.0}, allowed_tokens=allowed_mask([1, 2], 40)).bind(3, 40, "cpu")
    assert one.structure() == same.structure() and one.copy_(same).bias_ids.tolist() == [[9]] and one.allowed[0, 0] == 6
    assert isinstance(one, BoundRules)
    some = torch.tensor([1, 2]).numpy()                                      # ids of any whole type
    assert LogitRules(allowed_tokens=list(some)).bind(3, 40, "cpu").allowed[0, 0] == 6 and LogitRules(allowed_tokens=some).bind(3, 40, "cpu").allowed[0, 0] == 6


@pytest.mark.parametrize("kw", [dict(repetition_penalty=0.0), dict(repetition_penalty=math.inf), dict(repetition_penalty=[1.0, 1.0, 1.0]), dict(frequency_penalty=math.nan),
                                dict(logit_bias={40: 1.0}), dict(logit_bias={-1: 1.0}), dict(logit_bias={1: math.nan}), dict(logit_bias=[{1: 1.0}]),
                                dict(allowed_tokens=[40]), dict(allowed_tokens=[[1]]), dict(allowed_tokens=torch.zeros(1, dtype=torch.int32)),
                                dict(allowed_tokens=torch.zeros(2, 2))])
def test_rules_are_refused(kw):
    with pytest.raises(ValueError):
        LogitRules(**kw).bind(2, 40, "cpu")


def test_rules_of_a_step_are_the_definition(model):
    """Greedy under every rule at once: each token is the arg-max of the model's logits under the definition."""
    ids = prompts(2, 7, 1)
    kw = dict(repetition_penalty=[1.3, 0.8], frequency_penalty=0.7, presence_penalty=[0.2, -0.1], logit_bias={5: 1.5, 9: -2.0}, allowed_tokens=range(0, 300, 3))
    got = model.generate(ids, max_new_tokens=9, eos_token_id=-5, rules=LogitRules(**kw)).sequences
    mask = allowed_mask(range(0, 300, 3), 300)[None]
    for t in range(7, 16):
        want = oracle.rules(model(got[:, :t]).logits[:, -1], got, [0, 0], [t, t], [7, 7], [1.3, 0.8], [0.7, 0.7], [0.2, -0.1],
                            torch.tensor([[5, 9]]), torch.tensor([[1.5, -2.0]]), mask)
        assert torch.equal(want.argmax(-1), got[:, t])
    assert all(t % 3 == 0 for row in got[:, 7:].tolist() for t in row)


def test_padding_is_not_a_token_that_occurred(model):
    ids, mask = prompts(2, 6, 2), torch.ones(2, 6, dtype=torch.int32)
    mask[1, :3] = 0
    rules = LogitRules(repetition_penalty=5.0)
    both = model.generate(ids, mask, max_new_tokens=6, eos_token_id=-5, rules=rules).sequences
    alone = model.generate(ids[1:, 3:], max_new_tokens=6, eos_token_id=-5, rules=rules).sequences
    assert torch.equal(both[1, 6:], alone[0, 3:])


def test_several_answers_and_prefixes_are_the_rows_written_out(model):
    ids, front = prompts(4, 5, 3), prompts(2, 6, 4)
    mask, fmask = torch.ones(4, 5, dtype=torch.int32), torch.ones(2, 6, dtype=torch.int32)
    mask[0, :2], mask[3, :5], fmask[1, :3] = 0, 0, 0                        # one prompt is its prefix alone
    joined, jmask = join_prefix(front, ids, fmask, mask, 0)
    want = model.generate(joined.repeat_interleave(2, 0), jmask.repeat_interleave(2, 0), max_new_tokens=4, eos_token_id=-5, pad_token_id=0).sequences
    got = model.generate(ids, mask, max_new_tokens=4, eos_token_id=-5, pad_token_id=0, num_return_sequences=2, prefix_ids=front, prefix_mask=fmask).sequences
    assert torch.equal(got, want) and got.shape == (8, 15)
    a = model.generate(ids[:1], max_new_tokens=8, do_sample=True, top_k=0, eos_token_id=-5, num_return_sequences=6, seed=3).sequences
    assert a.shape == (6, 13) and torch.equal(a[:, :5], ids[:1].expand(6, 5)) and len({tuple(r) for r in a.tolist()}) > 1
    for bad in (dict(num_return_sequences=0), dict(prefix_ids=front[0]), dict(prefix_ids=prompts(3, 4, 0)), dict(prefix_ids=front, max_length=9)):
        with pytest.raises(ValueError):
            model.generate(ids, **{"max_new_tokens": 2, "eos_token_id": -5, **bad})


def test_joined_prompts_keep_order_and_left_padding():
    g = torch.Generator().manual_seed(0)
    for G, n, P, S in ((1, 3, 4, 5), (2, 2, 1, 1), (3, 1, 6, 0), (1, 2, 0, 3)):
        front, ids = torch.randint(1, 99, (G, P), generator=g), torch.randint(1, 99, (G * n, S), generator=g)
        fp, ip = torch.randint(0, P + 1, (G,), generator=g), torch.randint(0, S + 1, (G * n,), generator=g)
        got, mask = join_prefix(front, ids, (torch.arange(P)[None] >= fp[:, None]).int(), (torch.arange(S)[None] >= ip[:, None]).int(), 0)
        for b in range(G * n):
            row = front[b // n, fp[b // n]:].tolist() + ids[b, ip[b]:].tolist()
            pads = P + S - len(row)
            assert got[b].tolist() == [0] * pads + row and mask[b].tolist() == [0] * pads + [1] * len(row)


def test_text_front_end(spm_model):
    tok = LLaMA2Tokenizer(spm_model)
    cfg = LLaMAConfig(vocab_size=len(tok), hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, max_sequence_length=128,
                      initializer_range=0.2, bos_token_id=tok.bos_id, eos_token_id=tok.eos_id)
    model = LLaMAForCausalLM(cfg, seed=1)
    gen = LLaMA(model.params, model, tok)
    texts = gen.generate_from_str(["the city", "hello world is here"], max_gen_len=5, temperature=0.0, top_p=1.0, prefix="The capital of germany", num_return_sequences=2)
    assert len(texts) == 4 and texts[0] == texts[1] and texts[2] == texts[3] and all(t.startswith("The capital of germany") for t in texts)
    only = [i for i in range(len(tok)) if i % 2 == 0]
    tokens, mask, _ = gen.encode_prompts(["hello"])
    out = gen.generate(tokens, mask, 6, temperature=0.7, rules=LogitRules(allowed_tokens=only + [tok.eos_id]), seed=2)
    assert all(t % 2 == 0 or t == tok.eos_id for t in out[0, tokens.shape[1]:].tolist())


def attention_case(dtype=torch.float32, **kw):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=dtype)      # noqa: E731
    c = dict(qkv=r(4, 8 * 64), pk=r(2, 2, 9, 64), pv=r(2, 2, 9, 64), kc=r(4, 2, 6, 64), vc=r(4, 2, 6, 64), cos=r(20, 32), sin=r(20, 32),
             n=torch.tensor([3], dtype=torch.int32), pad=None, plen=None, ppad=None)
    c.update(kw)
    return c


def step(c, **kw):
    return K.decode_attn_prefix(c["qkv"], c["pk"], c["pv"], c["kc"], c["vc"], c["cos"], c["sin"], c["n"], c["pad"], c["plen"], c["ppad"], 4, 2, 64, **kw)


@pytest.mark.parametrize("bad", [dict(qkv=torch.zeros(4, 512 - 64)), dict(pk=torch.zeros(3, 2, 9, 64), pv=torch.zeros(3, 2, 9, 64)), dict(pv=torch.zeros(2, 2, 8, 64)),
                                 dict(pk=torch.zeros(2, 1, 9, 64), pv=torch.zeros(2, 1, 9, 64)), dict(vc=torch.zeros(4, 2, 7, 64)), dict(kc=torch.zeros(3, 2, 6, 64), vc=torch.zeros(3, 2, 6, 64)),
                                 dict(pk=torch.zeros(2, 2, 0, 64), pv=torch.zeros(2, 2, 0, 64)), dict(n=torch.tensor([3])), dict(pad=torch.zeros(3, dtype=torch.int32)),
                                 dict(plen=torch.zeros(4, dtype=torch.int32)), dict(ppad=torch.zeros(2))])
def test_attention_refusals(bad):
    step(attention_case())
    with pytest.raises(ValueError):
        step(attention_case(**bad))


def test_prompt_attention_refusals():
    c = attention_case()
    q = torch.zeros(4, 3, 4, 64)
    run = lambda q=q, start=1, S=3, pad=None: K.prefill_attn_prefix(q, c["pk"], c["pv"], c["kc"], c["vc"], start, S, pad, None, None)      # noqa: E731
    assert run().shape == (4, 3, 256)
    for kw in (dict(q=q[0]), dict(S=2), dict(start=4), dict(start=-1), dict(q=torch.zeros(3, 3, 4, 64)), dict(pad=torch.zeros(4))):
        with pytest.raises(ValueError):
            run(**kw)


@pytest.mark.parametrize("full", [False, True])
def test_attention_on_the_cpu_path(full):
    """The CPU statement of both forms against the definition; a full cache stores nothing."""
    g = torch.Generator().manual_seed(3)
    B, groups, nh, nkv, hd, P, T = 4, 2, 4, 2, 64, 9, 6
    r = lambda *s: torch.randn(*s, generator=g)                   # noqa: E731
    own = T if full else 4
    plen, ppad, pad = [9, 5], [2, 5], [0, 1, 3, 2]
    pk, pv, kc, vc, qkv = r(groups, nkv, P, hd), r(groups, nkv, P, hd), r(B, nkv, T, hd), r(B, nkv, T, hd), r(B, (nh + 2 * nkv) * hd)
    cos, sin = oracle.tables(hd, 40)
    x = qkv.double().view(B, nh + 2 * nkv, hd)
    turned = torch.stack([oracle.rotate(x[b, :nh + nkv], plen[b // 2] - ppad[b // 2] + own - pad[b]) for b in range(B)])
    i = lambda v: torch.tensor(v, dtype=torch.int32)              # noqa: E731
    was = kc.clone()
    got = K.decode_attn_prefix(qkv, pk, pv, kc, vc, cos, sin, i([own]), i(pad), i(plen), i(ppad), nh, nkv, hd)
    k2, v2 = torch.cat([was[:, :, :own], turned[:, nh:, None].float()], 2), torch.cat([vc[:, :, :own], x[:, nh + nkv:, None].float()], 2)
    want, _ = oracle.attention(turned[:, None, :nh], pk, pv, k2, v2, [own], pad, plen, ppad)
    assert (got.double().view_as(want) - want).abs().max() < 1e-5
    assert torch.equal(kc, was) if full else not torch.equal(kc, was)


@pytest.mark.parametrize("shape", [(2,), (1, 2), (3, 2)])
def test_bound_masks_are_not_the_callers(shape):
    """What a request brings stays what it is: neither a later batch of the same form nor a mask of a step is written into it, and its own changes do not reach a batch at work."""
    mask = allowed_mask([1, 39], 40).expand(shape).clone()
    was, bound = mask.clone(), LogitRules(allowed_tokens=mask).bind(3, 40, "cpu")
    bound.copy_(LogitRules(allowed_tokens=torch.zeros_like(mask)).bind(3, 40, "cpu"))
    assert torch.equal(mask, was) and not bound.allowed.any()
    bound = LogitRules(allowed_tokens=mask).bind(3, 40, "cpu")
    mask.zero_()
    assert torch.equal(bound.allowed, was.view(-1, 2))


@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (50, 1.0), (0, 0.9), (50, 0.9)])
def test_a_row_without_a_token_left_takes_the_first(model, top_k, top_p):
    """Sampling from masks that leave nothing, or nothing in one row: token 0 as with the arg-max and on the GPU, the other rows as they would be."""
    ids, kw = prompts(2, 5, 1), dict(max_new_tokens=4, do_sample=True, top_k=top_k, top_p=top_p, eos_token_id=-5, seed=2)
    assert not model.generate(ids, rules=LogitRules(allowed_tokens=[]), **kw).sequences[:, 5:].any()
    one = model.generate(ids, rules=LogitRules(allowed_tokens=[[], range(40, 60)]), **kw).sequences[:, 5:]
    assert not one[0].any() and set(one[1].tolist()) <= set(range(40, 60))
    assert torch.equal(one[1], model.generate(ids, rules=LogitRules(allowed_tokens=[range(300), range(40, 60)]), **kw).sequences[1, 5:])
