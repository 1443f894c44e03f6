"""Requests with rules, several answers and common prefixes on the B200 engines, against the fp32 reference model and the definition of the rules."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200 import LLaMA, LLaMAConfig, LLaMAForCausalLM, LogitRules, allowed_mask      # noqa: E402
from jax_llama_b200.models import reference as ref                                             # noqa: E402
from jax_llama_b200.models.engine import B200Engine                                            # noqa: E402
from jax_llama_b200.models.llama import tree_to                                                # noqa: E402
from jax_llama_b200.models.reference import join_prefix                                        # noqa: E402

from . import prefix_oracle as oracle                                                          # noqa: E402

CFGS = {
    "gqa128": LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                          max_sequence_length=256, initializer_range=0.05),
    "mha64": LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=768, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=8,
                         max_sequence_length=256, initializer_range=0.05),
}


def make(name, **kw):
    cfg = CFGS[name]
    tree = tree_to(ref.init_params(cfg, seed=1), dtype=torch.bfloat16)
    eng = B200Engine.from_tree(cfg, tree_to(tree, device="cuda"), **kw)
    eng.share_above = eng.share_above_whole_step = 0         # keys held once however few they are
    return cfg, tree_to(tree, dtype=torch.float32), eng


def eng_tree(cfg):
    return tree_to(ref.init_params(cfg, seed=1), dtype=torch.bfloat16, device="cuda")


def rel(a, b):
    a, b = a.float().cpu(), b.float().cpu()
    return ((a - b).abs().max() / (b.abs().max() + 1e-6)).item()


def ids_of(rows, n, seed):
    return torch.randint(3, 1000, (rows, n), generator=torch.Generator().manual_seed(seed))


def padded(pads, n):
    return (torch.arange(n)[None] >= torch.tensor(pads)[:, None]).to(torch.int32)


@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("groups,rows,repeat,P,S,together", [(1, 3, 1, 70, 9, True), (2, 4, 3, 33, 5, True), (1, 1, 6, 40, 0, True), (3, 3, 2, 65, 0, True),
                                                             (1, 3, 1, 70, 9, False), (2, 4, 3, 33, 5, False), (1, 1, 6, 40, 0, False), (3, 3, 1, 20, 7, False)])
def test_logits_behind_a_prefix_match_the_written_out_rows(name, graph, groups, rows, repeat, P, S, together):
    """Prefix prefill, prompts behind it, steps: the logits of every fed token against the fp32 model on the joined rows (bf16 weights and activations on one
    side: the 3e-2 of the other engine tests).  S = 0: several answers to the prompts themselves."""
    cfg, tree32, eng = make(name, use_cuda_graph=graph)
    front, fpads = ids_of(groups, P, 1), [(3 * g) % 5 for g in range(groups)]
    fmask = padded(fpads, P)
    if S:
        ids, mask = ids_of(rows, S, 2), padded([(2 * b) % S if together else 0 for b in range(rows)], S)
        joined, jmask = join_prefix(front, ids, fmask, mask, 0)
        kw = dict(prefix_ids=front.cuda(), prefix_mask=fmask.cuda())
    else:
        ids, mask, joined, jmask, kw = front, fmask, front, fmask, {}
    full, fullm = joined.repeat_interleave(repeat, 0), jmask.repeat_interleave(repeat, 0)
    B, total = full.shape
    feed = ids_of(B, 4, 3)
    if not together:
        eng.mega_write_logits = True
        eng.share_above = eng.share_above_whole_step = 1 << 40
    for _ in range(2):                                       # the second time on the same caches and captured step
        stream = eng.begin_stream(ids.cuda(), mask.cuda(), max_length=total + 6, num_return_sequences=repeat, pad_token_id=0, **kw)
        assert (stream.cache.prefix is not None) == together and stream.st.B == B
        seen = [stream.logits().clone()]
        for t in range(4):
            stream.step(feed[:, t].to(torch.int32).pin_memory())
            seen.append(stream.logits().clone())
        whole = torch.cat([full, feed], 1)
        m = torch.cat([fullm, torch.ones(B, 4, dtype=torch.int32)], 1)
        want = ref.forward(tree32, cfg, whole, m, ref.default_position_ids(m, B, total + 4, "cpu")).logits[:, total - 1:]
        for t in range(5):
            assert rel(seen[t], want[:, t]) < 3e-2, t
        got = stream.sequences().cpu()
        assert torch.equal(got[:, :total][fullm > 0], full[fullm > 0]) and stream.length == total + 5


def test_greedy_behind_a_prefix_agrees_with_the_model():
    """Every token that generate() takes is the fp32 model's best one, or within the engine's rounding of it."""
    cfg, tree32, eng = make("gqa128")
    assert eng._together(5, 1, 1) and not B200Engine.from_tree(cfg, eng_tree(cfg))._together(5, 1, 1)
    front, ids = ids_of(1, 50, 5), ids_of(6, 7, 6)
    seqs = eng.generate(ids.cuda(), None, max_length=50 + 7 + 12, prefix_ids=front.cuda(), eos_token_id=-1).cpu()
    assert torch.equal(seqs[:, :57], torch.cat([front.expand(6, 50), ids], 1))
    logits = ref.forward(tree32, cfg, seqs).logits[:, 56:-1]
    gap = logits.amax(-1) - logits.gather(-1, seqs[:, 57:, None])[..., 0]
    assert (gap <= 6e-2 * logits.abs().amax()).all()         # 3e-2 on either side
    again = eng.generate(ids.cuda(), None, max_length=50 + 7 + 12, prefix_ids=front.cuda(), eos_token_id=-1).cpu()
    assert torch.equal(seqs, again)


def test_several_sampled_answers():
    cfg, tree32, eng = make("gqa128")
    model = LLaMAForCausalLM(cfg, _do_init=False)
    kw = dict(params={"engine": eng}, max_new_tokens=8, do_sample=True, temperature=1.0, top_k=0, eos_token_id=-1, num_return_sequences=5, seed=4)
    ids = ids_of(2, 30, 7).cuda()
    a = eng.generate(ids, None, max_length=38, do_sample=True, top_k=0, eos_token_id=-1, num_return_sequences=5, seed=4)
    assert a.shape == (10, 38) and torch.equal(a[:, :30], ids.repeat_interleave(5, 0))
    assert len({tuple(r) for r in a[:5, 30:].tolist()}) > 1
    assert torch.equal(a, eng.generate(ids, None, max_length=38, do_sample=True, top_k=0, eos_token_id=-1, num_return_sequences=5, seed=4))
    with pytest.raises(ValueError):
        eng.generate(ids, None, max_length=38, num_return_sequences=0)
    with pytest.raises(ValueError):
        eng.generate(ids, None, max_length=40, prefix_ids=ids_of(1, 20, 1).cuda())
    del model, kw


@pytest.mark.parametrize("name,B,prefix", [("gqa128", 2, 0), ("gqa128", 12, 0), ("mha64", 3, 0), ("gqa128", 4, 20)])
@pytest.mark.parametrize("graph", [True, False])
def test_rules_of_every_step_are_the_definition(name, B, prefix, graph):
    """Whole-step kernel, per-op path and the path behind a prefix: what is selected from are the model's own logits under the definition, the token is their
    arg-max; a second batch with other numbers runs on the same captured step."""
    cfg, _, eng = make(name, use_cuda_graph=graph)
    mask = torch.ones(B, 8, dtype=torch.int32)
    mask[-1, :3] = 0
    kw = dict(prefix_ids=ids_of(1, prefix, 9).cuda()) if prefix else {}
    for seed in (0, 1):
        g = torch.Generator().manual_seed(seed)
        rep, freq = (1.0 + torch.rand(B, generator=g)).tolist(), torch.rand(B, generator=g).tolist()
        bias = {int(t): float(v) for t, v in zip(torch.randint(0, 1000, (5,), generator=g), torch.randn(5, generator=g))}
        keep = torch.randperm(1000, generator=g)[:300].tolist()
        rules = LogitRules(repetition_penalty=rep, frequency_penalty=freq, presence_penalty=0.4, logit_bias=bias, allowed_tokens=keep)
        ids = ids_of(B, 8, seed)
        stream = eng.begin_stream(ids.cuda(), mask.cuda(), max_length=prefix + 20, rules=rules, **kw)
        n = prefix + 8
        bits = allowed_mask(keep, 1000)[None]
        b_ids, b_val = torch.tensor([list(bias)]), torch.tensor([list(bias.values())])
        pads = (mask == 0).sum(-1).tolist()
        for t in range(n, n + 6):
            said = stream.st.sequences.cpu()
            want = oracle.rules(stream.logits().cpu(), said, pads, [t] * B, [n] * B, rep, freq, [0.4] * B, b_ids, b_val, bits)
            got = stream.st.ruled.cpu().double()
            assert torch.equal(torch.isinf(got), torch.isinf(want)) and (got - want)[torch.isfinite(want)].abs().max() < 1e-4
            assert torch.equal(got.argmax(-1).to(torch.int32), said[:, t])
            stream.step()
        assert not graph or len(stream.st.graphs) == 1
    free = eng.begin_stream(ids.cuda(), mask.cuda(), max_length=prefix + 20, **kw)           # and rules do not outlive their batch
    assert free.st.rules is None


def test_sampling_under_a_mask_and_masks_that_follow_the_text():
    cfg, _, eng = make("gqa128")
    ids = ids_of(3, 6, 2).cuda()
    keep = list(range(100, 120))
    out = eng.generate(ids, None, max_length=26, do_sample=True, temperature=1.2, top_k=50, top_p=0.9, eos_token_id=-1, seed=1, rules=LogitRules(allowed_tokens=keep)).cpu()
    assert set(out[:, 6:].flatten().tolist()) <= set(keep) and len(set(out[:, 6:].flatten().tolist())) > 1
    stream = eng.begin_stream(ids, None, max_length=16, rules=LogitRules(allowed_tokens=[7], presence_penalty=1.0))
    assert stream.last_tokens().tolist() == [7, 7, 7]
    for t in (9, 500, 999):
        assert stream.step(allowed=allowed_mask([t], 1000)[None]).tolist() == [t] * 3
    with pytest.raises(ValueError):
        stream.step(allowed=allowed_mask([1], 1000)[None].expand(3, -1))
    with pytest.raises(ValueError):
        eng.begin_stream(ids, None, max_length=16).step(allowed=allowed_mask([1], 1000)[None])
    # a mask that leaves nothing: some token, and nothing else breaks
    stream = eng.begin_stream(ids, None, max_length=16, rules=LogitRules(allowed_tokens=[]))
    assert stream.step().tolist() == [0, 0, 0] and int(stream.step().max()) < 1000


def test_fed_tokens_are_what_was_said():
    cfg, _, eng = make("gqa128")
    stream = eng.begin_stream(ids_of(2, 6, 3).cuda(), None, max_length=16, rules=LogitRules(presence_penalty=1e4))
    feed = torch.tensor([11, 12], dtype=torch.int32).pin_memory()
    stream.step(feed)
    assert stream.st.ruled[0, 11] < -5e3 and stream.st.ruled[1, 12] < -5e3 and stream.st.ruled[0, 12] > -5e3
    assert stream.sequences()[:, 6].tolist() == [11, 12]


def test_engines_of_other_layers_write_the_rows_out():
    """The hybrid engine has no form with shared keys: the same tokens as from the joined rows, rules included."""
    from jax_llama_b200.config import FoliraxConfig
    from jax_llama_b200.models.hybrid_engine import HybridEngine
    att = {"heads": 4, "kv_heads": 2, "dim": 64, "vdim": 64, "scale": 0.125, "rot": {"dims": 32, "base": 10000.0}}
    eng = HybridEngine.random_init(FoliraxConfig(vocab=1024, width=256, norm={"eps": 1e-5}, logit_scale=0.5, logit_softcap=30.0, layers=[
        {"type": "gla", "mixer": {"heads": 4, "dim": 32, "vdim": 64, "tau": 16.0}, "mlp": None},
        {"type": "attention", "mixer": att, "mlp": {"kind": "dense", "ff": 512}}]), "cuda:0", seed=0)
    front, ids = ids_of(1, 12, 1).cuda(), ids_of(2, 5, 2).cuda()
    rules = LogitRules(repetition_penalty=1.3, allowed_tokens=range(0, 1024, 2))
    got = eng.generate(ids, None, max_length=30, eos_token_id=-1, prefix_ids=front, num_return_sequences=2, rules=rules)
    joined, _ = join_prefix(front, ids)
    want = eng.generate(joined.repeat_interleave(2, 0), None, max_length=30, eos_token_id=-1, rules=rules)
    assert torch.equal(got, want) and (got[:, 17:] % 2 == 0).all()


def test_text_front_end_on_the_gpu(spm_model):
    from jax_llama_b200 import LLaMA2Tokenizer
    tok = LLaMA2Tokenizer(spm_model)
    # (the head's product takes multiples of 8 features: the tokenizer's 300 tokens and four that no text has)
    cfg = LLaMAConfig(vocab_size=(len(tok) + 7) // 8 * 8, hidden_size=512, intermediate_size=768, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_sequence_length=128, initializer_range=0.05, bos_token_id=tok.bos_id, eos_token_id=tok.eos_id)
    model = LLaMAForCausalLM(cfg, _do_init=False, dtype=torch.bfloat16)
    gen = LLaMA(tree_to(ref.init_params(cfg, seed=2), dtype=torch.bfloat16, device="cuda"), model, tok)
    texts = gen.generate_from_str(["the city", "hello world is here"], max_gen_len=6, temperature=0.9, prefix="The capital of germany", num_return_sequences=3,
                                  rules=LogitRules(presence_penalty=0.5, allowed_tokens=range(len(tok))), seed=1)
    assert len(texts) == 6 and all(t.startswith("The capital of germany") for t in texts)
    tokens, mask, _ = gen.encode_prompts(["hello"])
    h = gen.stream(tokens, mask, 8, temperature=0.0, num_return_sequences=2, rules=LogitRules(logit_bias={5: 1e4}))
    assert h.last_tokens().tolist() == [5, 5] and h.step().tolist() == [5, 5]


def test_copies_of_another_length_take_their_own_keys():
    """The same captured step and caches serve prompts of other lengths and counts, with and without copies."""
    cfg, tree32, eng = make("gqa128")
    eng.share_above = eng.share_above_whole_step = 1 << 40
    for rows, n, seed in ((1, 40, 1), (2, 23, 2), (4, 31, 3), (1, 40, 4)):
        ids = ids_of(rows, n, seed)
        got = eng.generate(ids.cuda(), None, max_length=60, num_return_sequences=4 // rows, eos_token_id=-1).cpu()
        logits = ref.forward(tree32, cfg, got).logits[:, n - 1:-1]
        gap = logits.amax(-1) - logits.gather(-1, got[:, n:, None])[..., 0]
        assert torch.equal(got[:, :n], ids.repeat_interleave(4 // rows, 0)) and (gap <= 6e-2 * logits.abs().amax()).all()


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 32)])
def test_masks_on_the_device_stay_the_callers(graph, shape):
    """Batches of the same form with masks that lie on the engine's device: each chooses from its own, and no mask is written over."""
    cfg, _, eng = make("gqa128", use_cuda_graph=graph)
    sets = [set(range(100, 120)), set(range(500, 520)), {7}]
    a, b, c = (allowed_mask(s, 1000).expand(shape).clone().cuda() for s in sets)
    was = [t.clone() for t in (a, b, c)]
    run = lambda m, seed: eng.generate(ids_of(3, 6, 2).cuda(), None, max_length=14, do_sample=True, top_k=0, eos_token_id=-1, seed=seed, rules=LogitRules(allowed_tokens=m))  # noqa: E731
    first = run(a, 1)
    for mask, allowed in ((b, sets[1]), (a, sets[0])):
        assert set(run(mask, 1)[:, 6:].flatten().tolist()) <= allowed
    assert torch.equal(run(a, 1), first)
    stream = eng.begin_stream(ids_of(3, 6, 2).cuda(), None, max_length=14, rules=LogitRules(allowed_tokens=b))
    assert stream.step(allowed=c.view(-1, 32)).tolist() == [7, 7, 7]
    assert all(torch.equal(t, w) for t, w in zip((a, b, c), was))


@pytest.mark.parametrize("top_k,top_p", [(0, 1.0), (50, 1.0), (0, 0.9), (49, 0.9)])
def test_a_row_without_a_token_left_takes_the_first(top_k, top_p):
    """Sampling from masks that leave nothing: token 0, as on the CPU, and the other rows as they would be."""
    from jax_llama_b200.ops import kernels as K
    cfg, _, eng = make("gqa128")
    kw = dict(max_length=10, do_sample=True, top_k=top_k, top_p=top_p, eos_token_id=-1, seed=2)
    ids = ids_of(2, 5, 1).cuda()
    assert not eng.generate(ids, None, rules=LogitRules(allowed_tokens=[]), **kw)[:, 5:].any()
    one = eng.generate(ids, None, rules=LogitRules(allowed_tokens=[[], range(400, 600)]), **kw)[:, 5:].tolist()
    assert one[0] == [0] * 5 and all(400 <= t < 600 for t in one[1])
    assert one[1] == eng.generate(ids, None, rules=LogitRules(allowed_tokens=[range(1000), range(400, 600)]), **kw)[1, 5:].tolist()
    for vocab in (1, 33, 1000, 20001, 128256):
        x = torch.full((2, vocab), -float("inf"), device="cuda")
        assert K.sample_full(x, temperature=0.7, top_k=top_k, top_p=top_p, seed=5).tolist() == [0, 0]


@pytest.mark.parametrize("groups,pads,S,repeat", [(1, [9, 0, 4], 9, 1), (2, [0, 5, 5, 2], 5, 2), (1, [1, 0, 1, 1, 0], 1, 1), (2, [3, 3, 3, 3], 3, 1), (2, [0] * 4, 0, 3), (1, [0], 0, 6)])
@pytest.mark.parametrize("name", list(CFGS))
def test_prompts_without_a_token_of_their_own(name, groups, pads, S, repeat):
    """Rows that are their prefix alone, among others or all of them: the prefix is still held once, and logits and tokens are those of the joined rows."""
    cfg, tree32, eng = make(name)
    rows, P = len(pads), 70
    front, fmask, ids, mask = ids_of(groups, P, 1), padded([(3 * g) % 5 for g in range(groups)], P), ids_of(rows, S, 2), padded(pads, S)
    joined, jmask = (t.repeat_interleave(repeat, 0) for t in join_prefix(front, ids, fmask, mask, 0))
    B, total = joined.shape
    feed, rules = ids_of(B, 4, 3), LogitRules(presence_penalty=0.5)
    for _ in range(2):
        stream = eng.begin_stream(ids.cuda(), mask.cuda(), max_length=total + 6, num_return_sequences=repeat, prefix_ids=front.cuda(), prefix_mask=fmask.cuda(), rules=rules)
        assert stream.cache.prefix is not None and stream.st.B == B
        seen = [stream.logits().clone()]
        for t in range(4):
            stream.step(feed[:, t].to(torch.int32).pin_memory())
            seen.append(stream.logits().clone())
        whole, m = torch.cat([joined, feed], 1), torch.cat([jmask, torch.ones(B, 4, dtype=torch.int32)], 1)
        want = ref.forward(tree32, cfg, whole, m, ref.default_position_ids(m, B, total + 4, "cpu")).logits[:, total - 1:]
        for t in range(5):
            assert rel(seen[t], want[:, t]) < 3e-2, t
        got = stream.sequences().cpu()
        assert torch.equal(got[:, :total][jmask > 0], joined[jmask > 0]) and torch.equal(got[:, total:total + 4], feed)
    seqs = eng.generate(ids.cuda(), mask.cuda(), max_length=total + 6, num_return_sequences=repeat, prefix_ids=front.cuda(), prefix_mask=fmask.cuda(), eos_token_id=-1).cpu()
    m = torch.cat([jmask, torch.ones(B, 6, dtype=torch.int32)], 1)
    logits = ref.forward(tree32, cfg, seqs, m, ref.default_position_ids(m, B, total + 6, "cpu")).logits[:, total - 1:-1]
    assert (logits.amax(-1) - logits.gather(-1, seqs[:, total:, None])[..., 0] <= 6e-2 * logits.abs().amax()).all()


@pytest.mark.parametrize("rules", [None, LogitRules(presence_penalty=0.1)])
def test_sequences_of_a_fed_stream(rules):
    """With rules the fed tokens, which are their history; without them the selected ones, as the documentation says."""
    cfg, _, eng = make("gqa128")
    stream = eng.begin_stream(ids_of(2, 6, 3).cuda(), None, max_length=16, rules=rules)
    chosen = [stream.last_tokens().clone()]
    feed = ids_of(2, 4, 9).to(torch.int32)
    for t in range(4):
        chosen.append(stream.step(feed[:, t].contiguous().pin_memory()).clone())
    said = torch.stack(chosen, 1) if rules is None else torch.cat([feed, chosen[-1][:, None]], 1)
    assert torch.equal(stream.sequences()[:, 6:].cpu(), said.long())
