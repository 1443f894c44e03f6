"""What the engine keeps between batches behind shared prefixes: caches and captured steps that serve many lengths, a bounded number of them."""
from types import SimpleNamespace

import pytest
import torch

from jax_llama_b200 import LLaMAConfig
from jax_llama_b200.models import reference as ref
from jax_llama_b200.models.engine import B200Engine
from jax_llama_b200.models.llama import tree_to


def test_slots_serve_every_length_of_their_step():
    few = set()
    for P in range(1, 20000):
        slots, least = B200Engine._shared_slots(P)
        assert least <= P <= slots and (slots - least < 64 or slots - least < P / 8)
        assert B200Engine._shared_slots(slots) == B200Engine._shared_slots(least) == (slots, least)
        few.add(slots)
    assert len(few) < 60
    own = lambda max_len, P: B200Engine._own_slots(B200Engine, max_len, B200Engine._shared_slots(P)[0])      # noqa: E731
    for P in (1, 64, 65, 1023, 1025, 4097, 8192):
        for more in (0, 1, 500):
            assert own(P + more, P) >= max(more, 1)


def test_room_is_made_by_the_longest_unused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda dev: SimpleNamespace(total_memory=8100 * 4 * 64))
    eng = SimpleNamespace(config=SimpleNamespace(num_hidden_layers=1), nkv=1, hd=64, device=None, kept_shared=3, kept_shared_part=1.0, _decode_states={},
                          _own_slots=lambda max_len, slots: max_len - slots)
    take = lambda *key: (B200Engine._make_room(eng, *key), eng._decode_states.__setitem__(key, 0))               # noqa: E731
    eng._decode_states[(2, 100)] = 0                                          # a batch without prefixes stays
    for n in range(6):
        take(2, 1000 + n, 1, 500)
    assert list(eng._decode_states) == [(2, 100), *((2, 1000 + n, 1, 500) for n in (3, 4, 5))]
    take(8, 900, 1, 100)                                                      # 6500 slots of 8100: one more, of 1510, finds room
    assert list(eng._decode_states) == [(2, 100), (2, 1005, 1, 500), (8, 900, 1, 100)]
    take(80, 900, 1, 100)                                                     # more than there is room for: itself alone
    assert list(eng._decode_states) == [(2, 100), (80, 900, 1, 100)]


CFG = LLaMAConfig(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, max_sequence_length=512,
                  initializer_range=0.05)


def make():
    tree = tree_to(ref.init_params(CFG, seed=1), dtype=torch.bfloat16)
    eng = B200Engine.from_tree(CFG, tree_to(tree, device="cuda"))
    eng.share_above = eng.share_above_whole_step = 0
    return eng, tree_to(tree, dtype=torch.float32)


def ids_of(rows, n, seed):
    return torch.randint(3, 1000, (rows, n), generator=torch.Generator().manual_seed(seed))


def near_best(tree32, seqs, n):
    """Every token from place n on is the fp32 model's best, or within both sides' rounding of it."""
    logits = ref.forward(tree32, CFG, seqs).logits[:, n - 1:-1]
    gap = logits.amax(-1) - logits.gather(-1, seqs[:, n:, None])[..., 0]
    return bool((gap <= 6e-2 * logits.abs().amax()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("together", [True, False])
def test_many_prompt_lengths_hold_a_few_states(together):
    """Six answers each to prompts of 40 lengths under one max_length: what is held stops growing, every batch is the model's, and a batch after longer ones does not see
    their keys."""
    eng, tree32 = make()
    if not together:
        eng.share_above = eng.share_above_whole_step = 1 << 40
    held, lengths = [], [70, 128, 65, 300, 299, 310, 72, *range(400, 433)]
    for i, P in enumerate(lengths):
        ids = ids_of(1, P, i)
        got = eng.generate(ids.cuda(), None, max_length=440, num_return_sequences=6, eos_token_id=-1).cpu()
        assert torch.equal(got[:, :P], ids.expand(6, P))
        if i < 8 or i % 8 == 0:
            assert near_best(tree32, got[:2, :P + 8], P)
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated())
    assert max(held[20:]) <= max(held[:10])
    assert len(eng._decode_states) <= eng.kept_shared
    assert together or all(getattr(st, "_front_cache", None) is None for st in eng._decode_states.values())


@pytest.mark.gpu
def test_lengths_of_one_step_share_a_captured_step():
    eng, _ = make()
    for P in (70, 100, 128):
        eng.generate(ids_of(1, P, P).cuda(), None, max_length=200, num_return_sequences=6, eos_token_id=-1)
    (st,) = eng._decode_states.values()
    assert len(st.graphs) == 1 and st._front_cache.capacity == 128 and st._cache.capacity == 200 - 65


@pytest.mark.gpu
def test_streams_at_work_keep_their_state():
    """Streams behind prefixes of other lengths of the same step, and as many other states as it takes to push theirs out."""
    eng, tree32 = make()
    run = lambda P: eng.begin_stream(ids_of(1, P, P).cuda(), None, max_length=200, num_return_sequences=6, eos_token_id=-1)      # noqa: E731
    streams = [run(P) for P in (70, 90)]
    assert streams[0].st is not streams[1].st
    for P in (130, 5, 180, 20, 150, 90, 88):
        eng.generate(ids_of(1, P, P).cuda(), None, max_length=220, num_return_sequences=6, eos_token_id=-1)
    for _ in range(10):
        for s in streams:
            s.step()
    for P, s in zip((70, 90), streams):
        got = s.sequences().cpu()
        assert torch.equal(got[:, :P], ids_of(1, P, P).expand(6, P)) and got.shape[1] == P + 11 and near_best(tree32, got[:2], P)
        s.close()
