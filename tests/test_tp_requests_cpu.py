"""Rules, several answers and prefixes under tensor parallelism: the engine's host side on two ranks (gloo), with a model that is a table of next-token logits, whose
shards of the vocabulary each rank holds.  The kernels are stood in for; what is checked is what the ranks launch, hold and choose."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from jax_llama_b200 import LLaMAConfig, LogitRules, allowed_mask
from jax_llama_b200.models.engine import B200Engine, DecodeState, SharedPrefix
from jax_llama_b200.models.reference import ModelOutput, join_prefix

from . import prefix_oracle as oracle

V = 96
CFG = LLaMAConfig(vocab_size=V, hidden_size=512, intermediate_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=4, max_sequence_length=64)


class Comm:
    group = None
    begin_sequence = end_sequence = nvls_end_forward = lambda self: None


class Engine(B200Engine):
    def __init__(self, table, tp, rank):
        self.config, self.tp, self.rank, self.comm, self.device = CFG, tp, rank, Comm(), torch.device("cpu")
        self.nh, self.nkv, self.hd, self.v_local = 8 // tp, 4 // tp, 64, V // tp
        self.mine = table[:, rank * self.v_local:(rank + 1) * self.v_local]
        self._decode_states, self.steps, self.gathered = {}, 0, 0

    def _mega_fits(self, batch):                                             # a step without rules would take the whole-step kernel
        return True

    def _make_room(self, *shared):
        pass

    def _decode_state(self, B, max_len, shared=()):
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)                  # noqa: E731
        none = torch.empty(0)
        return self._decode_states.setdefault((B, max_len, *shared), DecodeState(
            B=B, max_len=max_len, ids=i32(B), x=none, qkv=none, attn=none, mlp=none, logits=torch.zeros(B, self.v_local), tok=i32(B), finished=i32(B),
            sequences=i32(B, max_len), cur_len=i32(1), step=i32(1), n_unfinished=i32(1), splits=1, scratch=None))

    def forward(self, input_ids, attention_mask=None, cache=None, **kw):
        if cache.index == 0:
            cache.pad_left.copy_(self.pad_left_from_mask(attention_mask, *input_ids.shape, self.device))
        cache.set_index(cache.index + input_ids.shape[1])
        return ModelOutput(logits=self.mine[input_ids[:, -1]][:, None])

    def _embed(self, ids, out=None, cache=None, B=0, S=0):
        self.steps += 1
        return ids

    def _layers(self, x, B, S, cache, positions, ws=None):
        assert cache.prefix is None or (isinstance(cache.prefix, SharedPrefix) and cache.prefix.k.shape[2] == self.nkv)
        return ws.ids

    def _head(self, x, out=None):
        out.copy_(self.mine[x.long()])

    def _gather_logits(self, st):
        self.gathered += 1
        parts = [torch.empty_like(st.logits) for _ in range(self.tp)]
        dist.all_gather(parts, st.logits)
        return torch.cat(parts, -1)

    def _sample_full(self, st, cache, sampling, eos, pad, logits, wait_mega):
        assert logits.shape == (st.B, V) and not wait_mega
        st.tok.copy_(logits.argmax(-1))
        st.ids.copy_(st.tok)
        st.sequences[:, int(st.cur_len)] = st.tok
        st.cur_len += 1
        cache.len_dev += 1


REQUESTS = [  # prompts, tokens each, groups of prefixes, tokens of a prefix, answers, keys held once
    (3, 5, 0, 0, 1, False), (2, 6, 0, 0, 3, True), (2, 6, 0, 0, 3, False), (4, 3, 2, 7, 2, True), (4, 3, 2, 7, 1, False), (2, 0, 1, 8, 2, True)]


def tokens_of(eng, request):
    rows, S, groups, P, repeat, together = request
    eng.share_above = eng.share_above_whole_step = 0 if together else 1 << 40
    g = torch.Generator().manual_seed(rows + S)
    ids, front = torch.randint(0, V, (rows, S), generator=g), torch.randint(0, V, (groups, P), generator=g) if groups else None
    rules = LogitRules(repetition_penalty=1.4, frequency_penalty=[0.1 * r for r in range(rows)], presence_penalty=0.3, logit_bias={4: 2.0, 50: -1.0},
                       allowed_tokens=range(1, V, 2))
    B, total = rows * repeat, S + P
    st, cache, n = eng._begin(ids, None, total + 8, 0, rules, repeat, front, None)
    assert (n, st.B) == (total, B) and (cache.prefix is not None) == (together and repeat * rows > max(groups, 1 if groups else rows))
    eng._select_and_advance_after_prefill(st, cache, (False,), -1, 0)
    for _ in range(7):
        eng._decode_step(st, cache, (False,), -1, 0)
    whole = ids if front is None else join_prefix(front, ids)[0]
    return whole.repeat_interleave(repeat, 0), st.sequences.clone(), rules, total


def worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    table = torch.randn(V, V, generator=torch.Generator().manual_seed(3)) * 2
    eng = Engine(table, world, rank)
    for request in REQUESTS:
        before = eng.steps, eng.gathered
        prompt, seqs, rules, n = tokens_of(eng, request)
        assert (eng.steps - before[0], eng.gathered - before[1]) == (7, 8)   # the path whose logits are gathered
        both = [torch.empty_like(seqs) for _ in range(world)]
        dist.all_gather(both, seqs)
        assert all(torch.equal(seqs, t) for t in both) and torch.equal(seqs[:, :n].long(), prompt)
        B, freq = len(seqs), [f for f in rules.frequency_penalty for _ in range(request[4])]
        for t in range(n, n + 8):
            want = oracle.rules(table[seqs[:, t - 1].long()], seqs, [0] * B, [t] * B, [n] * B, [1.4] * B, freq, [0.3] * B, torch.tensor([[4, 50]]),
                                torch.tensor([[2.0, -1.0]]), allowed_mask(range(1, V, 2), V)[None])
            assert torch.equal(want.argmax(-1).to(torch.int32), seqs[:, t])
    out[rank] = True
    dist.destroy_process_group()


def test_two_ranks_choose_alike_and_by_the_definition():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = mp.Manager().dict()
    mp.spawn(worker, args=(2, port, out), nprocs=2, join=True)
    assert dict(out) == {0: True, 1: True}
