"""What attention over shared keys keeps beyond the 8 bits of one bfloat16 number: queries and probabilities of a step are two of them, at any count of rows, and so are the
probabilities of prompts with up to 128 queries of a key head."""
import math

import pytest
import torch

from jax_llama_b200.ops import kernels as K

from . import prefix_oracle as oracle

DEV = "cuda"

STEPS = [  # rows, groups, nh, nkv, hd
    (8, 1, 8, 8, 128), (10, 5, 32, 8, 64),                               # up to eight queries of a (group, key head)
    (16, 1, 32, 8, 128), (60, 2, 16, 4, 64), (32, 1, 32, 8, 128),        # up to 128
    (33, 1, 32, 8, 128), (33, 1, 32, 8, 64), (140, 2, 16, 4, 128), (200, 1, 8, 8, 64),       # more
]


def case(B, groups, nh, nkv, hd, size, seed):
    """Two shared keys of opposite values and a new token without key or value: out = (w1 - w2) v, small where the two scores are alike, while an error of either weight shows
    whole.  `size`: of the queries."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)      # noqa: E731
    qkv = torch.cat([rnd(B, nh * hd) * size, torch.zeros(B, 2 * nkv * hd, dtype=torch.bfloat16)], 1)
    v = rnd(groups, nkv, 1, hd)
    return qkv, rnd(groups, nkv, 2, hd), torch.cat([v, -v], 2)


def weights(c, B, groups, nh, nkv, hd, round_q=None, round_p=None):
    """fp64: (out, sum of weights times |values|, largest sum of |q k| / sqrt(d)) of the step at position 2, the queries and weights rounded where asked."""
    qkv, pk, pv = c
    q = oracle.rotate(qkv[:, :nh * hd].double().view(B, nh, hd), 2)
    q = (q if round_q is None else round_q(q)).view(groups, B // groups, nkv, nh // nkv, hd)
    k, v = (torch.cat([t.double(), torch.zeros(groups, nkv, 1, hd)], 2) for t in (pk, pv))
    s = torch.einsum("gbnhd,gnkd->gbnhk", q, k) / math.sqrt(hd)
    size = torch.einsum("gbnhd,gnkd->gbnhk", q.abs(), k.abs()) / math.sqrt(hd)
    p = (s - s.amax(-1, keepdim=True)).exp()
    total = p.sum(-1, keepdim=True)
    if round_p is not None:
        p = round_p(p)
    out, mag = (torch.einsum("gbnhk,gnkd->gbnhd", p / total, x).reshape(B, nh, hd) for x in (v, v.abs()))
    return out, mag, size.amax(-1).reshape(B, nh, 1)


def bound(out, mag, size):
    """The result is rounded once, 2^-8 of it.  A weight has 16 bits (2^-16) and the error of its score twice, its own and the sum's: of a query in two numbers 2^-16 of
    sum |q k| / sqrt(d), and as much for a rotation and a sum in fp32 (four roundings of 2^-24 and hd of them: 2^-17), in nats: 3 2^-16.  2^-18 for what is left: the
    exponential, the division and the sums of three values."""
    return 2 ** -8 * out.abs() + (2 ** -16 + 2 ** -18 + 3 * 2 ** -16 * size) * mag + 1e-30


def one(t):
    return t.to(torch.bfloat16).double()


def two(t):
    return one(t) + one(t - one(t))


@pytest.mark.parametrize("B,groups,nh,nkv,hd", STEPS)
def test_the_bound_sees_a_rounding_to_one_number(B, groups, nh, nkv, hd):
    """The mistakes that the test below is for, made in the definition."""
    for size, mistake in ((0.25, dict(round_p=one)), (2.0, dict(round_q=one))):
        c, at = case(B, groups, nh, nkv, hd, size, B + hd), (B, groups, nh, nkv, hd)
        want, mag, s = weights(c, *at)
        for kw, seen in ((dict(round_p=two, round_q=two), False), (mistake, True)):
            err = (one(weights(c, *at, **kw)[0]) - want).abs()
            assert bool((err > bound(want, mag, s)).any()) == seen


@pytest.mark.gpu
@pytest.mark.parametrize("size", [0.25, 2.0])
@pytest.mark.parametrize("B,groups,nh,nkv,hd", STEPS)
def test_a_step_has_sixteen_bits(B, groups, nh, nkv, hd, size):
    qkv, pk, pv = c = case(B, groups, nh, nkv, hd, size, B + hd)
    want, mag, s = weights(c, B, groups, nh, nkv, hd)
    cos, sin = oracle.tables(hd, 8)
    kc = torch.zeros(B, nkv, 4, hd, dtype=torch.bfloat16, device=DEV)
    got = K.decode_attn_prefix(qkv.to(DEV), pk.to(DEV), pv.to(DEV), kc, kc.clone(), cos.to(DEV), sin.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV), None, None, None,
                               nh, nkv, hd)
    err = (got.cpu().double().view(B, nh, hd) - want).abs()
    assert (err <= bound(want, mag, s)).all(), float((err / bound(want, mag, s)).max())


PROMPTS = [(1, 1, 8, 8, 128, 40), (1, 1, 8, 8, 64, 128), (4, 1, 32, 8, 64, 4), (8, 2, 8, 2, 128, 3), (3, 1, 16, 2, 64, 5), (16, 1, 32, 4, 128, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("B,groups,nh,nkv,hd,S", PROMPTS)
def test_a_prompt_of_one_tile_has_sixteen_bits(B, groups, nh, nkv, hd, S):
    """The same two keys in front of tokens without key or value; queries come rotated, in one number each."""
    qkv, pk, pv = case(B * S, groups, nh, nkv, hd, 0.25, B + S)
    q = qkv[:, :nh * hd].view(B, S, nh, hd)
    kc = torch.zeros(B, nkv, S, hd, dtype=torch.bfloat16, device=DEV)
    got = K.prefill_attn_prefix(q.to(DEV), pk.to(DEV), pv.to(DEV), kc, kc.clone(), 0, S, None, None, None).cpu().double().view(B, S, nh, hd)
    head, row = torch.arange(nh) // (nh // nkv), torch.arange(B) // (B // groups)
    k, v = (t.double()[row][:, head] for t in (pk, pv))                      # [B, nh, 2, hd]
    s = torch.einsum("bshd,bhkd->bshk", q.double(), k) / math.sqrt(hd)
    size = (torch.einsum("bshd,bhkd->bshk", q.double().abs(), k.abs()) / math.sqrt(hd)).amax(-1, keepdim=True)
    own = torch.zeros(B, S, nh, 1, dtype=torch.float64) + torch.log(torch.arange(1.0, S + 1, dtype=torch.float64))[:, None, None]      # s + 1 keys of score 0
    w = torch.softmax(torch.cat([s, own], -1), -1)[..., :2]
    want, mag = torch.einsum("bshk,bhkd->bshd", w, v), torch.einsum("bshk,bhkd->bshd", w, v.abs())
    err, most = (got - want).abs(), bound(want, mag, size)
    assert (err <= most).all(), float((err / most).max())
    one_number = one(torch.einsum("bshk,bhkd->bshd", one(w / w.amax(-1, keepdim=True)) * w.amax(-1, keepdim=True), v))
    assert ((one_number - want).abs() > most).any()                          # (what the bound is for)
