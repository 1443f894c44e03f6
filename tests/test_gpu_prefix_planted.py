"""Attention over shared keys, every slot in its turn: queries that lean on two keys each, so that a key that is left out or counted twice shows in the result."""
import math

import pytest
import torch

from jax_llama_b200.ops import kernels as K

from . import prefix_oracle as oracle
from .test_gpu_prefix_attn import PROMPTS, STEPS

LEAN = 8.0                 # a query is so many times the sum of its two keys, which have norm sqrt(d): two scores of 8 sqrt(d) or more, others of 4.5 standard deviations of 8 sqrt(2)


def draw(B, groups, nkv, hd, P, T, ragged, used, seed, dev):
    """Keys of norm sqrt(hd) and values in bf16, NaN in slots that hold none, and which slots of [shared, own] a row has, [B, P + T]; `used`: own slots filled."""
    g = torch.Generator().manual_seed(seed)
    keys = lambda *s: (lambda x: (x * hd ** 0.5 / x.norm(dim=-1, keepdim=True)).to(torch.bfloat16))(torch.randn(*s, hd, generator=g))      # noqa: E731
    whole = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))      # noqa: E731
    plen = [P] + [whole(0, P) if ragged else P for _ in range(groups - 1)]
    ppad = [whole(0, n // 3) if ragged else 0 for n in plen]
    pad = [whole(0, used - 1) if ragged and used > 1 else 0 for _ in range(B)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)      # noqa: E731
    c = dict(pk=keys(groups, nkv, P), pv=keys(groups, nkv, P), kc=keys(B, nkv, T), vc=keys(B, nkv, T))
    at = torch.arange(P)
    shared = torch.stack([(at >= a) & (at < b) for a, b in zip(ppad, plen)])
    own = torch.arange(T)[None] >= torch.tensor(pad)[:, None]
    for name, keep in (("pk", shared), ("pv", shared), ("kc", own & (torch.arange(T) < used)), ("vc", own & (torch.arange(T) < used))):
        c[name] = c[name].masked_fill(~keep[:, None, :, None], math.nan).to(dev)
    c.update(plen=i32(plen), ppad=i32(ppad), pad=i32(pad), has=torch.cat([shared.repeat_interleave(B // groups, 0), own], 1).to(dev))
    return c


def joined(c, B, groups):
    """fp64 keys and values of every row, [B, nkv, P + T, hd]."""
    return [torch.cat([c[a].repeat_interleave(B // groups, 0), c[b]], 2).double() for a, b in (("pk", "kc"), ("pv", "vc"))]


def definition(q, k, v, seen, twice=None):
    """fp64 q [B, S, nh, hd] over keys [B, nkv, N, hd], seen [B, S, N] -> (out, sum of weights times |values|, largest sum of |q k| / sqrt(d)); zeros where nothing is
    seen.  `twice`: slots [N] with a second vote."""
    B, S, nh, hd = q.shape
    nkv = k.shape[1]
    k, v = (t.nan_to_num(0.0) for t in (k, v))
    q = q.view(B, S, nkv, nh // nkv, hd)
    s = torch.einsum("bsjgd,bjnd->bsjgn", q, k) / math.sqrt(hd)
    if twice is not None:
        s = s + math.log(2.0) * twice
    w = torch.softmax(s.masked_fill(~seen[:, :, None, None], -math.inf), -1).nan_to_num(0.0)
    size = (torch.einsum("bsjgd,bjnd->bsjgn", q.abs(), k.abs()) / math.sqrt(hd)).masked_fill(~seen[:, :, None, None], 0.0).amax(-1, keepdim=True)
    out, mag = (torch.einsum("bsjgn,bjnd->bsjgd", w, x).reshape(B, S, nh, hd) for x in (v, v.abs()))
    return out, mag, size.reshape(B, S, nh, 1)


def bound(out, mag, size):
    """The result is rounded once and so is a weight, 2^-8 each; a score is off by 2^-16 of sum |q k| / sqrt(d) for a query in two numbers and half of that for sums in fp32,
    and counts twice, its own weight and the sum's."""
    return 2 ** -8 * out.abs() + (2 ** -8 + 3 * 2 ** -16 * size) * mag + 1e-30


def lean(k, seen, number, g):
    """Queries [B, S, nh, hd] that lean on the `number`th key (modulo their count, [B, S, nh]) of those seen [B, S, N] and on another one."""
    B, S, nh = number.shape
    n = seen.sum(-1)[..., None].clamp(min=1)                                 # [B, S, 1]
    order = (~seen).to(torch.int8).argsort(dim=-1, stable=True)              # the seen slots first
    first = number % n
    other = (first + 1 + torch.randint(0, 1 << 30, number.shape, generator=g).to(number.device) % (n - 1).clamp(min=1)) % n
    head = torch.arange(nh, device=k.device) // (nh // k.shape[1])
    row = torch.arange(B, device=k.device)[:, None, None]
    pick = lambda i: k[row, head, torch.gather(order, 2, i.view(B, S, nh))].nan_to_num(0.0)      # noqa: E731
    return LEAN * (pick(first) + pick(other))


def off(got, want):
    err = (got.double() - want[0]).abs() / bound(*want)
    return float(err.nan_to_num(math.inf).max()) if err.numel() else 0.0


@pytest.mark.parametrize("hd", [64, 128])
def test_a_slot_lost_or_counted_twice_shows(hd):
    """The mistakes that the tests below are for, made in the definition: whatever the slot, some query of a round over all of them is off the bound."""
    B, groups, nh, nkv, P, T, used = 3, 1, 4, 2, 300, 20, 15
    c, g = draw(B, groups, nkv, hd, P, T, False, used, hd, "cpu"), torch.Generator().manual_seed(1)
    k, v = joined(c, B, groups)
    seen = (c["has"] & (torch.arange(P + T) < P + used))[:, None]
    n = (B * nh // nkv, nh // nkv)
    each = torch.arange(B)[:, None, None] * n[1] + torch.arange(nh) % n[1]
    rounds = [lean(k, seen, each + r * n[0], g) for r in range(-(-(P + used) // n[0]))]
    wants = [definition(q, k, v, seen) for q in rounds]
    assert all(off(w[0].to(torch.bfloat16), w) <= 1.0 for w in wants)
    for slot in (0, 1, 63, 64, 127, 128, 255, 256, 290, 299, P, P + 7, P + used - 1):
        without, twice = seen.clone(), torch.zeros(P + T, dtype=torch.float64)
        without[:, :, slot], twice[slot] = False, 1.0
        assert max(off(definition(q, k, v, without)[0], w) for q, w in zip(rounds, wants)) > 4.0
        assert max(off(definition(q, k, v, seen, twice)[0], w) for q, w in zip(rounds, wants)) > 4.0


@pytest.mark.gpu
@pytest.mark.parametrize("B,groups,nh,nkv,hd,P,T,own,ragged", STEPS)
def test_every_key_of_a_step(B, groups, nh, nkv, hd, P, T, own, ragged):
    dev, G = "cuda", nh // nkv
    c, g = draw(B, groups, nkv, hd, P, T, ragged, own, B + P, dev), torch.Generator().manual_seed(P)
    cos, sin = (t.to(dev) for t in oracle.tables(hd, P + T + 1))
    pos = ((c["plen"] - c["ppad"]).repeat_interleave(B // groups) + own - c["pad"]).long()
    turn = torch.complex(cos[pos].double(), sin[pos].double())[:, None]      # [B, 1, hd / 2]
    rotate = lambda x, t: torch.view_as_real(torch.view_as_complex(x.double().reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * t).reshape(x.shape)      # noqa: E731
    new = draw(B, 1, 2 * nkv, hd, 1, 1, False, 1, 7, dev)["kc"].reshape(B, -1)           # keys and values of the new token
    scratch = K.prefix_attn_scratch(B, 1, groups, nh, nkv, hd, P, torch.device(dev))
    run = lambda q: K.decode_attn_prefix(torch.cat([q.reshape(B, -1), new], 1), c["pk"], c["pv"], c["kc"], c["vc"], cos, sin,      # noqa: E731
                                         torch.tensor([own], dtype=torch.int32, device=dev), c["pad"], c["plen"], c["ppad"], nh, nkv, hd, scratch=scratch)
    run(torch.zeros(B, nh * hd, dtype=torch.bfloat16, device=dev))           # the new key as the cache holds it
    k, v = joined(c, B, groups)
    seen = (c["has"] & (torch.arange(P + T, device=dev) < P + own + 1))[:, None]
    row, head = torch.arange(B, device=dev)[:, None, None], torch.arange(nh, device=dev) % G
    many, worst = (B // groups) * G, 0.0
    shared = [row % (B // groups) * G + head + r * many for r in range(-(-(P + own + 1) // many))]
    behind = [seen.sum(-1)[..., None] - 1 - (head + r * G) % (own + 1 - c["pad"].long()[:, None, None]) for r in range(-(-(own + 1) // G))]
    for number in shared + behind:
        raw = rotate(lean(k, seen, number, g)[:, 0], turn.conj()).to(torch.bfloat16)
        worst = max(worst, off(run(raw).view(B, 1, nh, hd), definition(rotate(raw, turn)[:, None], k, v, seen)))
    assert worst <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("B,groups,nh,nkv,hd,P,start,S,T,ragged", PROMPTS)
def test_every_key_of_a_prompt(B, groups, nh, nkv, hd, P, start, S, T, ragged):
    dev, G = "cuda", nh // nkv
    c, g = draw(B, groups, nkv, hd, P, T, ragged, start + S, B + S, dev), torch.Generator().manual_seed(P)
    k, v = joined(c, B, groups)
    slot = start + torch.arange(S, device=dev)
    own = torch.arange(T, device=dev)[None] <= slot[:, None]                 # [S, T]
    seen = c["has"][:, None] & torch.cat([torch.ones(S, P, dtype=torch.bool, device=dev), own], 1)[None]
    seen = seen & (slot[None] >= c["pad"][:, None])[..., None]               # a query in front of its row's first token is padding
    row, token, head = torch.arange(B, device=dev)[:, None, None], torch.arange(S, device=dev)[:, None], torch.arange(nh, device=dev) % G
    many, worst = (B // groups) * S * G, 0.0
    last = seen[:, :, P:].sum(-1)[..., None]
    shared = [(row % (B // groups) * S + token) * G + head + r * many for r in range(-(-(P + start + S) // many))]
    behind = [seen.sum(-1)[..., None] - 1 - ((token + r * S) * G + head) % last.clamp(min=1) for r in range(-(-2 * (start + S) // (S * G)))]
    for number in shared + behind:
        q = lean(k, seen, number.expand(B, S, nh), g).to(torch.bfloat16)
        got = K.prefill_attn_prefix(q, c["pk"], c["pv"], c["kc"], c["vc"], start, S, c["pad"], c["plen"], c["ppad"])
        worst = max(worst, off(got.view(B, S, nh, hd), definition(q.double(), k, v, seen)))
    assert worst <= 1.0
