"""Attention of rows whose group shares keys: the one-token and the prompt form against the definition in 64 bits."""
import pytest
import torch

from jax_llama_b200.ops import kernels as K

from . import prefix_oracle as oracle

DEV = "cuda"
NAN = float("nan")


def bound(want, mag):
    """The result is rounded once (2^-8 of it), every weight once (2^-8 of the weight: 2^-8 of the sum of weights times |values|); scores are off by the
    query's second rounding (2^-16) and the sums' last bits, at |q| |k| / sqrt(d) <= 16 below 2^-11 of a weight with its share of the sum."""
    return 2 ** -8 * want.abs() + (2 ** -8 + 2 ** -10) * mag + 1e-30


def case(B, groups, nh, nkv, hd, P, T, ragged, seed, own):
    """Random caches whose unused slots hold NaN; `own`: the most own keys in front of this call's."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)
    draw = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=g).tolist()
    c = dict(pk=rnd(groups, nkv, P, hd), pv=rnd(groups, nkv, P, hd), kc=rnd(B, nkv, T, hd), vc=rnd(B, nkv, T, hd), rnd=rnd)
    if ragged:
        c["plen"] = draw(0, P, groups)
        c["plen"][0] = P
        c["ppad"] = [draw(0, n, 1)[0] for n in c["plen"]]
        c["pad"] = draw(0, own, B)
    else:
        c["plen"], c["ppad"], c["pad"] = [P] * groups, [0] * groups, [0] * B
    return c


def dirty(c, used):
    """NaN wherever no key is: outside the groups' shared keys, in front of the rows' pads and from slot `used` on."""
    pk, pv, kc, vc = (c[n].clone() for n in ("pk", "pv", "kc", "vc"))
    for g in range(pk.shape[0]):
        for t in (pk, pv):
            t[g, :, :c["ppad"][g]] = NAN
            t[g, :, c["plen"][g]:] = NAN
    for b in range(kc.shape[0]):
        for t in (kc, vc):
            t[b, :, :c["pad"][b]] = NAN
            t[b, :, used:] = NAN
    return [t.to(DEV) for t in (pk, pv, kc, vc)]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


STEPS = [  # rows, groups, nh, nkv, hd, P, T, own keys, ragged
    (1, 1, 4, 1, 128, 1, 1, 0, False),           # one row, one shared key, the new token alone
    (2, 1, 8, 8, 64, 64, 8, 3, False),           # a whole tile
    (2, 2, 8, 2, 128, 65, 70, 69, True),         # a tile and one key; the last slot
    (6, 2, 8, 1, 64, 200, 90, 40, True),         # eight query heads
    (5, 5, 4, 2, 128, 130, 65, 64, True),        # a group each
    (34, 1, 4, 1, 64, 150, 33, 17, True),        # 136 queries of a key head: two tiles
    (70, 2, 8, 4, 128, 300, 20, 5, True),
    (3, 1, 4, 4, 128, 1500, 700, 650, True),     # splits of both kinds
    (2, 1, 2, 1, 64, 3000, 1400, 1300, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,groups,nh,nkv,hd,P,T,own,ragged", STEPS)
def test_one_token(B, groups, nh, nkv, hd, P, T, own, ragged):
    c = case(B, groups, nh, nkv, hd, P, T, ragged, B + P, own)
    qkv = c["rnd"](B, (nh + 2 * nkv) * hd)
    cos, sin = oracle.tables(hd, P + T + 1)
    x = qkv.double().view(B, nh + 2 * nkv, hd)
    turned = torch.stack([oracle.rotate(x[b, :nh + nkv], c["plen"][b // (B // groups)] - c["ppad"][b // (B // groups)] + own - c["pad"][b]) for b in range(B)])
    pk, pv, kc, vc = dirty(c, own)
    before = kc.clone(), vc.clone()
    scratch = K.prefix_attn_scratch(B, 1, groups, nh, nkv, hd, P, torch.device(DEV))
    scratch.fill_(NAN)                                                       # a workspace may hold anything
    args = (pk, pv, kc, vc, cos.to(DEV), sin.to(DEV), i32([own]), i32(c["pad"]) if ragged else None, i32(c["plen"]) if ragged else None,
            i32(c["ppad"]) if ragged else None, nh, nkv, hd)
    got = K.decode_attn_prefix(qkv.to(DEV), *args, scratch=scratch)
    again = K.decode_attn_prefix(qkv.to(DEV), *args, scratch=scratch)
    assert torch.equal(got, again)                                           # sums in a fixed order
    # the cache: one slot, the rotated key rounded once from fp32 (an fp32 rotation may fall on the other side of a tie)
    keep = torch.arange(T, device=DEV) != own
    for now, was in zip((kc, vc), before):
        assert torch.equal(now[:, :, keep].view(torch.int16), was[:, :, keep].view(torch.int16))
    assert torch.equal(vc[:, :, own].cpu(), qkv.view(B, nh + 2 * nkv, hd)[:, nh + nkv:])
    kn = kc[:, :, own].cpu().double()
    assert ((kn - turned[:, nh:]).abs() <= 2 ** -8 * turned[:, nh:].abs() + 2 ** -20).all()
    c["kc"][:, :, own], c["vc"][:, :, own] = kc[:, :, own].cpu(), vc[:, :, own].cpu()
    want, mag = oracle.attention(turned[:, None, :nh], c["pk"], c["pv"], c["kc"], c["vc"], [own], c["pad"], c["plen"], c["ppad"])
    err = (got.cpu().double().view_as(want) - want).abs()
    assert torch.isfinite(err).all() and (err <= bound(want, mag)).all(), float((err / bound(want, mag)).max())


PROMPTS = [  # rows, groups, nh, nkv, hd, P, start, S, T, ragged
    (1, 1, 4, 1, 128, 1, 0, 1, 1, False),
    (2, 1, 8, 8, 64, 64, 0, 64, 64, False),
    (2, 2, 8, 2, 128, 70, 5, 33, 40, True),
    (4, 2, 8, 1, 64, 200, 0, 17, 80, True),
    (3, 3, 4, 2, 128, 130, 60, 70, 130, True),
    (5, 1, 4, 1, 128, 900, 3, 40, 64, True),
    (4, 1, 32, 32, 64, 100, 0, 130, 130, True),      # one key head per query head: a row's queries fill two tiles, 256 of them
    (2, 1, 32, 32, 128, 200, 11, 256, 300, False),   # whole tiles, enough of them: one launch over both sets of keys
    (3, 3, 32, 32, 64, 70, 2, 256, 258, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,groups,nh,nkv,hd,P,start,S,T,ragged", PROMPTS)
def test_prompt(B, groups, nh, nkv, hd, P, start, S, T, ragged):
    c = case(B, groups, nh, nkv, hd, P, T, ragged, B + S, start + S - 1)
    if ragged:
        c["pad"][-1] = start + S                                             # a row of padding alone
    q = c["rnd"](B, S, nh, hd)
    pk, pv, kc, vc = dirty(c, start + S)
    got = K.prefill_attn_prefix(q.to(DEV), pk, pv, kc, vc, start, S, i32(c["pad"]) if ragged else None, i32(c["plen"]) if ragged else None,
                                i32(c["ppad"]) if ragged else None)
    some = torch.arange(0, S, max(1, S // 24)).tolist() + [S - 1]            # queries that the slow oracle answers
    want, mag = oracle.attention(q[:, some].double(), c["pk"], c["pv"], c["kc"], c["vc"], [start + i for i in some], c["pad"], c["plen"], c["ppad"])
    out = got.cpu().double().view(B, S, nh, hd)
    assert torch.isfinite(out).all()
    err = (out[:, some] - want).abs()
    assert (err <= bound(want, mag)).all(), float((err / bound(want, mag)).max())
    for b in range(B):                                                       # padding: exact zeros
        assert (out[b, :max(0, c["pad"][b] - start)] == 0).all()
