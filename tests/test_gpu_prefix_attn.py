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
    (12, 1, 8, 4, 128, 1500, 700, 650, True),    # 24 queries of a key head, splits of both kinds
    (30, 3, 4, 4, 64, 900, 200, 130, True),
    (8, 1, 8, 8, 64, 2000, 30, 20, True),        # up to eight queries: rows of several tokens, angles of their own
    (4, 2, 16, 4, 128, 700, 300, 250, True),
    (6, 3, 8, 2, 64, 40, 500, 480, True),
    (8, 4, 16, 4, 128, 600, 60, 50, True),
    (10, 5, 16, 16, 64, 1300, 9, 0, True),
    (75, 1, 4, 1, 64, 1000, 12, 5, True),        # 300 queries of a key head: a pair of tiles and one tile that is not full
    (100, 1, 4, 1, 128, 700, 20, 11, False),     # 400: two pairs, the last tile with 16 queries
    (66, 2, 16, 2, 128, 520, 9, 0, True),        # 264: the second pair has eight queries
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
    (2, 2, 16, 2, 64, 600, 4, 70, 80, True),         # both sets of keys in three splits, 560 queries of a key head
    (1, 1, 8, 2, 128, 2500, 0, 300, 300, False),     # in four
    (40, 1, 16, 2, 64, 1000, 7, 3, 16, True),        # the shared keys for all rows together, in splits, then the own keys
    (1, 1, 8, 2, 128, 2500, 9, 1, 12, True),         # one token
    (15, 3, 32, 32, 64, 300, 0, 3, 20, True),        # a few tokens: own keys by a warp each
    (12, 2, 16, 8, 128, 130, 70, 5, 90, True),
    (6, 1, 8, 1, 128, 2000, 100, 2, 102, False),
    (40, 4, 32, 8, 128, 300, 0, 7, 20, True),        # more tiles than SMs, two to an SM: one launch
    (20, 2, 8, 8, 64, 500, 30, 100, 140, True),
    (24, 1, 16, 8, 128, 3000, 3, 40, 50, False),     # and the own keys behind the shared ones
    (60, 1, 32, 4, 64, 1500, 0, 12, 12, True),
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
    assert torch.equal(got, K.prefill_attn_prefix(q.to(DEV), pk, pv, kc, vc, start, S, i32(c["pad"]) if ragged else None, i32(c["plen"]) if ragged else None,
                                                  i32(c["ppad"]) if ragged else None))          # sums in a fixed order
    some = torch.arange(0, S, max(1, S // 24)).tolist() + [S - 1]            # queries that the slow oracle answers
    want, mag = oracle.attention(q[:, some].double(), c["pk"], c["pv"], c["kc"], c["vc"], [start + i for i in some], c["pad"], c["plen"], c["ppad"])
    out = got.cpu().double().view(B, S, nh, hd)
    assert torch.isfinite(out).all()
    err = (out[:, some] - want).abs()
    assert (err <= bound(want, mag)).all(), float((err / bound(want, mag)).max())
    for b in range(B):                                                       # padding: exact zeros
        assert (out[b, :max(0, c["pad"][b] - start)] == 0).all()


def small(dev, B=3, groups=1, nh=4, nkv=2, hd=64, P=90, T=20, seed=3):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    cos, sin = oracle.tables(hd, P + T + 1)
    return dict(qkv=rnd(B, (nh + 2 * nkv) * hd), pk=rnd(groups, nkv, P, hd), pv=rnd(groups, nkv, P, hd), kc=rnd(B, nkv, T, hd), vc=rnd(B, nkv, T, hd), cos=cos.to(dev), sin=sin.to(dev),
                cache_len=i([7]), pad_left=i([2] * B), prefix_len=i([P - 3] * groups), prefix_pad=i([1] * groups), nh=nh, nkv=nkv, hd=hd)


def call(c, **kw):
    c = dict(c, **kw)
    return K.decode_attn_prefix(c["qkv"], c["pk"], c["pv"], c["kc"], c["vc"], c["cos"], c["sin"], c["cache_len"], c["pad_left"], c["prefix_len"], c["prefix_pad"],
                                c["nh"], c["nkv"], c["hd"], scratch=c.get("scratch"))


def agree(got, want):
    """Two results of the same sum, each within the bound of their definition: 2 (2^-8 |out| + 2^-7 mean |v|), with mean |v| below 5 for values of a normal draw."""
    assert ((got.cpu().float() - want.float()).abs() <= 2 * (2 ** -8 * want.float().abs() + 2 ** -7 * 5)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("full", [20, 25])
def test_full_cache_stores_nothing(full):
    """From slot T on the new token sees every key and itself, and the cache stays as it is."""
    c, d = small("cpu"), small(DEV)
    kc, vc = d["kc"].clone(), d["vc"].clone()
    got = call(d, cache_len=i32([full]))
    assert torch.equal(d["kc"], kc) and torch.equal(d["vc"], vc)
    agree(got, call(c, cache_len=torch.tensor([full], dtype=torch.int32)))


@pytest.mark.gpu
def test_row_bounds_outside_the_caches():
    """Bounds that no cache has are taken as the nearest that it has: the calls of the two sides agree, and nothing outside is touched."""
    for kw in (dict(pad_left=[50, 0, 7]), dict(prefix_len=[500]), dict(prefix_pad=[80]), dict(prefix_len=[0]), dict(prefix_len=[5], prefix_pad=[9])):
        c, d = small("cpu"), small(DEV)
        host = {k: torch.tensor(v, dtype=torch.int32) for k, v in kw.items()}
        agree(call(d, **{k: v.to(DEV) for k, v in host.items()}), call(c, **host))
    d = small(DEV)
    assert torch.isfinite(call(d, cache_len=i32([-4])).float()).all()        # slot 0


@pytest.mark.gpu
def test_a_nan_reaches_the_rows_that_see_it():
    d = small(DEV, B=4, groups=2)
    d["pk"][1, 0, 40, 3] = NAN
    out = torch.isnan(call(d).float()).view(2, 2, 2, 2, 64)                  # [group, row, key head, query head, :]
    assert out[1, :, 0].all() and not out[0].any() and not out[1, :, 1].any()
    d = small(DEV)
    d["vc"][1, 1, 4, 9] = NAN
    out = torch.isnan(call(d).float()).view(3, 2, 2, 64)
    assert out[1, 1, :, 9].all() and int(out.sum()) == 2


@pytest.mark.gpu
def test_graphs_on_two_streams():
    """Two captured steps with workspaces of their own, replayed at the same time on streams of their own, and again after the token count moved on."""
    made, want = [], []
    for seed in (3, 4):
        d = small(DEV, B=40, T=300, seed=seed)
        d["cache_len"].fill_(200)
        d["scratch"] = K.prefix_attn_scratch(40, 1, 1, 4, 2, 64, 90, torch.device(DEV))
        want.append([call(dict(d, kc=d["kc"].clone(), vc=d["vc"].clone()), cache_len=i32([n])).clone() for n in (200, 260)])
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=s):
            out = call(d)
        made.append((d, g, s, out))
    torch.cuda.synchronize()
    for at, n in enumerate((200, 260)):
        for d, *_ in made:
            d["cache_len"].fill_(n)
        torch.cuda.synchronize()
        for _ in range(3):
            for _, g, s, _ in made:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        if at == 0:
            for (_, _, _, out), w in zip(made, want):
                assert torch.equal(out, w[0])
        else:                                                                # slot 200 holds the first step's token now
            for d, _, _, out in made:
                assert torch.equal(out, call(dict(d, kc=d["kc"].clone(), vc=d["vc"].clone())))


@pytest.mark.gpu
def test_workspaces_and_devices_are_refused(monkeypatch):
    d = small(DEV)
    need = K.prefix_attn_scratch(3, 1, 1, 4, 2, 64, 90, torch.device(DEV))
    with pytest.raises(Exception, match="scratch"):
        call(d, scratch=need[:need.numel() // 2])
    with pytest.raises(Exception, match="16-byte"):
        call(d, scratch=torch.empty(need.numel() + 8, device=DEV)[1:])
    with pytest.raises(ValueError):
        K.prefix_attn_scratch(3, 1, 2, 4, 2, 64, 90, torch.device(DEV))
    monkeypatch.setattr(K, "_get_device", lambda: 1)
    for f in (lambda: call(d), lambda: K.constrain_logits(torch.zeros(1, 8, device=DEV))):
        with pytest.raises(ValueError, match="current device"):
            f()


@pytest.mark.gpu
def test_no_rows_and_no_tokens():
    d = small(DEV)
    none = dict(d, qkv=d["qkv"][:0], kc=d["kc"][:0].contiguous(), vc=d["vc"][:0].contiguous(), pad_left=None)
    assert call(none).shape == (0, 256)
    q = torch.empty(3, 0, 4, 64, dtype=torch.bfloat16, device=DEV)
    assert K.prefill_attn_prefix(q, d["pk"], d["pv"], d["kc"], d["vc"], 0, 0, None, None, None).shape == (3, 0, 256)


@pytest.mark.gpu
def test_another_stream_than_the_tensors_own():
    """Work queued on a stream of its own behind the copies that fill its inputs."""
    d = small(DEV, B=40, T=300)
    want = call(dict(d, kc=d["kc"].clone(), vc=d["vc"].clone()))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in d.items()}
        late["qkv"].zero_()
        late["qkv"].copy_(d["qkv"])
        got = call(late)
        q = torch.randn(40, 6, 4, 64, device=DEV).to(torch.bfloat16)
        one = K.prefill_attn_prefix(q, d["pk"], d["pv"], d["kc"], d["vc"], 3, 6, d["pad_left"], None, None)
    s.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(one, K.prefill_attn_prefix(q, d["pk"], d["pv"], d["kc"], d["vc"], 3, 6, d["pad_left"], None, None))


@pytest.mark.parametrize("dev", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("count", [-4, -1, -1000])
def test_a_negative_count_is_slot_0(count, dev):
    """On either side: the result and both caches are those of a call at slot 0."""
    c, d = small(dev), small(dev)
    got, want = (call(t, cache_len=torch.tensor([n], dtype=torch.int32, device=dev)) for t, n in ((c, count), (d, 0)))
    assert torch.equal(got, want) and torch.equal(c["kc"], d["kc"]) and torch.equal(c["vc"], d["vc"])
