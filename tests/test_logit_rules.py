"""The rules of a request on its logits: penalties, biases, masks; the CPU statement and the kernel against the definition in 64 bits, and the refusals."""
import math

import pytest
import torch

from jax_llama_b200.ops import kernels as K

from . import prefix_oracle as oracle

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def mask_of(rows, V, keep, g):
    bits = torch.rand(rows, (V + 31) // 32 * 32, generator=g) < keep
    words = (bits.view(rows, -1, 32).long() << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def close(got, want, x, scale):
    """Every step rounds once in fp32 (2^-24 of its value, of the terms' sizes where they cancel); -inf where the definition has it."""
    got, want = got.double().cpu(), want.cpu()
    assert torch.equal(torch.isneginf(got), torch.isneginf(want))
    f = torch.isfinite(want)
    assert ((got - want).abs()[f] <= 6 * 2 ** -24 * scale[f] + 1e-37).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,V,T,dtype,n_bias,mask,seed", [
    (1, 1, 1, torch.float32, 1, "rows", 0), (1, 33, 5, torch.float32, 0, "none", 1), (3, 31, 64, torch.bfloat16, 4, "one", 2), (2, 4097, 200, torch.float16, 40, "rows", 3),
    (5, 8192, 33, torch.float32, 70, "one", 4), (2, 5003, 1100, torch.float32, 3, "none", 5), (4, 777, 0, torch.float32, 5, "rows", 6)])
def test_rules(B, V, T, dtype, n_bias, mask, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, V, generator=g) * 4).to(dtype)
    x[0, 0] = -math.inf
    tokens = (torch.rand(B, T, generator=g) ** 3 * V).to(torch.int32).clamp(max=V - 1)
    if T > 4:
        tokens[:, 2], tokens[:, 3] = -1, V                                   # ids outside the vocabulary
    rnd = lambda lo, hi: torch.randint(lo, hi + 1, (B,), generator=g, dtype=torch.int32)
    starts, lengths, prompts = rnd(0, T // 2), rnd(0, T + 3), rnd(0, T)      # lengths below starts and beyond the buffer among them
    rep, freq, pres = 0.7 + torch.rand(B, generator=g), torch.randn(B, generator=g), torch.randn(B, generator=g)
    ids = torch.randint(-1, V + 1, (B, n_bias), generator=g, dtype=torch.int32)
    if n_bias > 3:
        ids[:, 1:4] = ids[:, :1]                                             # the same id four times
    bias = torch.randn(B, n_bias, generator=g)
    allowed = None if mask == "none" else mask_of(B if mask == "rows" else 1, V, 0.4, g)
    if mask == "rows":
        allowed[-1] = 0                                                      # a row whose mask leaves nothing
    want = oracle.rules(x, tokens, starts.tolist(), lengths.tolist(), prompts.tolist(), rep.tolist(), freq.tolist(), pres.tolist(), ids, bias, allowed)
    scale = x.double().nan_to_num(0, 0, 0).abs() * 2 + (T * 4.0 + 4) * (tokens.numel() > 0) * freq.abs().max() + pres.abs().max() + 5.0 * bias.abs().sum() / max(B, 1)
    d = lambda t: None if t is None else t.to(dev)
    out = torch.empty(B, V + 5, device=dev)[:, :V]                           # any row pitch
    wide = torch.empty(B, V + 3, dtype=dtype, device=dev)[:, :V]
    wide.copy_(x)
    got = K.constrain_logits(wide, tokens=d(tokens), starts=d(starts), lengths=d(lengths), prompt_lengths=d(prompts), repetition=d(rep), frequency=d(freq),
                             presence=d(pres), bias_ids=d(ids), bias_values=d(bias), allowed=d(allowed), out=out)
    assert got is out and torch.equal(wide.cpu().view(torch.int16 if dtype != torch.float32 else torch.int32), x.view(torch.int16 if dtype != torch.float32 else torch.int32))
    close(got, want, x, scale)
    if dtype == torch.float32:                                               # in place
        same = K.constrain_logits(wide, tokens=d(tokens), starts=d(starts), lengths=d(lengths), prompt_lengths=d(prompts), repetition=d(rep), frequency=d(freq),
                                  presence=d(pres), bias_ids=d(ids), bias_values=d(bias), allowed=d(allowed), out=wide)
        assert same is wide and torch.equal(wide, out)


@pytest.mark.parametrize("dev", DEVICES)
def test_one_number_for_all_rows(dev):
    """Scalars and bounds of one element stand for every row; what is left out changes nothing, and a token that does not occur keeps its bits."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 500, generator=g)
    tokens = torch.randint(0, 500, (3, 40), generator=g, dtype=torch.int32)
    i = lambda v: torch.tensor([v], dtype=torch.int32, device=dev)
    got = K.constrain_logits(x.to(dev), tokens=tokens.to(dev), starts=i(3), lengths=i(30), prompt_lengths=i(20), repetition=1.3, presence=0.5)
    want = oracle.rules(x, tokens, [3] * 3, [30] * 3, [20] * 3, [1.3] * 3, [0.0] * 3, [0.5] * 3)
    close(got, want, x, x.abs().double() * 2 + 1)
    for b in range(3):
        absent = torch.ones(500, dtype=torch.bool)
        absent[tokens[b, 3:30].long()] = False
        assert torch.equal(got[b].cpu()[absent], x[b, absent])
    assert torch.equal(K.constrain_logits(x.to(dev)).cpu(), x)
    assert torch.equal(K.constrain_logits(x.to(dev), tokens=tokens.to(dev)).cpu(), x)
    assert K.constrain_logits(x[:0].to(dev)).shape == (0, 500)


@pytest.mark.parametrize("dev", DEVICES)
def test_nan_and_infinities_stay_where_they_are(dev):
    x = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, -1.0, math.nan, 2.0]])
    tokens = torch.tensor([[0, 1, 2, 3, 4]], dtype=torch.int32)
    allowed = torch.tensor([[0b1011111]], dtype=torch.int32)
    got = K.constrain_logits(x.to(dev), tokens=tokens.to(dev), repetition=2.0, frequency=1.0, allowed=allowed.to(dev)).cpu()
    assert torch.isnan(got[0, 0]) and got[0, 1:].tolist() == [math.inf, -math.inf, -0.5, -3.0, -math.inf, 2.0]


def test_refusals():
    x = torch.zeros(2, 40)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bad = [dict(tokens=torch.zeros(2, 4)), dict(tokens=i(3, 4)), dict(tokens=i(2, 8)[:, ::2]), dict(lengths=i(2)), dict(tokens=i(2, 4), lengths=i(3)),
           dict(tokens=i(2, 4), starts=torch.zeros(2)), dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=math.nan), dict(repetition=torch.ones(3)),
           dict(frequency=torch.ones(2, dtype=torch.float64)), dict(bias_ids=i(2, 3)), dict(bias_ids=i(2, 3), bias_values=torch.zeros(2, 4)),
           dict(bias_ids=i(3, 3), bias_values=torch.zeros(3, 3)), dict(bias_ids=i(1, 8193), bias_values=torch.zeros(1, 8193)), dict(allowed=i(2, 1)), dict(allowed=i(2, 2).float()), dict(allowed=i(3, 2)), dict(out=torch.zeros(2, 41)),
           dict(out=torch.zeros(2, 40, dtype=torch.bfloat16))]
    for kw in bad:
        with pytest.raises(ValueError):
            K.constrain_logits(x, **kw)
    for logits in (torch.zeros(40), torch.zeros(2, 40, dtype=torch.float64), torch.zeros(40, 2).t()):
        with pytest.raises(ValueError):
            K.constrain_logits(logits)


@pytest.mark.parametrize("dev", DEVICES)
def test_out_may_be_the_logits_or_apart(dev):
    buf = torch.randn(3, 100, generator=torch.Generator().manual_seed(1)).to(dev)
    want = buf[:, :40] - 0.0
    for bad in (buf[:, 1:41], buf[:, 39:79], buf[:, 20:60]):
        with pytest.raises(ValueError):
            K.constrain_logits(buf[:, :40], out=bad)
    half = buf.view(-1).view(torch.bfloat16)[:120].view(3, 40)
    with pytest.raises(ValueError):
        K.constrain_logits(half, out=buf.view(-1)[:120].view(3, 40))
    assert torch.equal(K.constrain_logits(buf[:, :40], out=buf[:, 40:80]), want) and torch.equal(buf[:, 40:80], want)
    assert torch.equal(K.constrain_logits(buf[:, :40], out=buf[:, :40]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("B,V,T,dtype,n_bias,seed", [(8, 128000, 5001, torch.float32, 1200, 0), (9, 128259, 4100, torch.bfloat16, 0, 1), (4, 100003, 2500, torch.bfloat16, 600, 2),
                                                     (3, 40001, 1030, torch.float16, 300, 3), (1, 3001, 9, torch.float32, 8192, 4)])
def test_long_histories_and_many_biases(B, V, T, dtype, n_bias, seed):
    """Every width of slice, history and entries beyond what is asked for ahead, rows of tokens at any 4-byte boundary."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, V, generator=g) * 4).to(dtype)
    tokens = (torch.rand(B, T + 4, generator=g) ** 2 * V).to(torch.int32).clamp(max=V - 1)[:, 1:T + 1]
    rnd = lambda lo, hi: torch.randint(lo, hi + 1, (B,), generator=g, dtype=torch.int32)
    starts, lengths, prompts = rnd(0, 50), rnd(T - 9, T), rnd(0, T)
    rep, freq, pres = 0.7 + torch.rand(B, generator=g), torch.randn(B, generator=g), torch.randn(B, generator=g)
    ids = torch.randint(0, V, (B, n_bias), generator=g, dtype=torch.int32)
    if n_bias:
        ids[:, 5:n_bias:n_bias // 20] = ids[:, :1]                           # an id up to 23 times, from every round of entries
    bias = torch.randn(B, n_bias, generator=g)
    allowed = mask_of(1, V, 0.9, g)
    wanted = [oracle.rules(x[b:b + 1], tokens[b:b + 1], [int(starts[b])], [int(lengths[b])], [int(prompts[b])], [float(rep[b])], [float(freq[b])], [float(pres[b])],
                           ids[b:b + 1], bias[b:b + 1]) for b in range(B)]
    want = torch.cat(wanted)
    bits = (allowed.long()[:, torch.arange(V) // 32] >> (torch.arange(V) % 32)) & 1
    want = want.masked_fill(bits == 0, -math.inf)
    scale = x.double().abs() * 2 + (T * 4.0 + 4) * freq.abs().max() + pres.abs().max() + 5.0 * bias.abs().sum(1, keepdim=True)
    d = lambda t: t.to("cuda")
    buf = torch.full((B, T + 6), 7, dtype=torch.int32, device="cuda")
    buf[:, 1:T + 1] = d(tokens)
    got = K.constrain_logits(d(x), tokens=buf[:, 1:T + 1], starts=d(starts), lengths=d(lengths), prompt_lengths=d(prompts), repetition=d(rep), frequency=d(freq),
                             presence=d(pres), bias_ids=d(ids) if n_bias else None, bias_values=d(bias) if n_bias else None, allowed=d(allowed))
    close(got, want, x, scale)


@pytest.mark.gpu
def test_a_captured_call_follows_the_text():
    """The history is read at replay: tokens and lengths that changed in between count."""
    x, tokens, n = torch.randn(2, 900, device="cuda"), torch.zeros(2, 30, dtype=torch.int32, device="cuda"), torch.tensor([0], dtype=torch.int32, device="cuda")
    out, g = torch.empty_like(x), torch.cuda.CUDAGraph()
    kw = dict(tokens=tokens, lengths=n, repetition=1.5, frequency=0.25)
    with torch.cuda.graph(g):
        K.constrain_logits(x, out=out, **kw)
    for k in (0, 3, 30):
        tokens.copy_(torch.randint(0, 900, (2, 30), generator=torch.Generator().manual_seed(k)))
        n.fill_(k)
        g.replay()
        assert torch.equal(out, K.constrain_logits(x, **kw))
        assert (out != x).any().item() == (k > 0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("r", [1e-45, 1e-40, 2.0 ** -127, 0.3, 1.7, 2.0 ** 126, 2.0 ** 127, 3.4e38, math.inf])
def test_a_penalty_divides(r, dev):
    """x / r and x r as fp32 has them, each rounded once, over the whole range of penalties and logits."""
    x = torch.cat([torch.randn(200, generator=torch.Generator().manual_seed(5)) * 10.0 ** torch.arange(-40, 40).repeat_interleave(5)[:200].float(),
                   torch.tensor([1.0, 7.5, 3e38, 1e-45, math.inf, -1.0, -7.5, -3e38, -1e-45])])[None].float()
    want = torch.where(x > 0, x / torch.tensor(r), x * torch.tensor(r))
    tokens = torch.arange(x.shape[1], dtype=torch.int32)[None]
    for rep in (r, torch.tensor([r], device=dev)):
        got = K.constrain_logits(x.to(dev), tokens=tokens.to(dev), prompt_lengths=torch.tensor([x.shape[1]], dtype=torch.int32, device=dev), repetition=rep).cpu()
        assert torch.equal(got.nan_to_num(nan=123.0, posinf=math.inf, neginf=-math.inf), want.nan_to_num(nan=123.0, posinf=math.inf, neginf=-math.inf))


@pytest.mark.parametrize("dev", DEVICES)
def test_biases_of_one_token_are_summed_and_added_once(dev):
    """In the order of the entries: 1e8 and -1e8 leave a logit its bits, and 1 is lost behind 1e8, not in front of its opposite."""
    x = torch.tensor([[0.1, 0.2, 0.3]])
    ids = torch.tensor([[0, 1, 0, 1, 1]], dtype=torch.int32)
    bias = torch.tensor([[1e8, 1e8, -1e8, 1.0, -1e8]])
    got = K.constrain_logits(x.to(dev), bias_ids=ids.to(dev), bias_values=bias.to(dev)).cpu()
    assert torch.equal(got, x)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [40, 5003])
def test_one_row_of_logits_for_all(V, dev):
    """Rows that are one another's memory are read, each under its own rules; as a place for results they are refused, and so is one that overlaps the row."""
    g = torch.Generator().manual_seed(V)
    row, tokens = torch.randn(1, V, generator=g).to(dev), torch.randint(0, V, (3, 20), generator=g, dtype=torch.int32).to(dev)
    kw = dict(tokens=tokens, repetition=1.5, presence=0.25)
    assert torch.equal(K.constrain_logits(row.expand(3, V), **kw), K.constrain_logits(row.repeat(3, 1), **kw))
    half = V // 2
    for logits, out in ((row.expand(3, V), row.expand(3, V)), (row[:, :half].expand(2, half), row.view(-1)[:2 * half].view(2, half))):
        with pytest.raises(ValueError, match="overlaps"):
            K.constrain_logits(logits, tokens=tokens[:len(out)], out=out)
