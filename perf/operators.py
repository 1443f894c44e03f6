"""The operators of several answers to one prompt, and of many questions to one document: what is measured of them.

Three operators, each in a plain form of elementary torch operations and as the framework's call:

* ``step``    one new token of every row: its rotation and append to the row's own keys, attention over the prefix that the rows of a group share and
              over the row's own keys;
* ``prompt``  attention of S new tokens of every row (already rotated and appended) over the shared prefix and, causally, over the row's own keys;
* ``rules``   the logits of a step under the rules of a request: penalties for tokens that occurred, biases, a mask of allowed tokens.

``run`` takes the plain form unless ``own`` is set.
"""
import math

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # two samples of a short prompt on a model with 64-wide heads: the smallest step, where the launches count
        dict(name="step 2 rows, 96 shared", op="step", groups=1, rows=2, nh=32, nkv=8, hd=64, prefix=96, ragged=False, filled=3, cap=64),
        # sixteen samples of one prompt, a while into the answer
        dict(name="step 16 rows, 2048 shared", op="step", groups=1, rows=16, nh=32, nkv=8, hd=128, prefix=2048, ragged=False, filled=130, cap=512),
        # four prompts of unequal lengths with sixteen samples each, left-padded, odd sizes
        dict(name="step 4 x 16 rows, 3501 shared", op="step", groups=4, rows=16, nh=32, nkv=8, hd=128, prefix=3501, ragged=True, filled=701, cap=1021),
        # one head of keys per head of queries, 48 requests behind a long system prompt
        dict(name="step 48 rows, own heads", op="step", groups=1, rows=48, nh=32, nkv=32, hd=128, prefix=6000, ragged=False, filled=64, cap=256),
        # the largest: 96 requests over a document of 32 k tokens
        dict(name="step 96 rows, 32768 shared", op="step", groups=1, rows=96, nh=32, nkv=8, hd=128, prefix=32768, ragged=False, filled=500, cap=1000),
        # four short questions behind a short system prompt, 64-wide heads
        dict(name="prompt 4 x 17, 200 shared", op="prompt", groups=1, rows=4, nh=32, nkv=8, hd=64, prefix=200, ragged=False, start=0, S=17, cap=64),
        # many short questions to one document
        dict(name="prompt 16 x 48, 8192 shared", op="prompt", groups=1, rows=16, nh=32, nkv=8, hd=128, prefix=8192, ragged=False, start=0, S=48, cap=256),
        # two documents, four left-padded questions of middling length to each, a second turn (own keys before this call's)
        dict(name="prompt 2 x 4 x 333, 1500 shared", op="prompt", groups=2, rows=4, nh=32, nkv=8, hd=128, prefix=1500, ragged=True, start=77, S=333, cap=640),
        # the largest prompt: two long continuations of a long document
        dict(name="prompt 2 x 2048, 16384 shared", op="prompt", groups=1, rows=2, nh=32, nkv=8, hd=128, prefix=16384, ragged=False, start=0, S=2048, cap=2048),
        # one request of a small vocabulary with penalties: the smallest call
        dict(name="rules 1 x 32000", op="rules", rows=1, vocab=32000, dtype="float32", history=300, ragged=False, repetition=True, counts=False, biases=0, mask="none"),
        # a batch of chats: penalties of every kind and a few biases, histories of unequal lengths, an odd vocabulary
        dict(name="rules 17 x 128259", op="rules", rows=17, vocab=128259, dtype="float32", history=2049, ragged=True, repetition=True, counts=True, biases=24, mask="none"),
        # constrained decoding of a large batch: a grammar's mask for every row, long histories
        dict(name="rules 96 x 128256, masks", op="rules", rows=96, vocab=128256, dtype="float32", history=4000, ragged=True, repetition=True, counts=True, biases=300, mask="rows"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "step", "prompt", "prompt", "rules"])
    if op == "rules":
        return dict(op="rules", rows=_log(rng, 1, 96), vocab=_log(rng, 1000, 128256), dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]),
                    history=_log(rng, 1, 4000), ragged=rng.random() < 0.7, repetition=rng.random() < 0.7, counts=rng.random() < 0.7,
                    biases=rng.choice([0, 0, _log(rng, 1, 300)]), mask=rng.choice(["none", "rows", "shared"]))
    hd = rng.choice([64, 128, 128])
    nkv = rng.choice([1, 2, 8, 8, 32])
    nh = min(32, nkv * rng.choice([1, 2, 4, 8]))
    groups = rng.choice([1, 1, 1, 2, 3, 5])
    prefix = _log(rng, 1, 32768)
    ragged = rng.random() < 0.5
    if op == "step":
        most = max(1, min(96, (96 * 32768 * 8) // (groups * prefix * nkv * 4)))
        rows = _log(rng, 1, most)
        filled = _log(rng, 1, 500) - 1
        return dict(op="step", groups=groups, rows=rows, nh=nh, nkv=nkv, hd=hd, prefix=prefix, ragged=ragged, filled=filled, cap=filled + 1 + rng.randrange(200))
    budget = 2 * 32 * 2048 * 18432 / (groups * nh * (prefix + 2048))        # query rows: the scores of the plain form stay below the largest listed case's
    tokens = max(2, min(4096, int(budget)))
    rows = _log(rng, 1, min(16, tokens // 2))
    S = _log(rng, 1, max(1, min(2048, tokens // rows)))
    start = rng.choice([0, 0, _log(rng, 1, 100)])
    return dict(op="prompt", groups=groups, rows=rows, nh=nh, nkv=nkv, hd=hd, prefix=prefix, ragged=ragged, start=start, S=S, cap=start + S + rng.randrange(64))


# --------------------------------------------------------------------------- inputs
def _tables(hd, positions):
    """cos / sin of the interleaved rotation, fp32 [positions, hd / 2], angles in 64 bits."""
    inv = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv[None]
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)

    if case["op"] == "rules":
        B, V, L = case["rows"], case["vocab"], case["history"]
        s = dict(case, logits=(randn(B, V, dtype=torch.float32) * 3.0).to(getattr(torch, case["dtype"])))
        # what was said so far: few frequent tokens, many rare ones
        s["tokens"] = (torch.rand(B, L + 7, generator=g, device=DEV).pow(4.0) * V).to(torch.int32).clamp_(0, V - 1)
        s["starts"] = randint(0, L // 3 + 1, B) if case["ragged"] else None
        s["lengths"] = randint(L - L // 3, L + 1, B) if case["ragged"] else torch.full((B,), L, dtype=torch.int32, device=DEV)
        s["prompt_lengths"] = torch.full((B,), L // 2, dtype=torch.int32, device=DEV)
        s["repetition_t"] = 1.0 + 0.5 * torch.rand(B, generator=g, device=DEV) if case["repetition"] else None
        s["frequency_t"] = 0.6 * torch.rand(B, generator=g, device=DEV) if case["counts"] else None
        s["presence_t"] = 0.9 * torch.rand(B, generator=g, device=DEV) - 0.2 if case["counts"] else None
        n = case["biases"]
        s["bias_ids"] = torch.argsort(torch.rand(B, max(V, n), generator=g, device=DEV) if B * V < (1 << 25) else torch.rand(1, V, generator=g, device=DEV).expand(B, V),
                                      dim=-1)[:, :n].to(torch.int32).contiguous() if n else None
        s["bias_values"] = randn(B, n, dtype=torch.float32) * 4.0 if n else None
        words = (V + 31) // 32
        rows = {"none": 0, "shared": 1, "rows": B}[case["mask"]]
        # a grammar allows little: one token of sixteen
        s["allowed"] = (randint(-2 ** 31, 2 ** 31 - 1, rows, words) & randint(-2 ** 31, 2 ** 31 - 1, rows, words) & randint(-2 ** 31, 2 ** 31 - 1, rows, words)
                        & randint(-2 ** 31, 2 ** 31 - 1, rows, words)) if rows else None
        s["result"] = torch.empty(B, V, dtype=torch.float32, device=DEV)
        return s
    G, R, nh, nkv, hd, P, cap = (case[k] for k in ("groups", "rows", "nh", "nkv", "hd", "prefix", "cap"))
    B = G * R
    s = dict(case, B=B, prefix_k=randn(G, nkv, P, hd), prefix_v=randn(G, nkv, P, hd), k_cache=randn(B, nkv, cap, hd), v_cache=randn(B, nkv, cap, hd))
    own_keys = case["filled"] if case["op"] == "step" else case["start"]
    if case["ragged"]:
        s["prefix_len"] = randint(P - P // 3, P + 1, G)
        s["prefix_pad"] = randint(0, P // 4 + 1, G)
        s["pad_left"] = randint(0, (own_keys if case["op"] == "step" else own_keys + case["S"] // 2) + 1, B)
    else:
        s["prefix_len"] = torch.full((G,), P, dtype=torch.int32, device=DEV)
        s["prefix_pad"] = s["pad_left"] = None
    if case["op"] == "step":
        s["qkv"] = randn(B, (nh + 2 * nkv) * hd)
        s["cos"], s["sin"] = _tables(hd, P + cap)
        s["cache_len"] = torch.full((1,), case["filled"], dtype=torch.int32, device=DEV)
    else:
        s["q"] = randn(B, case["S"], nh, hd)
    return s


# --------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"step": _plain_step, "prompt": _plain_prompt, "rules": _plain_rules}[state["op"]](state)


def _own(s):
    from jax_llama_b200.ops import kernels as K
    if s["op"] == "rules":
        return K.constrain_logits(s["logits"], tokens=s["tokens"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"], starts=s["starts"],
                                  repetition=s["repetition_t"], frequency=s["frequency_t"], presence=s["presence_t"],
                                  bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"], out=s["result"])
    if "scratch" not in s:                                                   # kept with the cache, as a serving loop keeps it
        s["scratch"] = K.prefix_attn_scratch(s["B"], s["S"] if s["op"] == "prompt" else 1, s["groups"], s["nh"], s["nkv"], s["hd"], s["prefix"], torch.device(DEV))
    if s["op"] == "step":
        out = K.decode_attn_prefix(s["qkv"], s["prefix_k"], s["prefix_v"], s["k_cache"], s["v_cache"], s["cos"], s["sin"], s["cache_len"], s["pad_left"],
                                   s["prefix_len"], s["prefix_pad"], s["nh"], s["nkv"], s["hd"], scratch=s["scratch"])
        return {"out": out, "k": s["k_cache"], "v": s["v_cache"]}
    return K.prefill_attn_prefix(s["q"], s["prefix_k"], s["prefix_v"], s["k_cache"], s["v_cache"], s["start"], s["S"], s["pad_left"],
                                 s["prefix_len"], s["prefix_pad"], scratch=s["scratch"])


def _two_part_attention(s, q, seen_own):
    """q fp32 [B, S, nh, hd]; seen_own bool [B, S, cap]: own keys that each query sees.  softmax over the shared and the own keys together; a query that
    sees no own key is padding and gives zeros."""
    B, S, nh, hd = q.shape
    G, R, nkv, P = s["groups"], s["rows"], s["nkv"], s["prefix"]
    n = nh // nkv
    at = torch.arange(P, device=DEV)[None]
    seen_shared = at < s["prefix_len"][:, None]
    if s["prefix_pad"] is not None:
        seen_shared = seen_shared & (at >= s["prefix_pad"][:, None])
    q = q.view(B, S, nkv, n, hd).permute(0, 2, 1, 3, 4) * (1.0 / math.sqrt(hd))                                     # [B, nkv, S, n, hd]
    qg = q.reshape(G, R, nkv, S * n, hd).permute(0, 2, 1, 3, 4).reshape(G, nkv, R * S * n, hd)
    low = torch.finfo(torch.float32).min
    a = (qg @ s["prefix_k"].float().transpose(-1, -2)).masked_fill_(~seen_shared[:, None, None], low)               # [G, nkv, R S n, P]
    b = (q.reshape(B, nkv, S * n, hd) @ s["k_cache"].float().transpose(-1, -2)).view(B, nkv, S, n, -1)
    b = b.masked_fill_(~seen_own[:, None, :, None], low).view(B, nkv, S * n, -1)
    b_max = b.amax(-1, keepdim=True).view(G, R, nkv, S * n, 1).permute(0, 2, 1, 3, 4).reshape(G, nkv, R * S * n, 1)
    m = torch.maximum(a.amax(-1, keepdim=True), b_max)
    a = a.sub_(m).exp_().masked_fill_(~seen_shared[:, None, None], 0.0)
    own_m = m.view(G, nkv, R, S * n, 1).permute(0, 2, 1, 3, 4).reshape(B, nkv, S * n, 1)
    b = b.sub_(own_m).exp_().view(B, nkv, S, n, -1).masked_fill_(~seen_own[:, None, :, None], 0.0).view(B, nkv, S * n, -1)

    def by_row(t):
        return t.view(G, nkv, R, S * n, -1).permute(0, 2, 1, 3, 4).reshape(B, nkv, S * n, -1)

    # slots that hold no key may hold anything: their values do not count
    v_shared = s["prefix_v"].float().masked_fill(~seen_shared[:, None, :, None], 0.0)
    v_own = s["v_cache"].float().masked_fill(~seen_own.any(1)[:, None, :, None], 0.0)
    total = by_row(a.sum(-1, keepdim=True)) + b.sum(-1, keepdim=True)
    o = (by_row(a @ v_shared) + b @ v_own) / total
    o = o.view(B, nkv, S, n, hd).permute(0, 2, 1, 3, 4).reshape(B, S, nh * hd)
    return o.masked_fill(~seen_own.any(-1)[..., None], 0.0)


def _rotate(x, cos, sin):
    """Pairs (2 i, 2 i + 1) of the last dimension by the tables' angle; cos / sin broadcast over heads."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _positions(s):
    """Rotary position of the new token of every row."""
    shared = s["prefix_len"] if s["prefix_pad"] is None else s["prefix_len"] - s["prefix_pad"]
    own_keys = s["filled"] if s["pad_left"] is None else s["filled"] - s["pad_left"]
    return (shared.repeat_interleave(s["rows"]) + own_keys).long()


def _plain_step(s):
    B, nh, nkv, hd, t = s["B"], s["nh"], s["nkv"], s["hd"], s["filled"]
    x = s["qkv"].view(B, nh + 2 * nkv, hd).float()
    p = _positions(s)
    qk = _rotate(x[:, :nh + nkv], s["cos"][p][:, None], s["sin"][p][:, None])
    s["k_cache"][:, :, t] = qk[:, nh:].to(torch.bfloat16)
    s["v_cache"][:, :, t] = s["qkv"].view(B, nh + 2 * nkv, hd)[:, nh + nkv:]
    at = torch.arange(s["cap"], device=DEV)[None]
    seen = (at <= t).expand(B, -1)
    if s["pad_left"] is not None:
        seen = seen & (at >= s["pad_left"][:, None])
    out = _two_part_attention(s, qk[:, None, :nh], seen[:, None])
    return {"out": out.view(B, nh * hd).to(torch.bfloat16), "k": s["k_cache"], "v": s["v_cache"]}


def _plain_prompt(s):
    B, S = s["B"], s["S"]
    at = torch.arange(s["cap"], device=DEV)[None, None]
    slot = s["start"] + torch.arange(S, device=DEV)[None, :, None]
    seen = (at <= slot).expand(B, S, -1)
    if s["pad_left"] is not None:
        seen = seen & (at >= s["pad_left"][:, None, None])
    return _two_part_attention(s, s["q"].float(), seen).to(torch.bfloat16)


def _plain_rules(s):
    B, V = s["rows"], s["vocab"]
    x = s["logits"].float()
    at = torch.arange(s["tokens"].shape[1], device=DEV)[None]
    said = at < s["lengths"][:, None]
    if s["starts"] is not None:
        said = said & (at >= s["starts"][:, None])
    ids = s["tokens"].long()
    any_count = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, said.float())
    out_count = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, (said & (at >= s["prompt_lengths"][:, None])).float())
    if s["repetition_t"] is not None:
        r = s["repetition_t"][:, None]
        x = torch.where(any_count > 0, torch.where(x > 0, x / r, x * r), x)
    if s["frequency_t"] is not None:
        x = x - s["frequency_t"][:, None] * out_count - s["presence_t"][:, None] * (out_count > 0)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    if s["allowed"] is not None:
        v = torch.arange(V, device=DEV)
        x = x.masked_fill(((s["allowed"][:, v // 32] >> (v % 32)) & 1) == 0, float("-inf"))
    return x


# --------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rules":
        return _exact_rules(s)
    return _exact_attention(s)


def _exact_attention(s):
    """Every row on its own: its visible keys in one list, then softmax."""
    B, nh, nkv, hd = s["B"], s["nh"], s["nkv"], s["hd"]
    step = s["op"] == "step"
    S = 1 if step else s["S"]
    t0 = s["filled"] if step else s["start"]
    k_own, v_own = s["k_cache"].double(), s["v_cache"].double()
    if step:
        x = s["qkv"].double().view(B, nh + 2 * nkv, hd)
        pairs = torch.view_as_complex(x[:, :nh + nkv].reshape(B, nh + nkv, hd // 2, 2).contiguous())
    out = torch.zeros(B, S, nh * hd, dtype=torch.float64, device=DEV)
    new_k = k_own.clone() if step else None
    for b in range(B):
        g = b // s["rows"]
        lo = int(s["prefix_pad"][g]) if s["prefix_pad"] is not None else 0
        hi = int(s["prefix_len"][g])
        pad = int(s["pad_left"][b]) if s["pad_left"] is not None else 0
        if step:
            p = hi - lo + t0 - pad
            turned = torch.view_as_real(pairs[b] * torch.complex(s["cos"][p].double(), s["sin"][p].double())[None]).reshape(nh + nkv, hd)
            q = turned[None, :nh]
            new_k[b, :, t0] = turned[nh:]
            # what the cache holds of the new key is rounded to its type, and that is what attention reads
            k_own[b, :, t0] = turned[nh:].to(torch.bfloat16).double()
            v_own[b, :, t0] = x[b, nh + nkv:]
        else:
            q = s["q"][b].double()
        keys = torch.cat([s["prefix_k"][g, :, lo:hi].double(), k_own[b, :, pad:t0 + S]], 1)
        vals = torch.cat([s["prefix_v"][g, :, lo:hi].double(), v_own[b, :, pad:t0 + S]], 1)
        n_shared = max(hi - lo, 0)
        slots = torch.arange(pad, t0 + S, device=DEV)
        for h in range(nkv):
            for a in range(0, S, 512):
                z = min(S, a + 512)
                w = torch.einsum("sgd,kd->sgk", q[a:z, h * (nh // nkv):(h + 1) * (nh // nkv)], keys[h]) / math.sqrt(hd)
                ok = torch.cat([torch.ones(z - a, n_shared, dtype=torch.bool, device=DEV), slots[None] <= torch.arange(t0 + a, t0 + z, device=DEV)[:, None]], 1)
                w = w.masked_fill(~ok[:, None], float("-inf")).softmax(-1)
                y = torch.einsum("sgk,kd->sgd", w, vals[h])
                y = torch.where((torch.arange(t0 + a, t0 + z, device=DEV) >= pad)[:, None, None], y, torch.zeros_like(y))
                out[b, a:z].view(z - a, nh, hd)[:, h * (nh // nkv):(h + 1) * (nh // nkv)] = y
    if step:
        return {"out": out.view(B, nh * hd), "k": new_k, "v": v_own}
    return out


def _exact_rules(s):
    """Row by row, with the occurrences counted by sorting."""
    x = s["logits"].double()
    for b in range(s["rows"]):
        lo = int(s["starts"][b]) if s["starts"] is not None else 0
        hi, cut = int(s["lengths"][b]), int(s["prompt_lengths"][b])
        ids, _ = torch.unique(s["tokens"][b, lo:hi].long(), return_counts=True)
        if s["repetition_t"] is not None:
            r, v = s["repetition_t"][b].double(), x[b, ids]
            x[b, ids] = torch.where(v > 0, v / r, v * r)
        if s["frequency_t"] is not None:
            ids, n = torch.unique(s["tokens"][b, max(lo, cut):hi].long(), return_counts=True)
            x[b, ids] -= s["frequency_t"][b].double() * n.double() + s["presence_t"][b].double()
        if s["bias_ids"] is not None:
            x[b].index_add_(0, s["bias_ids"][b].long(), s["bias_values"][b].double())
        if s["allowed"] is not None:
            words = s["allowed"][b if s["allowed"].shape[0] > 1 else 0].long() & 0xFFFFFFFF
            bits = ((words[:, None] >> torch.arange(32, device=DEV)[None]) & 1).view(-1)[: s["vocab"]]
            x[b, bits == 0] = float("-inf")
    return x


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "rules":
        B, V = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        mask = {"none": 0, "shared": 1, "rows": B}[case["mask"]] * ((V + 31) // 32) * 4
        return {"bytes": B * V * (size + 4) + B * case["history"] * 4 + B * case["biases"] * 8 + mask, "flops": B * V}
    G, R, nh, nkv, hd, P = (case[k] for k in ("groups", "rows", "nh", "nkv", "hd", "prefix"))
    B = G * R
    row = nkv * hd * 2 * 2                                                    # keys and values of a token
    if case["op"] == "step":
        t = case["filled"]
        return {"bytes": G * P * row + B * (t + 1) * row + B * (nh + 2 * nkv) * hd * 2 + B * nh * hd * 2, "flops": 4.0 * B * nh * hd * (P + t + 1)}
    t, S = case["start"], case["S"]
    return {"bytes": G * P * row + B * (t + S) * row + 2 * B * S * nh * hd * 2, "flops": 4.0 * B * nh * hd * (S * (P + t) + S * (S + 1) / 2)}
