"""Attention over shared and own keys and the rules on logits, from their definitions in 64 bits, row by row."""
import math

import torch


def attention(q, pk, pv, kc, vc, slots, pad, plen, ppad):
    """q fp64 [B, S, nh, hd] of tokens in `slots`; -> (out, sum of weights times |values|) fp64 [B, S, nh, hd]; a query in front of its row's pad gives zeros."""
    B, S, nh, hd = q.shape
    groups, nkv = pk.shape[0], pk.shape[1]
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    for b in range(B):
        g = b // (B // groups)
        for i, slot in enumerate(slots):
            if slot < pad[b]:
                continue
            k = torch.cat([pk[g, :, ppad[g]:plen[g]], kc[b, :, pad[b]:slot + 1]], 1).double()
            v = torch.cat([pv[g, :, ppad[g]:plen[g]], vc[b, :, pad[b]:slot + 1]], 1).double()
            for h in range(nh):
                j = h // (nh // nkv)
                w = torch.softmax(k[j] @ q[b, i, h] / math.sqrt(hd), 0)
                out[b, i, h], mag[b, i, h] = w @ v[j], w @ v[j].abs()
    return out, mag


def rotate(x, pos, base=10000.0):
    """x [..., hd] fp64 -> pairs (2 i, 2 i + 1) turned by pos · base^(-2 i / hd), with the angle's cos and sin rounded to fp32 as the tables hold them."""
    hd = x.shape[-1]
    a = pos * base ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * torch.complex(a.cos().float().double(), a.sin().float().double())
    return torch.view_as_real(z).reshape(x.shape)


def tables(hd, n, base=10000.0):
    a = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)[None]
    return a.cos().float(), a.sin().float()


def rules(x, tokens=None, starts=None, lengths=None, prompts=None, rep=None, freq=None, pres=None, bias_ids=None, bias=None, allowed=None):
    """fp64 [B, V]; row bounds and coefficients as lists of numbers per row."""
    x = x.double().clone()
    B, V = x.shape
    for b in range(B):
        if tokens is not None:
            said, answered = {}, {}
            for i in range(max(starts[b], 0), min(lengths[b], tokens.shape[1])):
                t = int(tokens[b, i])
                if 0 <= t < V:
                    said[t] = said.get(t, 0) + 1
                    if i >= prompts[b]:
                        answered[t] = answered.get(t, 0) + 1
            for t in said:
                x[b, t] = x[b, t] / rep[b] if x[b, t] > 0 else x[b, t] * rep[b]
            for t, n in answered.items():
                x[b, t] = x[b, t] - freq[b] * n - pres[b]
        if bias_ids is not None:
            r = b if bias_ids.shape[0] > 1 else 0
            for t, v in zip(bias_ids[r].tolist(), bias[r].tolist()):
                if 0 <= t < V:
                    x[b, t] += v
        if allowed is not None:
            for t in range(V):
                if not (int(allowed[b if allowed.shape[0] > 1 else 0, t // 32]) >> (t % 32)) & 1:
                    x[b, t] = -math.inf
    return x
