"""Python front-ends of the sm_100a kernels.

Every op takes torch tensors.  CUDA bf16 tensors run the hand-written kernel through the C ABI on the
current stream (legal under CUDA-graph capture); CPU tensors run the fp32 PyTorch statement of the same
op, which is also the oracle the GPU tests compare against.  There is no third path: a CUDA tensor with
no native library raises.
"""
from __future__ import annotations

import math
import os
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F

from . import _lib

PLAIN, RESIDUAL, SWIGLU = 0, 1, 2
_NUM_SMS = {}
_SMALL_M_PATH = os.environ.get("JLLAMA_SMALL_M", "gemv")    # measured faster in the graph-replayed step than "gemv_tma"


_get_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """The current stream's handle (the callers hold CUDA tensors: CUDA is initialised).  torch.cuda.current_stream() builds a Stream object
    first: 3.2 us a call, a quarter of what a small linear costs the host; these two 0.2."""
    if _raw_stream is None or _get_device is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_get_device())


def num_sms(device: Optional[torch.device] = None) -> int:
    idx = torch.cuda.current_device() if device is None or device.index is None else device.index
    if idx not in _NUM_SMS:
        _NUM_SMS[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _NUM_SMS[idx]


_GEMM_WS: dict = {}


def ensure_gemm_workspace(device: Optional[torch.device] = None, nbytes: int = 4) -> None:
    """Allow split-K on this device: small-batch GEMMs with few weight-row tiles (N = 4096 at batch 9..128) then spread their K
    range over all SMs, a cluster per tile (the partial sums meet in distributed shared memory: the registered buffer is only the
    permission).  Done once, outside any stream capture (the engine calls it at construction); without it such GEMMs do not split."""
    idx = torch.cuda.current_device() if device is None or device.index is None else device.index
    if idx in _GEMM_WS or torch.cuda.is_current_stream_capturing() or os.environ.get("JLLAMA_NO_SPLITK") == "1":
        return
    with torch.cuda.device(idx):
        ws = torch.empty(nbytes // 4, dtype=torch.float32, device=f"cuda:{idx}")
        tickets = torch.zeros(2, dtype=torch.int32, device=f"cuda:{idx}")
        _lib.check(_lib.lib().jl_gemm_set_workspace(ws.data_ptr(), ws.numel() * 4, tickets.data_ptr(), tickets.numel()),
                   "jl_gemm_set_workspace")
    _GEMM_WS[idx] = (ws, tickets)


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _bf16c(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.bfloat16 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bf16 tensor (got {t.dtype}, contiguous={t.is_contiguous()})")


# --------------------------------------------------------------------------- embedding
def embed(ids: torch.Tensor, table: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if not table.is_cuda:
        return table[ids.long().clamp(0, table.shape[0] - 1)]
    _bf16c(table, "table")
    ids32 = ids.to(torch.int32).contiguous().view(-1)
    if out is None:
        out = torch.empty((ids32.numel(), table.shape[1]), dtype=table.dtype, device=table.device)
    _lib.check(_lib.lib().jl_embed(ids32.data_ptr(), table.data_ptr(), out.data_ptr(), ids32.numel(),
                                   table.shape[1], table.shape[0], _stream()), "jl_embed")
    return out


# --------------------------------------------------------------------------- RMSNorm
def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, delta: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, update_x: bool = True) -> torch.Tensor:
    """out = RMSNorm(x (+ delta)) · w.  With `delta`, x is updated in place to x + delta (residual)."""
    if not x.is_cuda:
        if delta is not None:
            s = x + delta
            if update_x:
                x.copy_(s)
        else:
            s = x
        xf = s.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()).to(x.dtype)
    _bf16c(x, "x"); _bf16c(w, "w")
    if delta is not None:
        _bf16c(delta, "delta")
    h = x.shape[-1]
    m = x.numel() // h
    if out is None:
        out = torch.empty_like(x)
    _lib.check(_lib.lib().jl_rmsnorm(x.data_ptr(), _p(delta), w.data_ptr(), out.data_ptr(),
                                     x.data_ptr() if (delta is not None and update_x) else 0,
                                     m, h, float(eps), _stream()), "jl_rmsnorm")
    return out


# --------------------------------------------------------------------------- RoPE + KV append
def rope_kv_write(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cos: torch.Tensor,
                  sin: torch.Tensor, B: int, S: int, nh: int, nkv: int, hd: int,
                  cache_len: Optional[torch.Tensor] = None, pad_left: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> None:
    """qkv [B·S, (nh+2nkv)·hd]; caches [B, nkv, T, hd]; cos/sin fp32 [max_pos, hd/2].  In-place on qkv's q
    block (or into q_out) and on the caches.  cache_len: int32 scalar tensor (device) or None (= 0)."""
    T = k_cache.shape[2]
    if not qkv.is_cuda:
        base = int(cache_len.item()) if cache_len is not None else 0
        x = qkv.view(B, S, nh + 2 * nkv, hd)
        slots = base + torch.arange(S)
        if positions is not None:
            pos = positions.view(B, S).long()
        else:
            pl = pad_left.long() if pad_left is not None else torch.zeros(B, dtype=torch.long)
            pos = (slots[None, :] - pl[:, None])
        pos = pos.clamp(0, cos.shape[0] - 1)
        c, s = cos[pos][:, :, None, :], sin[pos][:, :, None, :]          # [B,S,1,hd/2]
        qk = x[:, :, :nh + nkv].float()
        re, im = qk[..., 0::2], qk[..., 1::2]
        rot = torch.stack([re * c - im * s, re * s + im * c], -1).flatten(-2).to(qkv.dtype)
        if q_out is not None:
            q_out.view(B, S, nh, hd).copy_(rot[:, :, :nh])
        else:
            x[:, :, :nh] = rot[:, :, :nh]
        k_cache[:, :, base:base + S] = rot[:, :, nh:].transpose(1, 2)
        v_cache[:, :, base:base + S] = x[:, :, nh + nkv:].transpose(1, 2)
        return
    _bf16c(qkv, "qkv"); _bf16c(k_cache, "k_cache"); _bf16c(v_cache, "v_cache")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos/sin tables must be fp32")
    if positions is not None:
        positions = positions.to(torch.int32).contiguous()
    _lib.check(_lib.lib().jl_rope_kv_write(qkv.data_ptr(), _p(q_out), k_cache.data_ptr(), v_cache.data_ptr(),
                                           cos.data_ptr(), sin.data_ptr(), _p(cache_len), _p(pad_left),
                                           _p(positions), B, S, nh, nkv, hd, T, cos.shape[0], _stream()),
               "jl_rope_kv_write")


# --------------------------------------------------------------------------- SwiGLU
def swiglu(x: torch.Tensor, interleaved: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    f = x.shape[-1] // 2
    if not x.is_cuda:
        g, u = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :f], x[..., f:])
        return (F.silu(g.float()) * u.float()).to(x.dtype)
    _bf16c(x, "x")
    m = x.numel() // (2 * f)
    if out is None:
        out = torch.empty((*x.shape[:-1], f), dtype=x.dtype, device=x.device)
    _lib.check(_lib.lib().jl_swiglu(x.data_ptr(), out.data_ptr(), m, f, int(interleaved), _stream()), "jl_swiglu")
    return out


# --------------------------------------------------------------------------- linear layers
def _linear_ref(x, w, norm_w, eps, residual, mode, out_f32):
    xf = x.float()
    if norm_w is not None:
        xf = (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * norm_w.float()).to(x.dtype).float()
    y = (xf @ w.float().t())
    if out_f32:
        return y
    y = y.to(x.dtype)
    if mode == RESIDUAL:
        return (y.float() + residual.float()).to(x.dtype)
    if mode == SWIGLU:
        return (F.silu(y[..., 0::2].float()) * y[..., 1::2].float()).to(x.dtype)
    return y


def linear(x: torch.Tensor, w: torch.Tensor, *, norm_w: Optional[torch.Tensor] = None, eps: float = 1e-5,
           residual: Optional[torch.Tensor] = None, mode: int = PLAIN, out_f32: bool = False,
           out: Optional[torch.Tensor] = None, force: Optional[str] = None) -> torch.Tensor:
    """y = f(x) Wᵀ with W [N, K] for the per-op path (the whole-step decode kernel has its own GEMV).  Dispatch
    by token count: M ≤ 4 → register-streaming GEMV with RMSNorm fused (JLLAMA_SMALL_M=gemv_tma selects the
    TMA-ring GEMV, which falls back when the activations do not fit next to its ring), otherwise the tcgen05
    GEMM (swap-AB up to M = 128, and to 256 with few features).  `force` ∈ {"gemv_tma", "gemv", "gemm"} pins the kernel.  Up to 128
    rows w is a parameter: it is read ahead of this library's kernels directly before the call, which must not write it.
    An `int8.Int8Weight` for w makes it a layer in 8-bit integers (`int8.linear_int8`; no `force`): that is a parameter, read ahead, at any number of rows
    (`linear_int8` with `resident=False` is for weights that are written directly before)."""
    if not isinstance(w, torch.Tensor):
        from .int8 import linear_int8
        if force is not None:
            raise ValueError(f"linear: no path {force!r} for 8-bit weights")
        return linear_int8(x, w, norm_w=norm_w, eps=eps, residual=residual, mode=mode, out_f32=out_f32, out=out, resident=True)
    if not x.is_cuda:
        return _linear_ref(x, w, norm_w, eps, residual, mode, out_f32)
    _bf16c(x, "x"); _bf16c(w, "w")
    n, k = w.shape
    m = x.numel() // k
    odim = n // 2 if mode == SWIGLU else n
    if out is None:
        out = x.new_empty((m, odim), dtype=torch.float32 if out_f32 else x.dtype)
    sms = num_sms(x.device)
    if force is None:
        path = ("gemv_tma" if _SMALL_M_PATH == "gemv_tma" else "gemv") if m <= 4 else "gemm"
    else:
        path = force
    L = _lib.lib()
    if path == "gemv_tma":
        rc = L.jl_gemv_tma(x.data_ptr(), w.data_ptr(), _p(norm_w), _p(residual), out.data_ptr(), m, n, k,
                           float(eps), mode, int(out_f32), sms, _stream())
        if rc == 3 and force is None:
            path = "gemv"                      # activations too large for the TMA ring: register-streaming kernel
        else:
            _lib.check(rc, "jl_gemv_tma")
    if path == "gemv":
        if m > 8:
            raise ValueError("gemv path handles at most 8 rows")
        _lib.check(L.jl_gemv(x.data_ptr(), w.data_ptr(), _p(norm_w), _p(residual), out.data_ptr(), m, n, k,
                             float(eps), mode, int(out_f32), sms, _stream()), "jl_gemv")
    elif path == "gemm":
        if norm_w is not None:
            x = rmsnorm(x.view(m, k), norm_w, eps)
        if m <= 256 or n <= 64:                            # the sizes whose kernel may split K
            ensure_gemm_workspace(x.device)
        _lib.check(L.jl_gemm(x.data_ptr(), w.data_ptr(), _p(residual), out.data_ptr(), m, n, k, mode,
                             int(out_f32), sms, _stream()), "jl_gemm")
    elif path == "gemm_2cta":
        # the CTA-pair kernel alone (tests): shapes it does not cover are an error here, not a fallback
        if norm_w is not None:
            x = rmsnorm(x.view(m, k), norm_w, eps)
        rc = L.jl_gemm_2cta(x.data_ptr(), w.data_ptr(), _p(residual), out.data_ptr(), m, n, k, mode, sms, _stream())
        if rc == 3:
            raise ValueError(f"jl_gemm_2cta does not cover M={m}, N={n}, K={k} (needs M >= 256, N % 256 == 0, K % 64 == 0)")
        _lib.check(rc, "jl_gemm_2cta")
    elif path != "gemv_tma":
        raise ValueError(f"unknown linear path {path!r}")
    return out


# --------------------------------------------------------------------------- decode attention
def decode_attn_plan(B: int, nh: int, nkv: int, hd: int, max_len: int, device: torch.device
                     ) -> Tuple[int, Optional[torch.Tensor]]:
    """(splits, scratch) for jl_decode_attn at this shape; scratch is reused across layers and steps."""
    L = _lib.lib()
    splits = int(L.jl_decode_attn_splits(B, nkv, max_len, num_sms(device)))
    nbytes = int(L.jl_decode_attn_scratch_bytes(B, nh, hd, splits))
    scratch = torch.empty(max(nbytes, 4) // 4, dtype=torch.float32, device=device) if splits > 1 else None
    return splits, scratch


def decode_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                cache_len: Optional[torch.Tensor], pad_left: Optional[torch.Tensor], n_new: int = 1,
                splits: int = 1, scratch: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [B, nh, hd] (already rotated); caches [B, nkv, T, hd] → [B, nh·hd]."""
    B, nh, hd = q.shape
    nkv, T = k_cache.shape[1], k_cache.shape[2]
    scale = 1.0 / math.sqrt(hd)
    if not q.is_cuda:
        length = (int(cache_len.item()) if cache_len is not None else 0) + n_new
        k = k_cache[:, :, :length].float().repeat_interleave(nh // nkv, dim=1)
        v = v_cache[:, :, :length].float().repeat_interleave(nh // nkv, dim=1)
        s = torch.einsum("bhd,bhtd->bht", q.float(), k) * scale
        if pad_left is not None:
            s = s.masked_fill(torch.arange(length)[None, None, :] < pad_left.long()[:, None, None], float("-inf"))
        return torch.einsum("bht,bhtd->bhd", torch.softmax(s, -1), v).to(q.dtype).reshape(B, nh * hd)
    if q.dtype != torch.bfloat16 or q.stride(2) != 1 or q.stride(1) != hd:
        raise ValueError("q must be bf16 [B, nh, hd] with dense heads (batch pitch may be larger)")
    if out is None:
        out = torch.empty((B, nh * hd), dtype=q.dtype, device=q.device)
    _lib.check(_lib.lib().jl_decode_attn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _p(cache_len),
                                         _p(pad_left), _p(scratch), out.data_ptr(), B, nh, nkv, hd, T, n_new,
                                         scale, splits, q.stride(0) if B > 1 else 0, _stream()), "jl_decode_attn")
    return out


def decode_attn_fused_plan(B: int, nh: int, nkv: int, hd: int, max_len: int, device: torch.device
                           ) -> Tuple[int, torch.Tensor]:
    """(splits, zeroed scratch) for `decode_attn_fused` at this shape."""
    L = _lib.lib()
    splits = int(L.jl_decode_attn_fused_splits(B, nkv, max_len, num_sms(device)))
    nbytes = int(L.jl_decode_attn_fused_scratch_bytes(B, nh, nkv, hd, splits))
    return splits, torch.zeros((nbytes + 3) // 4, dtype=torch.int32, device=device)


def set_decode_attn_variant(variant: int) -> None:
    """Pins the kernel behind `decode_attn_fused`: 0 = by shape (default), 1 = SIMT, 2 = tensor-core.
    Process-wide; for tests and A/B timing."""
    _lib.check(_lib.lib().jl_decode_attn_fused_set_variant(int(variant)), "jl_decode_attn_fused_set_variant")


def decode_attn_fused(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cos: torch.Tensor,
                      sin: torch.Tensor, cache_len: torch.Tensor, pad_left: Optional[torch.Tensor], nh: int,
                      nkv: int, hd: int, splits: int = 1, scratch: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RoPE + KV append + GQA decode attention + split merge in one launch.  qkv [B, (nh+2nkv)·hd] is the
    raw fused projection of the new token; the caches are updated in place at slot `cache_len`."""
    B = qkv.shape[0]
    if not qkv.is_cuda:
        work = qkv.clone()
        rope_kv_write(work, k_cache, v_cache, cos, sin, B, 1, nh, nkv, hd, cache_len=cache_len, pad_left=pad_left)
        return decode_attn(work.view(B, nh + 2 * nkv, hd)[:, :nh], k_cache, v_cache, cache_len, pad_left, 1)
    _bf16c(qkv, "qkv"); _bf16c(k_cache, "k_cache"); _bf16c(v_cache, "v_cache")
    if scratch is None:
        splits, scratch = 1, torch.zeros(max(B * nkv, 1), dtype=torch.int32, device=qkv.device)
    if out is None:
        out = torch.empty((B, nh * hd), dtype=qkv.dtype, device=qkv.device)
    _lib.check(_lib.lib().jl_decode_attn_fused(qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                               cos.data_ptr(), sin.data_ptr(), cache_len.data_ptr(), _p(pad_left),
                                               scratch.data_ptr(), out.data_ptr(), B, nh, nkv, hd,
                                               k_cache.shape[2], cos.shape[0], 1.0 / math.sqrt(hd), splits,
                                               _stream()), "jl_decode_attn_fused")
    return out


# --------------------------------------------------------------------------- prefill attention
def prefill_attn_ref(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, start: int, S: int,
                     pad_left: Optional[torch.Tensor]) -> torch.Tensor:
    """Dense causal attention of S new tokens (slots start..start+S) against the cache; q [B, S, nh, hd]."""
    B, _, nh, hd = q.shape
    nkv = k_cache.shape[1]
    length = start + S
    k = k_cache[:, :, :length].float().repeat_interleave(nh // nkv, dim=1)
    v = v_cache[:, :, :length].float().repeat_interleave(nh // nkv, dim=1)
    s = torch.einsum("bqhd,bhkd->bhqk", q.float(), k) / math.sqrt(hd)
    qpos = torch.arange(start, length, device=q.device)[:, None]
    kpos = torch.arange(length, device=q.device)[None, :]
    ok = (kpos <= qpos)[None, None]
    if pad_left is not None:
        ok = ok & (kpos[None, None] >= pad_left.long()[:, None, None, None])
    s = s.masked_fill(~ok, torch.finfo(torch.float32).min)
    return torch.einsum("bhqk,bhkd->bqhd", torch.softmax(s, -1), v).to(q.dtype).reshape(B, S, nh * hd)


def prefill_attn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, start: int, S: int,
                 pad_left: Optional[torch.Tensor], cache_len: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, force: Optional[str] = None) -> torch.Tensor:
    """Causal flash attention of S new tokens per row against the (already appended) cache.

    q [B, S, nh, hd] rotated; caches [B, nkv, T, hd]; keys [pad_left[b], start+S) are visible, causally.
    head_dim 128 → tcgen05 kernel, 64 → warp-level tensor-core kernel; force="mma" pins the latter (64 / 128).
    """
    if not q.is_cuda:
        return prefill_attn_ref(q, k_cache, v_cache, start, S, pad_left)
    if not _lib.has("jl_flash_prefill"):
        raise _lib.NativeLibraryError("jl_flash_prefill is not built into libjllama_b200.so")
    _bf16c(q, "q")
    B, _, nh, hd = q.shape
    nkv, T = k_cache.shape[1], k_cache.shape[2]
    if out is None:
        out = torch.empty((B, S, nh * hd), dtype=q.dtype, device=q.device)
    if force == "mma":
        _lib.check(_lib.lib().jl_prefill_attn_mma(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _p(pad_left),
                                                  out.data_ptr(), B, S, nh, nkv, hd, T, start, 1.0 / math.sqrt(hd),
                                                  _stream()), "jl_prefill_attn_mma")
        return out
    _lib.check(_lib.lib().jl_flash_prefill(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _p(cache_len),
                                           _p(pad_left), out.data_ptr(), B, S, nh, nkv, hd, T, start,
                                           1.0 / math.sqrt(hd), _stream()), "jl_flash_prefill")
    return out


# --------------------------------------------------------------------------- attention over a prefix that the rows of a group share
# (The checks below run on every call of a decode step: identities and whole numbers, a message is put together only for what fails.)
_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16


def _here(dev: int, who: str) -> None:
    """Launches go to the current device's stream: tensors of another device are refused."""
    if _get_device is not None and dev != _get_device():
        raise ValueError(f"{who}: tensors on cuda:{dev}, current device cuda:{_get_device()}")


def _rows(t: Optional[torch.Tensor], n: int, dev: int, name: str, or_one: bool = False) -> None:
    """`t`, if given, is int32 [n] (or [1]) on device number `dev` (-1: the CPU)."""
    if t is None:
        return
    m = t.numel()
    if t.dtype is not _I32 or (m != n and not (or_one and m == 1)) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be int32, contiguous, of {n}{' or 1' if or_one else ''} elements, on the other tensors' device (got {t.dtype}, {tuple(t.shape)}, {t.device})")


def _prefix_shapes(who: str, B: int, nkv: int, hd: int, dev: int, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor) -> Tuple[int, int, int]:
    """(groups, P, T) of the two caches, or a refusal."""
    ps, cs = prefix_k.shape, k_cache.shape
    if len(ps) != 4 or len(cs) != 4 or prefix_v.shape != ps or v_cache.shape != cs:
        raise ValueError(f"{who}: keys and values are [groups, nkv, P, hd] and [B, nkv, T, hd]")
    groups, pn, P, ph = ps
    rows, cn, T, ch = cs
    if pn != nkv or cn != nkv or ph != hd or ch != hd or rows != B or groups < 1 or B % groups or P < 1 or T < 1:
        raise ValueError(f"{who}: prefix {tuple(ps)} and own keys {tuple(cs)} for {B} rows, {nkv} key heads of {hd}")
    for t in (prefix_k, prefix_v, k_cache, v_cache):
        if t.get_device() != dev or (dev >= 0 and (t.dtype is not _BF16 or not t.is_contiguous())):
            raise ValueError(f"{who}: keys and values are contiguous bf16 tensors on the queries' device (got {t.dtype}, contiguous={t.is_contiguous()}, {t.device})")
    if dev >= 0:
        _here(dev, who)
    return groups, P, T


def _prefix_counts(prefix_len: Optional[torch.Tensor], prefix_pad: Optional[torch.Tensor], groups: int, P: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """First and last + 1 shared key of every group (CPU path)."""
    lo = prefix_pad.long().clamp(min=0) if prefix_pad is not None else torch.zeros(groups, dtype=torch.long)
    hi = prefix_len.long().clamp(max=P) if prefix_len is not None else torch.full((groups,), P, dtype=torch.long)
    return lo, hi


def _prefix_attn_ref(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                     pad_left: Optional[torch.Tensor], lo: torch.Tensor, hi: torch.Tensor) -> torch.Tensor:
    """q [B, S, nh, hd] of tokens in `slots` [S] of their rows' own caches -> [B, S, nh·hd] in q's type; one softmax over shared and own keys."""
    B, S, nh, hd = q.shape
    groups, nkv, P, _ = prefix_k.shape
    T = k_cache.shape[2]
    row_group = torch.arange(B) // (B // groups)
    at = torch.arange(P)[None]
    shared = ((at >= lo[:, None]) & (at < hi[:, None]))[row_group]                                          # [B, P]
    own = torch.arange(T)[None, None] <= slots[None, :, None]
    own = own.expand(B, S, T)
    if pad_left is not None:
        own = own & (torch.arange(T)[None, None] >= pad_left.long()[:, None, None])
    seen = torch.cat([shared[:, None].expand(B, S, P), own], -1)
    live = seen.any(1)                                                                                      # slots that hold no key may hold anything
    k = torch.cat([prefix_k[row_group], k_cache], 2).float()
    v = torch.cat([prefix_v[row_group], v_cache], 2).float().masked_fill(~live[:, None, :, None], 0.0)
    k, v = k.repeat_interleave(nh // nkv, 1), v.repeat_interleave(nh // nkv, 1)
    s = torch.einsum("bshd,bhkd->bhsk", q.float(), k) / math.sqrt(hd)
    s = s.masked_fill(~seen[:, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    w = (s - torch.where(m == float("-inf"), torch.zeros_like(m), m)).exp()
    total = w.sum(-1, keepdim=True)
    o = torch.einsum("bhsk,bhkd->bshd", w / torch.where(total == 0, torch.ones_like(total), total), v)
    return o.masked_fill(~own.any(-1)[..., None, None], 0.0).to(q.dtype).reshape(B, S, nh * hd)


def prefix_attn_scratch(B: int, S: int, groups: int, nh: int, nkv: int, hd: int, prefix: int, device: torch.device) -> Optional[torch.Tensor]:
    """Workspace of `decode_attn_prefix` (S = 1) or `prefill_attn_prefix` for B rows in `groups` groups over prefixes of up to `prefix` slots.  One may serve all
    layers and steps of a stream of calls; calls that can run at the same time (two streams, two captured graphs) need one each."""
    if torch.device(device).type != "cuda":
        return None
    n = int(_lib.lib().jl_prefix_attn_scratch_bytes(B, S, groups, nh, nkv, hd, prefix))
    if n == 0:
        raise ValueError(f"prefix_attn_scratch: {B} rows of {S} tokens in {groups} groups, {nh} / {nkv} heads of {hd}, prefix {prefix}")
    return torch.empty((n + 15) // 16 * 4, dtype=torch.float32, device=device)


def decode_attn_prefix(qkv: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cos: torch.Tensor,
                       sin: torch.Tensor, cache_len: torch.Tensor, pad_left: Optional[torch.Tensor], prefix_len: Optional[torch.Tensor],
                       prefix_pad: Optional[torch.Tensor], nh: int, nkv: int, hd: int, *, scratch: Optional[torch.Tensor] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`decode_attn_fused` where the rows of a group share the keys in front of their own: RoPE + append to the row's own cache + attention over both.

    qkv [B, (nh+2nkv)·hd] is the raw projection of the new token of every row; prefix_k / prefix_v [groups, nkv, P, hd] hold every group's shared keys in slots
    [prefix_pad[g], prefix_len[g]) (int32 [groups]; None: all P, from 0), read once for the B / groups rows of the group (rows of a group are neighbours);
    k_cache / v_cache [B, nkv, T, hd] the rows' own keys from pad_left[b] (int32 [B] or None) on.  The new token takes slot cache_len (int32 [1], device; nothing is
    stored once the cache is full) at rotary position (prefix_len - prefix_pad)[g] + cache_len - pad_left[b].  -> [B, nh·hd]."""
    who = "decode_attn_prefix"
    B, width = qkv.shape if qkv.dim() == 2 else (-1, -1)
    if width != (nh + 2 * nkv) * hd:
        raise ValueError(f"{who}: qkv {tuple(qkv.shape)} for {nh} + 2 x {nkv} heads of {hd}")
    dev = qkv.get_device()
    groups, P, T = _prefix_shapes(who, B, nkv, hd, dev, prefix_k, prefix_v, k_cache, v_cache)
    _rows(cache_len, 1, dev, "cache_len"); _rows(pad_left, B, dev, "pad_left")
    _rows(prefix_len, groups, dev, "prefix_len"); _rows(prefix_pad, groups, dev, "prefix_pad")
    if dev < 0:
        lo, hi = _prefix_counts(prefix_len, prefix_pad, groups, P)
        slot = min(max(int(cache_len.item()), 0), T)
        x = qkv.view(B, nh + 2 * nkv, hd)
        pos = (hi - lo).clamp(min=0).repeat_interleave(B // groups) + slot
        if pad_left is not None:
            pos = pos - pad_left.long()
        pos = pos.clamp(0, cos.shape[0] - 1)
        c, s = cos[pos][:, None], sin[pos][:, None]
        re, im = x[:, :nh + nkv, 0::2].float(), x[:, :nh + nkv, 1::2].float()
        rot = torch.stack([re * c - im * s, re * s + im * c], -1).flatten(-2)
        kn, vn = rot[:, nh:].to(k_cache.dtype)[:, :, None], x[:, nh + nkv:].to(v_cache.dtype)[:, :, None]
        if slot < T:
            k_cache[:, :, slot:slot + 1], v_cache[:, :, slot:slot + 1] = kn, vn
        pad = torch.clamp(pad_left.long(), max=slot) if pad_left is not None else None        # the new token sees itself
        o = _prefix_attn_ref(rot[:, None, :nh], prefix_k, prefix_v, torch.cat([k_cache[:, :, :slot], kn], 2), torch.cat([v_cache[:, :, :slot], vn], 2),
                             torch.tensor([slot]), pad, lo, hi)
        return o.view(B, nh * hd).to(qkv.dtype)
    _bf16c(qkv, "qkv")
    table = cos.shape
    if cos.dtype is not _F32 or sin.dtype is not _F32 or sin.shape != table or table[1] != hd // 2 or not (cos.is_contiguous() and sin.is_contiguous()) \
            or cos.get_device() != dev or sin.get_device() != dev:
        raise ValueError(f"{who}: cos/sin tables are fp32 [positions, {hd // 2}] on {qkv.device}")
    if scratch is None:
        scratch = prefix_attn_scratch(max(B, groups), 1, groups, nh, nkv, hd, P, qkv.device)
    if out is None:
        out = qkv.new_empty((B, nh * hd))
    else:
        _bf16c(out, "out")
        if out.numel() != B * nh * hd:
            raise ValueError(f"{who}: out {tuple(out.shape)} for {B} x {nh * hd}")
    rc = _lib.lib().jl_decode_attn_prefix(qkv.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), cos.data_ptr(),
                                          sin.data_ptr(), cache_len.data_ptr(), _p(pad_left), _p(prefix_len), _p(prefix_pad), scratch.data_ptr(), scratch.nbytes,
                                          out.data_ptr(), B, groups, nh, nkv, hd, P, T, table[0], hd ** -0.5, _stream())
    if rc:
        _lib.check(rc, "jl_decode_attn_prefix")
    return out


def prefill_attn_prefix(q: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, start: int, S: int,
                        pad_left: Optional[torch.Tensor], prefix_len: Optional[torch.Tensor], prefix_pad: Optional[torch.Tensor], *,
                        scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`prefill_attn` where the rows of a group share the keys in front of their own.  q [B, S, nh, hd] rotated, the S new tokens of every row appended to its own
    cache in slots start..start+S; shared keys as in `decode_attn_prefix` (every query sees all of its group's), own keys [pad_left[b], slot of the query].  Queries
    in front of pad_left give zeros.  -> [B, S, nh·hd]."""
    who = "prefill_attn_prefix"
    B, s_q, nh, hd = q.shape if q.dim() == 4 else (0, -1, 0, 0)
    if s_q != S:
        raise ValueError(f"{who}: q {tuple(q.shape)} is not [B, {S}, heads, head_dim]")
    nkv, dev = k_cache.shape[1] if k_cache.dim() == 4 else 0, q.get_device()
    groups, P, T = _prefix_shapes(who, B, nkv, hd, dev, prefix_k, prefix_v, k_cache, v_cache)
    if start < 0 or start + S > T:
        raise ValueError(f"{who}: slots {start}..{start + S} of a cache of {T}")
    _rows(pad_left, B, dev, "pad_left"); _rows(prefix_len, groups, dev, "prefix_len"); _rows(prefix_pad, groups, dev, "prefix_pad")
    if dev < 0:
        lo, hi = _prefix_counts(prefix_len, prefix_pad, groups, P)
        return _prefix_attn_ref(q, prefix_k, prefix_v, k_cache[:, :, :start + S], v_cache[:, :, :start + S], start + torch.arange(S), pad_left, lo, hi)
    _bf16c(q, "q")
    if scratch is None:
        scratch = prefix_attn_scratch(max(B, groups), max(S, 1), groups, nh, nkv, hd, P, q.device)
    if out is None:
        out = q.new_empty((B, S, nh * hd))
    else:
        _bf16c(out, "out")
        if out.numel() != B * S * nh * hd:
            raise ValueError(f"{who}: out {tuple(out.shape)} for {B} x {S} x {nh * hd}")
    rc = _lib.lib().jl_prefill_attn_prefix(q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), _p(pad_left), _p(prefix_len),
                                           _p(prefix_pad), scratch.data_ptr(), scratch.nbytes, out.data_ptr(), B, S, groups, nh, nkv, hd, P, T, start, hd ** -0.5,
                                           _stream())
    if rc:
        _lib.check(rc, "jl_prefill_attn_prefix")
    return out


# --------------------------------------------------------------------------- the rules of a request on its logits
def _constrain_ref(x: torch.Tensor, tokens: Optional[torch.Tensor], starts: torch.Tensor, lengths: torch.Tensor, prompts: torch.Tensor, rep: torch.Tensor,
                   freq: torch.Tensor, pres: torch.Tensor, bias_ids: Optional[torch.Tensor], bias: Optional[torch.Tensor], allowed: Optional[torch.Tensor]) -> torch.Tensor:
    x = x.float().clone()
    B, V = x.shape
    for b in range(B):
        if tokens is not None:
            lo, hi, cut = max(int(starts[b]), 0), min(int(lengths[b]), tokens.shape[1]), int(prompts[b])
            said = tokens[b].long()
            for first, part in ((True, said[lo:hi]), (False, said[max(lo, cut):hi])):
                ids, n = torch.unique(part[(part >= 0) & (part < V)], return_counts=True)
                if first:
                    x[b, ids] = torch.where(x[b, ids] > 0, x[b, ids] / rep[b], x[b, ids] * rep[b])
                else:
                    x[b, ids] = x[b, ids] - freq[b] * n.float() - pres[b]
        if bias_ids is not None:
            ids, val = (t[b if t.shape[0] > 1 else 0] for t in (bias_ids, bias))
            ok = (ids >= 0) & (ids < V)
            x[b] += torch.zeros(V).index_add_(0, ids[ok].long(), val[ok])
        if allowed is not None:
            words = allowed[b if allowed.shape[0] > 1 else 0].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32)) & 1
            x[b, bits.view(-1)[:V] == 0] = float("-inf")
    return x


_LOGIT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _coefficient(v: Union[float, torch.Tensor, None], off: float, B: int, dev: int, name: str) -> Tuple[Optional[torch.Tensor], float]:
    """(fp32 [B], off) or (None, the number)."""
    if v is None:
        return None, off
    if isinstance(v, torch.Tensor):
        if v.dtype is not _F32 or v.dim() != 1 or v.shape[0] != B or not v.is_contiguous() or v.get_device() != dev:
            raise ValueError(f"constrain_logits: {name} is a number or fp32 [{B}] on the logits' device (got {v.dtype}, {tuple(v.shape)}, {v.device})")
        return v, off
    return None, float(v)


def _same_or_apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether y [B, V] is x, or has no byte of x: rows beside one another of one buffer are apart."""
    a, b, (B, V), n, m = x.data_ptr(), y.data_ptr(), x.shape, x.element_size(), y.element_size()
    p, q = (x.stride(0) * n, y.stride(0) * m) if B > 1 else (V * n, V * m)
    if a + (B - 1) * p + V * n <= b or b + (B - 1) * q + V * m <= a or B * V == 0:
        return True
    if p != q or p == 0:
        return False
    gap = (b - a) % p
    return (a == b and x.dtype is y.dtype) or (gap >= V * n and p - gap >= V * m)


def constrain_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                     prompt_lengths: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None, repetition: Union[float, torch.Tensor, None] = None,
                     frequency: Union[float, torch.Tensor, None] = None, presence: Union[float, torch.Tensor, None] = None,
                     bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rules of a request on the logits of a step, ahead of `argmax` / `sample_full`: fp32 [B, V] from logits [B, V] (fp32, bf16 or fp16; any row pitch).

    tokens int32 [B, T]: row b has said tokens[b, starts[b] : lengths[b]] (int32 [B], or [1] for all rows; None: 0 and T), the part from prompt_lengths[b] on (None:
    all of it) as its answer.  Ids outside the vocabulary are passed over.  For a token that occurs: x > 0 ? x / repetition : x · repetition; with n occurrences in
    the answer, n > 0: x - frequency · n - presence.  (A number, or fp32 [B]; None: off.  repetition > 0.)  Then x + bias_values of the entries of bias_ids
    (int32 / fp32 [B, n], or [1, n] for all rows, n <= 8192; an id outside the vocabulary is no entry, the same id twice adds the sum of both), then -inf where bit v % 32 of word v // 32
    of allowed (int32 [B, words] or [1, words]) is zero.  A row whose mask allows nothing is -inf throughout.  `out` may be `logits` itself when that is fp32; any
    other overlap is refused."""
    who = "constrain_logits"
    kind = _LOGIT_TYPES.get(logits.dtype)
    B, V = logits.shape if logits.dim() == 2 else (-1, -1)
    if kind is None or B < 0 or (V > 1 and logits.stride(1) != 1):
        raise ValueError(f"{who}: logits are [B, V], fp32, bf16 or fp16, with dense rows (got {logits.dtype}, {tuple(logits.shape)}, strides {logits.stride()})")
    dev = logits.get_device()
    T = ldt = n_start = n_len = n_prompt = 0
    if tokens is not None:
        T = tokens.shape[1] if tokens.dim() == 2 else -1
        if T < 0 or tokens.dtype is not _I32 or tokens.shape[0] != B or (T > 1 and tokens.stride(1) != 1) or tokens.get_device() != dev:
            raise ValueError(f"{who}: tokens are int32 [{B}, T] with dense rows on {logits.device} (got {tokens.dtype}, {tuple(tokens.shape)}, {tokens.device})")
        ldt = tokens.stride(0) if B > 1 else T
        if lengths is not None:
            _rows(lengths, B, dev, "lengths", True); n_len = lengths.numel()
        if prompt_lengths is not None:
            _rows(prompt_lengths, B, dev, "prompt_lengths", True); n_prompt = prompt_lengths.numel()
        if starts is not None:
            _rows(starts, B, dev, "starts", True); n_start = starts.numel()
    elif lengths is not None or prompt_lengths is not None or starts is not None:
        raise ValueError(f"{who}: row bounds without tokens")
    rep_t, rep = _coefficient(repetition, 1.0, B, dev, "repetition")
    freq_t, freq = _coefficient(frequency, 0.0, B, dev, "frequency")
    pres_t, pres = _coefficient(presence, 0.0, B, dev, "presence")
    if not rep > 0.0:
        raise ValueError(f"{who}: repetition {repetition} is not above zero")
    n_bias = ldb = 0
    if bias_ids is not None and bias_values is not None:
        shape = bias_ids.shape
        if len(shape) != 2 or bias_values.shape != shape or shape[0] not in (1, B) or bias_ids.dtype is not _I32 or bias_values.dtype is not _F32 \
                or not (bias_ids.is_contiguous() and bias_values.is_contiguous()) or bias_ids.get_device() != dev or bias_values.get_device() != dev:
            raise ValueError(f"{who}: biases are int32 and fp32 [{B} or 1, n] on {logits.device} (got {tuple(shape)}, {tuple(bias_values.shape)})")
        n_bias = shape[1]
        ldb = n_bias if shape[0] > 1 else 0
        if n_bias > 8192:
            raise ValueError(f"{who}: {n_bias} biases per row (at most 8192)")
    elif bias_ids is not None or bias_values is not None:
        raise ValueError(f"{who}: bias_ids and bias_values come together")
    lda = 0
    if allowed is not None:
        shape = allowed.shape
        if len(shape) != 2 or allowed.dtype is not _I32 or shape[0] not in (1, B) or shape[1] < (V + 31) // 32 or not allowed.is_contiguous() or allowed.get_device() != dev:
            raise ValueError(f"{who}: allowed is int32 [{B} or 1, {(V + 31) // 32} or more words] on {logits.device} (got {allowed.dtype}, {tuple(shape)})")
        lda = shape[1] if shape[0] > 1 else 0
    if out is not None and (out.dtype is not _F32 or out.shape != logits.shape or (V > 1 and out.stride(1) != 1) or out.get_device() != dev):
        raise ValueError(f"{who}: out is fp32 {tuple(logits.shape)} with dense rows on {logits.device} (got {out.dtype}, {tuple(out.shape)}, {out.device})")
    if out is not None and out is not logits and not _same_or_apart(logits, out):
        raise ValueError(f"{who}: out overlaps logits that it is not the same as")
    if dev < 0:
        def full(t: Optional[torch.Tensor], off: Union[int, float]) -> torch.Tensor:
            return torch.full((B,), off) if t is None else t.reshape(-1).expand(B)
        y = _constrain_ref(logits, tokens, full(starts, 0), full(lengths, T), full(prompt_lengths, 0), full(rep_t, rep), full(freq_t, freq), full(pres_t, pres),
                           bias_ids if n_bias else None, bias_values, allowed)
        return y if out is None else out.copy_(y)
    _here(dev, who)
    if out is None:
        out = logits.new_empty((B, V), dtype=torch.float32)
    rc = _lib.lib().jl_logit_rules(logits.data_ptr(), kind, B, V, logits.stride(0) if B > 1 else V, out.data_ptr(), out.stride(0) if B > 1 else V, _p(tokens), T, ldt,
                                   _p(starts), n_start, _p(lengths), n_len, _p(prompt_lengths), n_prompt, _p(rep_t), rep, _p(freq_t), freq, _p(pres_t), pres,
                                   _p(bias_ids), _p(bias_values), n_bias, ldb, _p(allowed), lda, _stream())
    if rc:
        _lib.check(rc, "jl_logit_rules")
    return out


# --------------------------------------------------------------------------- token selection
def argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if not logits.is_cuda:
        return logits.float().argmax(-1).to(torch.int32)
    B, V = logits.shape
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    _lib.check(_lib.lib().jl_argmax(logits.data_ptr(), B, V, logits.stride(0), 0, 0, out.data_ptr(), _stream()),
               "jl_argmax")
    return out


def topk_candidates(logits: torch.Tensor, k: int, idx_offset: int = 0,
                    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    B, V = logits.shape
    if not logits.is_cuda:
        vals, idx = torch.topk(logits.float(), min(k, V), dim=-1)
        return vals, (idx + idx_offset).to(torch.int32)
    if out is None:
        out = (torch.empty((B, k), dtype=torch.float32, device=logits.device),
               torch.empty((B, k), dtype=torch.int32, device=logits.device))
    _lib.check(_lib.lib().jl_topk(logits.data_ptr(), B, V, logits.stride(0), idx_offset, k, out[0].data_ptr(),
                                  out[1].data_ptr(), _stream()), "jl_topk")
    return out


def sample_candidates(vals: torch.Tensor, idx: torch.Tensor, *, n_lists: int = 1, list_stride: int = 0,
                      top_k: int = 0, top_p: float = 1.0, temperature: float = 1.0, seed: int = 0,
                      step: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """vals/idx: [n_lists, B, k] (or [B, k]).  CUDA only (the CPU path samples with ops.sampling)."""
    B, k = vals.shape[-2], vals.shape[-1]
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=vals.device)
    if list_stride == 0:
        list_stride = B * k
    _lib.check(_lib.lib().jl_sample(vals.data_ptr(), idx.data_ptr(), B, n_lists, list_stride, k, int(top_k or 0),
                                    float(top_p), float(temperature), int(seed), _p(step), out.data_ptr(),
                                    _stream()), "jl_sample")
    return out


# --------------------------------------------------------------------------- exact full-vocabulary selection
def sample_full(logits: torch.Tensor, *, temperature: float, top_k: int = 0, top_p: float = 1.0, seed: int = 0,
                step: Optional[torch.Tensor] = None, rows: Optional[int] = None) -> torch.Tensor:
    """Tokens [B] from fp32 logits [B, V] (or [V] read by `rows` independent draws): temperature → top-k → top-p →
    categorical over the whole vocabulary, exact and deterministic (csrc/sample_full.cu).  temperature 0 = arg-max."""
    if not logits.is_cuda or logits.dtype != torch.float32:
        raise ValueError("sample_full needs CUDA fp32 logits")
    if logits.dim() == 1:
        B, V, ld = int(rows or 1), logits.shape[0], 0
    else:
        B, V, ld = logits.shape[0], logits.shape[1], logits.stride(0)
    tok = logits.new_empty(B, dtype=torch.int32)
    _lib.check(_lib.lib().jl_sample_full(
        logits.data_ptr(), B, V, ld, float(temperature), int(top_k or 0), float(top_p), int(seed), _p(step), tok.data_ptr(),
        None, None, 1, 0, 0, 0, tok.data_ptr(), None, None, None, 0, 0, 0, None, None, None, None, _stream()),    # (no bookkeeping: no ticket)
        "jl_sample_full")
    return tok
