"""Layers whose weights and activations are 8-bit integers.

A row of numbers is held as int8 values and one fp32 scale: ``s = amax / 127``, ``q = 127 x / amax`` rounded to the nearest whole number, ties to even.  Weights
[N, K] have a scale per output feature and are laid out once (`Int8Weight`); activations get one per token in front of every product.  Sums are whole numbers
in 32 bits, exact; both scales, a residual or a gate meet them in fp32, and the result is rounded once.  Against bf16 a layer reads half the bytes and its products run
at twice the tensor cores' rate.

CUDA tensors run the hand-written kernels (csrc/int8_*.cu) on the current stream, legal under CUDA-graph capture; CPU tensors the PyTorch statement of the same
operator.  There is no backward pass, as for no operator of this package.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import _lib
from .kernels import PLAIN, RESIDUAL, SWIGLU, _here, _stream, num_sms

TYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
MAX_K = 131072                 # inputs of a layer: 127 * 127 * K stays below 2^31
MAX_EXPERTS = 1024
MAX_ROWS = 1 << 30
MAX_COLUMNS = 1 << 30          # of `quantize_rows`
RELU2 = 3                      # a mode beside `kernels`' PLAIN, RESIDUAL and SWIGLU: relu(y)²
MAX_CHOICES, MAX_CHOICE_K = 8, 16384          # rows and inputs of `choice_linear_int8`
_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32


# --------------------------------------------------------------------------- rows
def _rows_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    xd = x.double()
    amax = xd.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(amax) & (amax > 0)                       # (a NaN anywhere makes amax one)
    q = torch.where(fine, xd * 127.0 / torch.where(fine, amax, torch.ones_like(amax)), torch.zeros_like(xd)).round()
    s = torch.where(torch.isfinite(amax), amax / 127.0, torch.full_like(amax, float("nan"))).float()
    return q.to(_I8), s.squeeze(-1)


def _norm_ref(x: torch.Tensor, norm_w: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    if norm_w is None:
        return x
    xf = x.float()
    return xf / (xf.pow(2).mean(-1, keepdim=True) + eps).sqrt() * norm_w.float()


def _take(who: str, x: torch.Tensor, K: int) -> Tuple[torch.Tensor, int, int]:
    """x as rows [M, K] with dense rows, M and the row pitch, or a refusal.  (On every call of a decode step: a message is put together only for what fails.)"""
    shape = x.shape
    if len(shape) == 2 and shape[1] == K and K > 0 and x.dtype in TYPES:
        M = shape[0]
        if x.is_contiguous():
            return x, M, K
        pitch = x.stride(0) if M > 1 else K
        if (K == 1 or x.stride(1) == 1) and pitch >= K:
            return x, M, pitch
    elif len(shape) >= 1 and shape[-1] == K and K > 0 and x.dtype in TYPES and x.is_contiguous():
        return x.view(-1, K), x.numel() // K, K
    raise ValueError(f"{who}: x is rows of {K} numbers in bf16, fp16 or fp32: [M, {K}] with dense rows that do not overlap, or contiguous (got {x.dtype}, {tuple(shape)}, "
                     f"strides {x.stride()})")


def _few(who: str, rows: int) -> None:
    if rows > MAX_ROWS:
        raise ValueError(f"{who}: {rows} rows (at most {MAX_ROWS})")


def _gain(who: str, norm_w: torch.Tensor, x: torch.Tensor, K: int) -> None:
    if (norm_w.dtype is not x.dtype or norm_w.numel() != K or not norm_w.is_contiguous() or norm_w.get_device() != x.get_device()):
        raise ValueError(f"{who}: norm_w is {x.dtype} [{K}], contiguous, on {x.device} (got {norm_w.dtype}, {tuple(norm_w.shape)}, {norm_w.device})")


def quantize_rows(x: torch.Tensor, *, norm_w: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(values int8 [..., K], scales fp32 [...]) of the rows of x [..., K] (bf16, fp16 or fp32; two dimensions: any row pitch).  Both are what 64 bits would give: the
    scale is amax / 127 rounded once, a value is the whole number nearest to 127 x / amax.  At most MAX_ROWS rows of MAX_COLUMNS.  A row of zeros has scale 0; a row that holds an infinity or a NaN has scale
    NaN and values 0, so that what it is multiplied with is NaN.  With norm_w the rows are normed first (RMS, fp32, no rounding in between), on CUDA with the
    same bits beside any rows; of what fp32 leaves, a value whose quotient is next to a middle may be the neighbour of the one of 64 bits."""
    who = "quantize_rows"
    if x.dim() < 1:
        raise ValueError(f"{who}: x has no rows")
    K = x.shape[-1]
    x2, M, pitch = _take(who, x, K)
    _few(who, M)
    if K > MAX_COLUMNS:
        raise ValueError(f"{who}: rows of {K} numbers (at most {MAX_COLUMNS})")
    if norm_w is not None:
        _gain(who, norm_w, x2, K)
    shape = x.shape
    if out is None:
        q = torch.empty_like(x, dtype=_I8, memory_format=torch.contiguous_format)
        s = x.new_empty(M, dtype=_F32) if len(shape) == 2 else x.new_empty(shape[:-1], dtype=_F32)
    else:
        q, s = out
        if q.dtype is not _I8 or s.dtype is not _F32 or q.shape != shape or s.shape != shape[:-1] or not (q.is_contiguous() and s.is_contiguous()) \
                or q.get_device() != x.get_device() or s.get_device() != x.get_device():
            raise ValueError(f"{who}: out is int8 {tuple(shape)} and fp32 {tuple(shape[:-1])}, contiguous, on {x.device}")
        if not (_apart(x2, pitch, M, K, q) and _apart(x2, pitch, M, K, s)):
            raise ValueError(f"{who}: out overlaps x")
    if not x.is_cuda:
        v, sc = _rows_ref(_norm_ref(x2, norm_w, eps))
        q.view(-1, K).copy_(v)
        s.view(-1).copy_(sc)
        return q, s
    _here(x.get_device(), who)
    if M:
        rc = _lib.lib().jl_int8_rows(x2.data_ptr(), TYPES[x.dtype], M, K, pitch, 0, M, 0 if norm_w is None else norm_w.data_ptr(), eps, q.data_ptr(), K, s.data_ptr(), _stream())
        if rc:
            _lib.check(rc, "jl_int8_rows")
    return q, s


# --------------------------------------------------------------------------- weights
class Int8Weight:
    """Weights [N, K], or [E, N, K] of E experts, as int8 values and fp32 scales [N] / [E, N].  Rows lie on 16-byte boundaries (a copy is made where K is not a multiple
    of 16).  A SWIGLU layer's rows are interleaved: row 2j is the gate of result j, row 2j + 1 its up part (`models.engine.interleave_rows`).  Calls use the addresses of
    values and scales: new numbers are written into those, and no field is assigned."""

    __slots__ = ("values", "scales", "experts", "n", "k", "pitch", "device", "dev", "_held")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype is not _I8 or values.dim() not in (2, 3) or scales.dtype is not _F32 or scales.shape != values.shape[:-1] or scales.get_device() != values.get_device():
            raise ValueError(f"Int8Weight: values are int8 [N, K] or [E, N, K], scales fp32 of all but the last dimension, on one device (got {values.dtype} {tuple(values.shape)} on "
                             f"{values.device}, {scales.dtype} {tuple(scales.shape)} on {scales.device})")
        k = values.shape[-1]
        if not 1 <= k <= MAX_K or values.numel() == 0 or scales.numel() > MAX_ROWS:
            raise ValueError(f"Int8Weight: 1 to {MAX_K} inputs, at least one feature and at most {MAX_ROWS} (got {tuple(values.shape)})")
        pitch = -(-k // 16) * 16
        if pitch != k or not values.is_contiguous() or values.data_ptr() % 16:
            room = values.new_zeros((*values.shape[:-1], pitch))
            room[..., :k].copy_(values)
            values = room[..., :k]
        self.values, self.scales = values, scales.contiguous()
        self.experts = values.shape[0] if values.dim() == 3 else 0
        self.n, self.k, self.pitch = values.shape[-2], k, pitch
        self.device, self.dev = values.device, values.get_device()
        # what a call hands to the library: (values, row pitch, scales, features), and the SMs there are (asked once: a layer is called for every token)
        self._held = (values.data_ptr(), pitch, self.scales.data_ptr(), self.n), num_sms(self.device) if self.dev >= 0 else 0

    def __setattr__(self, name: str, value: object) -> None:
        if hasattr(self, "_held"):
            raise AttributeError(f"Int8Weight: {name} is not assigned once it is laid out (write into its values and scales, or make another one)")
        object.__setattr__(self, name, value)

    def __reduce__(self) -> tuple:
        """Copied and pickled as values and scales: the copy is laid out where its own are."""
        return Int8Weight, (self.values, self.scales)

    @classmethod
    def of(cls, w: torch.Tensor) -> "Int8Weight":
        """The rows of w [N, K] or [E, N, K] (bf16, fp16 or fp32) in 8 bits."""
        return cls(*quantize_rows(w.contiguous()))

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def nbytes(self) -> int:
        """Bytes that a pass over the weights reads."""
        return self.scales.numel() * (self.k + 4)

    def float(self) -> torch.Tensor:
        """The numbers that the values stand for, fp32."""
        return self.values.float() * self.scales[..., None]


# --------------------------------------------------------------------------- products
def _finish_ref(y: torch.Tensor, residual: Optional[torch.Tensor], mode: int, dtype: torch.dtype) -> torch.Tensor:
    if mode == SWIGLU:
        y = F.silu(y[..., 0::2]) * y[..., 1::2]
    elif mode == RELU2:
        y = F.relu(y).square()
    elif mode == RESIDUAL:
        y = y + residual.view(y.shape).float()
    return y.to(dtype)


def _apart(x: torch.Tensor, pitch: int, rows: int, k: int, out: torch.Tensor) -> bool:
    """Whether out (contiguous) has no byte between the first and the last of x's rows."""
    a, b = x.data_ptr(), out.data_ptr()
    return rows == 0 or a + ((rows - 1) * pitch + k) * x.element_size() <= b or b + out.numel() * out.element_size() <= a


def _result(who: str, x: torch.Tensor, pitch: int, rows: int, n: int, mode: int, out_f32: bool, out: Optional[torch.Tensor]) -> torch.Tensor:
    """The result [rows, n] (SWIGLU: [rows, n / 2]): `out`, if that is one, or a new one."""
    if mode == SWIGLU:
        if n % 2:
            raise ValueError(f"{who}: gate and up rows are interleaved, {n} rows are no pairs")
        n //= 2
    if out is None:
        return x.new_empty(rows, n, dtype=_F32) if out_f32 else x.new_empty(rows, n)          # (a tuple costs the host 0.4 µs more)
    dtype = _F32 if out_f32 else x.dtype
    if out.dtype is not dtype or out.numel() != rows * n or not out.is_contiguous() or out.get_device() != x.get_device():
        raise ValueError(f"{who}: out is {dtype} with {rows} x {n} elements, contiguous, on {x.device} (got {out.dtype}, {tuple(out.shape)}, {out.device})")
    if not _apart(x, pitch, x.shape[0], x.shape[1], out):
        raise ValueError(f"{who}: out overlaps x, which is read while results are written")
    return out


def linear_int8(x: torch.Tensor, w: Int8Weight, *, norm_w: Optional[torch.Tensor] = None, eps: float = 1e-5, residual: Optional[torch.Tensor] = None, mode: int = PLAIN,
                out_f32: bool = False, out: Optional[torch.Tensor] = None, resident: bool = False) -> torch.Tensor:
    """`kernels.linear` with 8-bit weights: [M, N] (SWIGLU: [M, N / 2]) in x's type, or fp32, from x [..., K] (bf16, fp16 or fp32), any M >= 0 and any N.

    The rows of x, normed first where norm_w is given, become int8 values and a scale each (`quantize_rows`), and y[m, n] = s_m s_n Σ q_mk q_nk.  mode: PLAIN; RESIDUAL adds
    `residual` (of the result's type and size; `out` may be it); SWIGLU gives silu(y[2j]) · y[2j + 1] of interleaved rows, where silu(y) is 0 from exp(-y) = 2^126 on (y below -87.3: it is less than 2^-119
    there); RELU2 relu(y)².  `resident`: w is a parameter that no kernel
    directly before the call writes; it may then be read ahead of those."""
    who = "linear_int8"
    if w.__class__ is not Int8Weight or w.experts:
        raise ValueError(f"{who}: w is an Int8Weight of one matrix")
    dev, k, n = x.get_device(), w.k, w.n
    x, M, pitch = _take(who, x, k)
    if dev != w.dev:
        raise ValueError(f"{who}: x on {x.device}, weights on {w.device}")
    if norm_w is not None:
        _gain(who, norm_w, x, k)
    out = _result(who, x, pitch, M, n, mode, out_f32, out)
    if residual is not None:
        if mode != RESIDUAL:
            raise ValueError(f"{who}: a residual in mode {mode}")
        if residual.dtype is not out.dtype or residual.numel() != M * n or not residual.is_contiguous() or residual.get_device() != dev:
            raise ValueError(f"{who}: residual is {out.dtype} with {M} x {n} elements, contiguous, on {x.device} (got {residual.dtype}, {tuple(residual.shape)}, {residual.device})")
        if residual.data_ptr() != out.data_ptr() and not _apart(residual, n, M, n, out):
            raise ValueError(f"{who}: out overlaps a residual that it is not")
    elif mode not in (PLAIN, SWIGLU, RELU2):
        raise ValueError(f"{who}: mode {mode} without a residual")
    if dev < 0:
        q, s = _rows_ref(_norm_ref(x, norm_w, eps))
        y = (q.double() @ w.values.double().t()).float() * s[:, None] * w.scales
        return out.copy_(_finish_ref(y, residual, mode, out.dtype).view(out.shape))
    _here(dev, who)
    if M:
        _few(who, M)
        held, sms = w._held
        L = _lib.lib()
        need = L.jl_linear_int8_scratch_bytes(M, n, k)
        # (held until both launches are issued: another thread of this stream would be given what is let go of here, and the library runs without the interpreter's lock)
        room = x.new_empty(need, dtype=torch.uint8) if need else None
        rc = L.jl_linear_int8(x.data_ptr(), TYPES[x.dtype], M, k, pitch, *held, 0 if norm_w is None else norm_w.data_ptr(), eps, 0 if residual is None else residual.data_ptr(),
                              out.data_ptr(), TYPES[out.dtype], mode, 0 if room is None else room.data_ptr(), need, resident, sms, _stream())
        if rc:
            _lib.check(rc, "jl_linear_int8")
    return out


def expert_order(idx: torch.Tensor, E: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(pos int32 [M·top], rows int32 [M·top], offsets int32 [E + 1]) of the pairs idx int32 [M, top] ordered by expert, with nothing between experts: the row of
    every pair (-1 for a choice that is no expert's), the token of every row (-1 behind the last), the first row of every expert and, last, how many rows there are.
    What `expert_linear_int8` takes.  An expert's pairs are in any order among themselves, on CUDA another one from call to call: `pos` is where each went."""
    who = "expert_order"
    if idx.dtype is not torch.int32 or idx.dim() != 2 or idx.shape[1] < 1 or not idx.is_contiguous() or E < 1:
        raise ValueError(f"{who}: choices are int32 [M, top], contiguous, at least one a token, of at least one expert (got {idx.dtype}, {tuple(idx.shape)}, {E} experts)")
    M, top = idx.shape
    if not idx.is_cuda:
        flat = idx.reshape(-1).long()
        key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
        order = torch.argsort(key, stable=True)
        count = torch.bincount(key, minlength=E + 1)
        used = int(count[:E].sum())
        pos = torch.full((M * top,), -1, dtype=torch.int32)
        pos[order[:used]] = torch.arange(used, dtype=torch.int32)
        rows = torch.where(torch.arange(M * top) < used, order // max(top, 1), torch.full_like(order, -1)).to(torch.int32)
        return pos, rows, torch.cat([torch.zeros(1, dtype=torch.int64), count[:E].cumsum(0)]).to(torch.int32)
    _here(idx.get_device(), who)
    pos = idx.new_empty(M * top)
    rows = idx.new_empty(M * top)
    offsets = idx.new_empty(E + 1)
    _lib.check(_lib.lib().jl_moe_order(idx.data_ptr(), M, top, E, pos.data_ptr(), rows.data_ptr(), offsets.data_ptr(), _stream()), "jl_moe_order")
    return pos, rows, offsets


def expert_linear_int8(x: torch.Tensor, w: Int8Weight, offsets: torch.Tensor, *, rows: Optional[torch.Tensor] = None, mode: int = PLAIN, out_f32: bool = False,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The layers of a mixture of experts with 8-bit weights [E, N, K]: rows ordered by expert, as many of each as there are, against that expert's weights.

    Row t of the result, offsets[e] <= t < offsets[e + 1] (int32 [E + 1], rising, on the device), is expert e's product with row rows[t] of x [M, K] (int32 [T]; an index
    that x does not have is a row of zeros), without `rows` with row t (T = M): [T, N] (SWIGLU: [T, N / 2]) in x's type, or fp32.  Rows in front of offsets[0] and from
    offsets[E] on are left as they were.  `expert_order` gives rows and offsets of a router's choice.  Scales, sums and modes (PLAIN, SWIGLU, RELU2) as in `linear_int8`."""
    who = "expert_linear_int8"
    if w.__class__ is not Int8Weight or not 1 <= w.experts <= MAX_EXPERTS:
        raise ValueError(f"{who}: w is an Int8Weight of 1 to {MAX_EXPERTS} experts")
    if mode not in (PLAIN, SWIGLU, RELU2):
        raise ValueError(f"{who}: mode {mode}")
    dev, k = x.get_device(), w.k
    x, M, pitch = _take(who, x, k)
    if dev != w.dev:
        raise ValueError(f"{who}: x on {x.device}, weights on {w.device}")
    for t, name in ((offsets, "offsets"), (rows, "rows")):
        if t is not None and (t.dtype is not _I32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != dev):
            raise ValueError(f"{who}: {name} is int32, one dimension, contiguous, on {x.device} (got {t.dtype}, {tuple(t.shape)}, {t.device})")
    if offsets.numel() != w.experts + 1:
        raise ValueError(f"{who}: {offsets.numel()} offsets for {w.experts} experts")
    T = M if rows is None else rows.numel()
    out = _result(who, x, pitch, T, w.n, mode, out_f32, out)
    if dev < 0:
        flat = out.view(T, w.n // 2 if mode == SWIGLU else w.n)
        q, s = _rows_ref(x)
        if rows is not None:
            there = ((rows >= 0) & (rows < M))
            at = rows.long().clamp(0, max(M - 1, 0))
            q = q[at] * there[:, None] if M else q.new_zeros((T, w.k))
            s = s[at].masked_fill(~there, 0.0) if M else s.new_zeros(T)              # (a product would keep the NaN of the row that stands in)
        ends = [min(max(int(v), 0), T) for v in offsets.tolist()]
        for e in range(w.experts):
            a, b = ends[e], ends[e + 1]
            if b > a:
                y = (q[a:b].double() @ w.values[e].double().t()).float() * s[a:b, None] * w.scales[e]
                flat[a:b] = _finish_ref(y, None, mode, out.dtype)
        return out
    _here(dev, who)
    if T:
        _few(who, max(M, T))
        held, sms = w._held
        L = _lib.lib()
        need = L.jl_experts_int8_scratch_bytes(T, w.n, k)
        room = x.new_empty(need, dtype=torch.uint8) if need else None                # (held, as in linear_int8)
        rc = L.jl_experts_int8(x.data_ptr(), TYPES[x.dtype], M, k, pitch, 0 if rows is None else rows.data_ptr(), T, offsets.data_ptr(), w.experts, *held, out.data_ptr(),
                               TYPES[out.dtype], mode, 0 if room is None else room.data_ptr(), need, sms, _stream())
        if rc:
            _lib.check(rc, "jl_experts_int8")
    return out


def choice_linear_int8(x: torch.Tensor, w: Int8Weight, choice: torch.Tensor, *, mode: int = PLAIN, out_f32: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`expert_linear_int8` for a decoding token or a few, without an order: [M·top, N] (SWIGLU: [M·top, N / 2]), row m·top + k is row m of x [M, K] against expert
    choice[m, k] (int32 [M, top], contiguous; zeros for a choice that is no expert's).  One launch; at most MAX_CHOICES rows of at most MAX_CHOICE_K numbers."""
    who = "choice_linear_int8"
    if w.__class__ is not Int8Weight or not 1 <= w.experts <= MAX_EXPERTS:
        raise ValueError(f"{who}: w is an Int8Weight of 1 to {MAX_EXPERTS} experts")
    if mode not in (PLAIN, SWIGLU, RELU2):
        raise ValueError(f"{who}: mode {mode}")
    dev, k = x.get_device(), w.k
    x, M, pitch = _take(who, x, k)
    if dev != w.dev:
        raise ValueError(f"{who}: x on {x.device}, weights on {w.device}")
    if choice.dtype is not _I32 or choice.dim() != 2 or choice.shape[0] != M or choice.shape[1] < 1 or not choice.is_contiguous() or choice.get_device() != dev:
        raise ValueError(f"{who}: choices are int32 [{M}, top], contiguous, on {x.device} (got {choice.dtype}, {tuple(choice.shape)}, {choice.device})")
    top = choice.shape[1]
    if M * top > MAX_CHOICES or k > MAX_CHOICE_K:
        raise ValueError(f"{who}: {M} x {top} rows of {k} numbers (at most {MAX_CHOICES} of {MAX_CHOICE_K}; more go through expert_order)")
    out = _result(who, x, pitch, M * top, w.n, mode, out_f32, out)
    if dev < 0:
        flat = out.view(M * top, w.n // 2 if mode == SWIGLU else w.n)
        q, s = _rows_ref(x)
        for i, e in enumerate(choice.reshape(-1).tolist()):
            m = i // top
            y = (q[m].double() @ w.values[e].double().t()).float() * s[m] * w.scales[e] if 0 <= e < w.experts else torch.zeros(w.n)
            flat[i] = _finish_ref(y, None, mode, out.dtype)
        return out
    _here(dev, who)
    if M:
        held, sms = w._held
        rc = _lib.lib().jl_choice_int8(x.data_ptr(), TYPES[x.dtype], M, k, pitch, choice.data_ptr(), top, w.experts, *held, out.data_ptr(), TYPES[out.dtype], mode, sms, _stream())
        if rc:
            _lib.check(rc, "jl_choice_int8")
    return out
