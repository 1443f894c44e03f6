"""Rows of 8-bit layers behind a norm: the same bits from every kernel, beside any rows, on any boundary."""
import pytest
import torch

from tests import int8_oracle as O

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def _ops():
    from jax_llama_b200.ops import int8 as I
    from jax_llama_b200.ops import kernels as K
    return I, K


def _randn(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _weight(*shape, seed=0):
    I, _ = _ops()
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    values = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
    return I.Int8Weight(values, torch.rand(shape[:-1], generator=g, device=DEV) * 1e-2 + 1e-4)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [1, 8, 45, 64, 113, 128, 500, 512, 1001, 2048, 2056, 4096, 4097, 8192, 11264, 14336, 16384, 16388, 20000, 32768, 40000])
def test_rows_have_the_same_bits_beside_any_rows(dtype, K):
    """Many rows, few, and one: 8 threads a row, a warp, 128, 256, rows in registers and rows read twice."""
    I, _ = _ops()
    x, g = _randn(700, K, seed=K, dtype=dtype, scale=2.0), _randn(K, seed=1, dtype=dtype)
    q, s = I.quantize_rows(x, norm_w=g)
    for a, b in ((0, 1), (3, 5), (100, 300), (0, 592), (7, 700)):
        p, r = I.quantize_rows(x[a:b], norm_w=g)
        assert torch.equal(p, q[a:b]) and torch.equal(r, s[a:b])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [16, 120, 512, 1000, 2048, 4096, 8184, 16384, 16400, 36000])
def test_rows_have_the_same_bits_on_any_boundary(dtype, K):
    """Rows whose first element is 0, 1, .. behind a 16-byte boundary, neighbours on different ones, and gains off the boundary."""
    I, _ = _ops()
    x, g = _randn(40, K, seed=K, dtype=dtype, scale=2.0), _randn(K, seed=1, dtype=dtype)
    q, s = I.quantize_rows(x, norm_w=g)
    for pitch, first in ((K + 1, 0), (K + 3, 2), (K + 8, 1), (K + 16 // x.element_size(), 3)):
        room = torch.full((40 * pitch + 8,), 99.0, dtype=dtype, device=DEV)
        y = room[first:first + 40 * pitch].view(40, pitch)[:, :K]
        y.copy_(x)
        p, r = I.quantize_rows(y, norm_w=g)
        assert torch.equal(p, q) and torch.equal(r, s)
    h = torch.empty(K + 1, dtype=dtype, device=DEV)[1:]
    h.copy_(g)
    p, r = I.quantize_rows(x, norm_w=h)
    assert torch.equal(p, q) and torch.equal(r, s)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("N,K", [(256, 512), (1000, 2048), (130, 72), (96, 1001), (2048, 4096), (64, 8192), (40, 16384), (48, 13001)])
def test_layers_have_the_same_bits_beside_any_rows(dtype, N, K):
    """One launch for few rows (a warp to eight a row), and the rows' own kernel ahead of products."""
    I, K_ = _ops()
    x, g, w = _randn(700, K, seed=2, dtype=dtype, scale=2.0), _randn(K, seed=3, dtype=dtype), _weight(N, K)
    for mode in (K_.PLAIN, K_.SWIGLU):
        full = I.linear_int8(x, w, norm_w=g, mode=mode)
        for M in (1, 2, 3, 4, 5, 8, 9, 40, 128, 300, 593):
            assert torch.equal(I.linear_int8(x[:M], w, norm_w=g, mode=mode), full[:M])
    q, s = I.quantize_rows(x, norm_w=g)
    off, want = O.bound(O.products(q, s, w.values, w.scales), dtype)
    assert bool(((I.linear_int8(x, w, norm_w=g).double() - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [7, 64, 1001, 4096, 16390, 40000])
@pytest.mark.parametrize("pitch", [0, 1])
def test_values_and_scales(dtype, K, pitch):
    """Against 64 bits.  A row's sum of squares is a chain of at most 8 additions in a piece, 3 of pieces 4096 apart and 12 of halves: its root is off by half of 24 roundings; with
    the mean's quotient and eps, the root, the reciprocal and two products the normed numbers are off by less than 12 + 6, so a value may be the neighbour where its quotient is within 127 * 40 of
    those of a middle (the row's largest is off as well, the quotient adds three), and the scale, of one number, by 18 and a rounding of its own."""
    I, _ = _ops()
    room = _randn(9, K + pitch, seed=K, dtype=dtype, scale=2.0)
    x, g = room[:, pitch:], _randn(K, seed=5, dtype=dtype)
    q, s = I.quantize_rows(x, norm_w=g, eps=1e-5)
    xd = x.double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g.double()
    amax = h.abs().amax(-1, keepdim=True)
    t = 127.0 * h / amax
    near = (t - t.floor() - 0.5).abs() < 127.0 * 40 * O.U
    assert bool(((q.double() - t.round()).abs() <= near).all())
    assert bool(((s.double() / (amax[:, 0] / 127.0) - 1).abs() <= 19 * O.U).all())


@pytest.mark.parametrize("K", [24, 1001, 4096, 20000])
def test_rows_that_hold_nothing_or_no_numbers(K):
    I, _ = _ops()
    x, g = _randn(6, K, dtype=BF), _randn(K, seed=1, dtype=BF)
    x[0], x[1, K // 2], x[2, K - 1] = 0, float("nan"), float("inf")
    q, s = I.quantize_rows(x, norm_w=g)
    assert s[0] == 0 and torch.isnan(s[1:3]).all() and not q[:3].any() and torch.isfinite(s[3:]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("K", [40, 1001, 8192, 20001, 40000])
@pytest.mark.parametrize("n", [9, 700])
def test_chosen_rows_behind_a_norm(dtype, K, n):
    """The library's own entry point takes an index with gains: rows in any order, and zeros for those that are not there."""
    from jax_llama_b200.ops import _lib
    I, _ = _ops()
    x, g = _randn(9, K, seed=K, dtype=dtype), _randn(K, seed=1, dtype=dtype)
    index = torch.randint(-2, 12, (n,), generator=torch.Generator().manual_seed(K)).to(torch.int32)
    index[:3] = torch.tensor([-1, 9, 4])
    q, s = torch.full((n, K), 5, dtype=torch.int8, device=DEV), torch.full((n,), 5.0, device=DEV)
    rows = index.to(DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.lib().jl_int8_rows(x.data_ptr(), I.TYPES[dtype], 9, K, K, rows.data_ptr(), n, g.data_ptr(), 1e-5, q.data_ptr(), K, s.data_ptr(), stream) == 0
    p, r = I.quantize_rows(x, norm_w=g)
    there = (index >= 0) & (index < 9)
    at = index[there].long().to(DEV)
    there = there.to(DEV)
    assert torch.equal(q[there], p[at]) and torch.equal(s[there], r[at])
    assert not q[~there].any() and not s[~there].any()
