"""8-bit integer layers on the CPU: the statement of the operators, their refusals, the layout of weights."""
import pytest
import torch

from jax_llama_b200.ops import int8 as I
from jax_llama_b200.ops import kernels as K
from tests import int8_oracle as O


def _randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _weight(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return I.Int8Weight(torch.randint(-127, 128, shape, generator=g, dtype=torch.int8), torch.rand(shape[:-1], generator=g) * 1e-2 + 1e-4)


def _check(got, off, want):
    assert bool(((got.double() - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K_", [(1, 1), (3, 7), (5, 64), (4, 1001)])
def test_rows(dtype, M, K_):
    x = _randn(M, K_, seed=K_, dtype=dtype)
    q, s = I.quantize_rows(x)
    assert q.dtype is torch.int8 and s.dtype is torch.float32
    wq, ws = O.rows(x)
    assert torch.equal(q.double(), wq) and torch.equal(s, ws)
    back = q.double() * s.double()[:, None]
    # half a value of the row, and what rounding the scale moves the largest value by
    assert bool(((back - x.double()).abs() <= s.double()[:, None] * (0.5 + 128 * 2.0 ** -24)).all())


def test_rows_that_hold_nothing_or_no_numbers():
    x = _randn(4, 9)
    x[0], x[1, 3], x[2, 4] = 0, float("nan"), float("-inf")
    q, s = I.quantize_rows(x)
    assert s[0] == 0 and torch.isnan(s[1]) and torch.isnan(s[2]) and not q[:3].any() and q[3].abs().max() == 127
    x = torch.tensor([[127.0, 0.5, 1.5, -0.5, -1.5, 2.5, 126.5]])        # ties go to the even value
    assert I.quantize_rows(x)[0].tolist() == [[127, 0, 2, 0, -2, 2, 126]]


def test_rows_in_place_of_given_results_and_more_dimensions():
    x = _randn(2, 3, 8)
    q, s = I.quantize_rows(x)
    assert q.shape == (2, 3, 8) and s.shape == (2, 3)
    out = (torch.empty(6, 8, dtype=torch.int8), torch.empty(6))
    assert I.quantize_rows(x.view(6, 8), out=out)[0] is out[0] and torch.equal(out[0], q.view(6, 8))


@pytest.mark.parametrize("M,N,K_", [(1, 4, 8), (5, 6, 33), (17, 30, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(M, N, K_, dtype):
    x, w = _randn(M, K_, seed=M, dtype=dtype), _weight(N, K_, seed=N)
    y = O.products(*O.rows(x), w.values, w.scales)
    _check(I.linear_int8(x, w), *O.bound(y, dtype))
    r = _randn(M, N, seed=3, dtype=dtype)
    _check(I.linear_int8(x, w, residual=r, mode=K.RESIDUAL), *O.bound(y, dtype, residual=r))
    _check(I.linear_int8(x, w, mode=K.SWIGLU), *O.bound_gated(y, dtype))
    assert torch.equal(K.linear(x, w), I.linear_int8(x, w))
    out = torch.empty(M, N)
    assert I.linear_int8(x, w, out_f32=True, out=out) is out
    g = _randn(K_, seed=8, dtype=dtype)
    assert I.linear_int8(x, w, norm_w=g).shape == (M, N)


def test_weights_of_a_matrix():
    w16 = _randn(6, 20, dtype=torch.bfloat16)
    w = I.Int8Weight.of(w16)
    assert w.shape == (6, 20) and w.pitch == 32 and w.experts == 0 and w.nbytes == 6 * 24
    assert w.values.stride(0) == 32 and not w.values.as_strided((6, 12), (32, 1), w.values.storage_offset() + 20).any()
    step = w16.double().abs().amax(-1, keepdim=True) / 127
    assert bool(((w.float().double() - w16.double()).abs() <= step * (0.5 + 128 * 2.0 ** -23)).all())
    e = I.Int8Weight.of(_randn(3, 6, 16))
    assert e.experts == 3 and e.n == 6 and e.scales.shape == (3, 6) and e.pitch == 16
    v = torch.zeros(4, 64, dtype=torch.int8)
    assert I.Int8Weight(v, torch.ones(4)).values.data_ptr() == v.data_ptr()      # as they lie, where that is on the boundary


def test_experts():
    E, N, K_, M = 4, 6, 24, 9
    w, x = _weight(E, N, K_), _randn(M, K_, dtype=torch.bfloat16)
    rows = torch.tensor([0, 3, 8, -1, 2, 2, 99], dtype=torch.int32)
    offsets = torch.tensor([1, 3, 3, 6, 6], dtype=torch.int32)
    out = torch.full((7, N), 5.0, dtype=torch.bfloat16)
    assert I.expert_linear_int8(x, w, offsets, rows=rows, out=out) is out
    assert bool((out[0] == 5).all()) and bool((out[6] == 5).all()) and not out[3].any()
    q, s = O.rows(x)
    for t, e in ((1, 0), (2, 0), (4, 2), (5, 2)):
        m = rows[t:t + 1].long()
        _check(out[t:t + 1], *O.bound(O.products(q[m], s[m], w.values[e], w.scales[e]), torch.bfloat16))
    assert I.expert_linear_int8(x, w, torch.tensor([0, 2, 4, 6, 9], dtype=torch.int32), mode=K.SWIGLU).shape == (M, N // 2)


def test_order():
    idx = torch.tensor([[2, 0], [0, -1], [1, 2], [7, 0]], dtype=torch.int32)
    pos, rows, offsets = I.expert_order(idx, 3)
    assert offsets.tolist() == [0, 3, 4, 6]
    assert pos.tolist() == [4, 0, 1, -1, 3, 5, -1, 2] and rows.tolist() == [0, 1, 3, 2, 0, 2, -1, -1]


def test_a_layer_of_experts_together():
    """Order, gate | up, down, weighted sum: what every (token, choice) pair alone gives."""
    M, top, E, W, ff = 7, 2, 5, 16, 12
    x, up, down = _randn(M, W), _weight(E, 2 * ff, W, seed=1), _weight(E, W, ff, seed=2)
    idx = torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(m))[:top] for m in range(M)]).to(torch.int32)
    pos, rows, offsets = I.expert_order(idx, E)
    y = I.expert_linear_int8(I.expert_linear_int8(x, up, offsets, rows=rows, mode=K.SWIGLU), down, offsets)
    got = y[pos.long()].view(M, top, W)
    for m in range(M):
        for c in range(top):
            e = int(idx[m, c])
            one = [I.Int8Weight(w.values[e], w.scales[e]) for w in (up, down)]
            assert torch.equal(got[m, c], I.linear_int8(I.linear_int8(x[m:m + 1], one[0], mode=K.SWIGLU), one[1])[0])


def test_squared_relu():
    w, x = _weight(7, 32), _randn(5, 32)
    y = I.linear_int8(x, w)
    assert torch.equal(I.linear_int8(x, w, mode=I.RELU2), y.clamp(min=0).square())
    e = I.Int8Weight(w.values[None], w.scales[None])
    assert torch.equal(I.expert_linear_int8(x, e, torch.tensor([0, 5], dtype=torch.int32), mode=I.RELU2), y.clamp(min=0).square())
    with pytest.raises(ValueError):
        I.linear_int8(x, w, mode=4)


def test_choices_without_an_order():
    w, x = _weight(3, 6, 16), _randn(2, 16)
    choice = torch.tensor([[2, 0], [-1, 1]], dtype=torch.int32)
    pos, rows, offsets = I.expert_order(choice, 3)
    for mode in (K.PLAIN, K.SWIGLU):
        y = I.choice_linear_int8(x, w, choice, mode=mode)
        z = I.expert_linear_int8(x, w, offsets, rows=rows, mode=mode)
        assert torch.equal(y[[0, 1, 3]], z[pos[[0, 1, 3]].long()]) and not y[2].any()
    assert I.choice_linear_int8(x[:0], w, choice[:0], out_f32=True).shape == (0, 6)


def test_experts_without_rows():
    assert I.expert_linear_int8(_randn(0, 16), _weight(3, 6, 16), torch.zeros(4, dtype=torch.int32), mode=K.SWIGLU).shape == (0, 3)


# --------------------------------------------------------------------------- refusals
def test_refusals_of_rows():
    for x in (torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.float64), torch.zeros(()), torch.zeros(3, 0), torch.zeros(4, 3).t(), torch.zeros(2, 3, 4).transpose(0, 1),
              torch.zeros(1, 4).expand(3, 4), torch.zeros(12).as_strided((3, 4), (2, 1))):
        with pytest.raises(ValueError):
            I.quantize_rows(x)
    x = torch.zeros(3, 4)
    for out in ((torch.zeros(3, 4), torch.zeros(3)), (torch.zeros(3, 4, dtype=torch.int8), torch.zeros(4)), (torch.zeros(4, 3, dtype=torch.int8).t(), torch.zeros(3))):
        with pytest.raises(ValueError):
            I.quantize_rows(x, out=out)
    room = torch.zeros(64, dtype=torch.int8)
    with pytest.raises(ValueError):
        I.quantize_rows(room[:48].view(torch.float32).view(3, 4), out=(room[40:52].view(3, 4), torch.zeros(3)))
    for g in (torch.zeros(3), torch.zeros(4, dtype=torch.bfloat16), torch.zeros(8)[::2]):
        with pytest.raises(ValueError):
            I.quantize_rows(x, norm_w=g)


def test_more_rows_than_there_may_be(monkeypatch):
    monkeypatch.setattr(I, "MAX_ROWS", 2)
    with pytest.raises(ValueError):
        I.quantize_rows(torch.zeros(3, 4))
    with pytest.raises(ValueError):
        I.Int8Weight(torch.zeros(3, 16, dtype=torch.int8), torch.ones(3))


def test_refusals_of_weights():
    v = torch.zeros(4, 16, dtype=torch.int8)
    for a, b in ((v.float(), torch.ones(4)), (v, torch.ones(5)), (v, torch.ones(4, dtype=torch.bfloat16)), (v[0], torch.ones(())), (v[None, None], torch.ones(1, 1, 4)),
                 (v[:0], torch.ones(0)), (v[:, :0], torch.ones(4)), (torch.zeros(1, I.MAX_K + 1, dtype=torch.int8), torch.ones(1))):
        with pytest.raises(ValueError):
            I.Int8Weight(a, b)


def test_refusals_of_linear():
    w, x = _weight(6, 16), _randn(3, 16)
    bad = [dict(x=x.double()), dict(x=_randn(3, 15)), dict(x=_randn(16, 3).t()), dict(mode=7), dict(mode=K.RESIDUAL), dict(residual=_randn(3, 6)), dict(mode=K.RESIDUAL, residual=_randn(3, 5)),
           dict(mode=K.RESIDUAL, residual=_randn(3, 6, dtype=torch.bfloat16)), dict(mode=K.RESIDUAL, residual=_randn(6, 3).t()), dict(out=torch.empty(3, 6, dtype=torch.bfloat16)),
           dict(out=torch.empty(3, 7)), dict(out=torch.empty(6, 3).t()), dict(norm_w=_randn(15)), dict(w=_weight(2, 6, 16)), dict(w=torch.zeros(6, 16))]
    for kw in bad:
        with pytest.raises(ValueError):
            I.linear_int8(kw.pop("x", x), kw.pop("w", w), **kw)
    with pytest.raises(ValueError):
        I.linear_int8(x, _weight(5, 16), mode=K.SWIGLU)
    square = _weight(16, 16)
    room = _randn(64 + 3 * 16)
    for a, b in ((0, 0), (0, 16), (16, 0), (0, 47), (47, 0)):                  # results that share numbers with x, or with a residual that they are not
        with pytest.raises(ValueError):
            I.linear_int8(room[a:a + 48].view(3, 16), square, out=room[b:b + 48].view(3, 16))
        if a != b:
            with pytest.raises(ValueError):
                I.linear_int8(x, square, mode=K.RESIDUAL, residual=room[a:a + 48].view(3, 16), out=room[b:b + 48].view(3, 16))
    assert torch.equal(I.linear_int8(room[:48].view(3, 16), square, out=room[48:96].view(3, 16)), I.linear_int8(room[:48].view(3, 16), square))
    r = _randn(3, 16, seed=4)
    want = I.linear_int8(x, square, mode=K.RESIDUAL, residual=r)
    assert torch.equal(I.linear_int8(x, square, mode=K.RESIDUAL, residual=r, out=r), want)
    with pytest.raises(ValueError):
        K.linear(x, w, force="gemm")


def test_refusals_of_experts():
    w, x = _weight(2, 6, 16), _randn(3, 16)
    off = torch.tensor([0, 1, 3], dtype=torch.int32)
    bad = [dict(offsets=off.long()), dict(offsets=off[:2]), dict(offsets=torch.zeros(6, dtype=torch.int32)[::2]), dict(rows=torch.zeros(3, dtype=torch.int64)), dict(rows=torch.zeros(3, 1, dtype=torch.int32)),
           dict(mode=K.RESIDUAL), dict(w=_weight(6, 16)), dict(out=torch.empty(2, 6)), dict(x=_randn(3, 8))]
    for kw in bad:
        with pytest.raises(ValueError):
            I.expert_linear_int8(kw.pop("x", x), kw.pop("w", w), kw.pop("offsets", off), **kw)
    for idx, E in ((torch.zeros(3, 2), 4), (torch.zeros(3, dtype=torch.int32), 4), (torch.zeros(3, 2, dtype=torch.int32), 0), (torch.zeros(3, 0, dtype=torch.int32), 2),
                   (torch.zeros(2, 3, dtype=torch.int32).t(), 4)):
        with pytest.raises(ValueError):
            I.expert_order(idx, E)


def test_refusals_of_the_engine():
    from jax_llama_b200 import LLaMAConfig
    from jax_llama_b200.models.engine import B200Engine
    cfg = LLaMAConfig(vocab_size=64, hidden_size=32, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2, max_sequence_length=16)
    with pytest.raises(ValueError):
        B200Engine(cfg, torch.zeros(1), [], torch.zeros(1), torch.zeros(1), weights="int4")
    with pytest.raises(NotImplementedError):
        B200Engine(cfg, torch.zeros(1), [], torch.zeros(1), torch.zeros(1), weights="int8", tp=2)


def test_refusals_of_choices():
    w, x, choice = _weight(2, 6, 16), _randn(3, 16), torch.zeros(3, 2, dtype=torch.int32)
    bad = [dict(choice=choice.long()), dict(choice=choice[:2]), dict(choice=choice[:, 0]), dict(choice=choice[:, :0]), dict(choice=torch.zeros(2, 3, dtype=torch.int32).t()),
           dict(choice=torch.zeros(3, 3, dtype=torch.int32)), dict(mode=K.RESIDUAL), dict(w=_weight(6, 16)), dict(w=_weight(2, 5, 16), mode=K.SWIGLU), dict(out=torch.empty(5, 6)),
           dict(x=_randn(3, 8)), dict(w=_weight(2, 2, I.MAX_CHOICE_K + 1), x=_randn(3, I.MAX_CHOICE_K + 1))]
    for kw in bad:
        with pytest.raises(ValueError):
            I.choice_linear_int8(kw.pop("x", x), kw.pop("w", w), kw.pop("choice", choice), **kw)
