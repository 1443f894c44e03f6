"""The kernels of 8-bit integer layers against 64 bits."""
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


def _values(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def _weight(*shape, seed=0):
    I, _ = _ops()
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    return I.Int8Weight(_values(*shape, seed=seed), torch.rand(shape[:-1], generator=g, device=DEV) * 1e-2 + 1e-4)


def _same_rows(got, x):
    q, s = O.rows(x.reshape(-1, x.shape[-1]))
    assert torch.equal(got[0].reshape(q.shape).double(), q)
    assert torch.equal(got[1].reshape(-1), s)


def _check(got, off, want):
    err = (got.double() - want).abs()
    assert bool((err <= off).all()), f"off by {(err / off.clamp(min=1e-300)).max().item():.3g} of the bound, at {(err > off).nonzero()[:3].tolist()}"


# --------------------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 16), (33, 64), (9, 100), (7, 504), (8, 512), (65, 1001), (2, 2040), (17, 2048), (4, 2056), (3, 4096), (2, 4097), (5, 8192),
                                 (3, 11008), (4, 14336), (2, 16384), (2, 28672), (1, 32776), (1, 70001)])
def test_rows(dtype, M, K):
    I, _ = _ops()
    x = _randn(M, K, seed=K, dtype=dtype, scale=3.0)
    _same_rows(I.quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,K", [(593, 8), (1001, 64), (2003, 128), (700, 16), (601, 104), (5000, 24), (602, 40), (593, 1), (1003, 7), (701, 45), (2001, 113), (599, 57), (601, 2047), (600, 4090), (3, 26683), (5, 32761), (2, 32770)])
def test_rows_of_many_lengths(dtype, M, K):
    I, _ = _ops()
    x = _randn(M, K, seed=K, dtype=dtype, scale=3.0)
    if M > 100:
        x[5], x[77, K // 2], x[78, 0], x[-1, -1] = 0, float("nan"), float("-inf"), float("inf")
        x[6] *= 1e-30 if dtype is not HF else 1e-6
    q, s = I.quantize_rows(x)
    fine = torch.isfinite(x).all(1)
    _same_rows((q[fine], s[fine]), x[fine])
    assert not q[~fine].any() and bool(s[~fine].isnan().all())
    g = _randn(K, seed=1, dtype=dtype)
    a, b = I.quantize_rows(x[fine], norm_w=g)
    xd = x[fine].double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g.double()
    amax = h.abs().amax(-1, keepdim=True)
    t = torch.where(amax > 0, 127.0 * h / amax, torch.zeros_like(h))
    near = (t - t.floor() - 0.5).abs() < 127.0 * 8 * O.U
    assert bool(((a.double() - t.round()).abs() <= near).all())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [64, 333, 4096])
def test_rows_on_the_middle_of_two_values(dtype, K):
    """Quotients on and next to k + 1/2: amax 127 and 254, elements on halves and one step of the type beside them."""
    I, _ = _ops()
    g = torch.Generator(device=DEV).manual_seed(5)
    rows = []
    for amax in (127.0, 254.0, 63.5, 1.0, 0.984375, 127.0 * 2 ** -14):
        k = torch.randint(-127, 127, (K,), generator=g, device=DEV).double()
        x = ((k + 0.5) * amax / 127.0).to(dtype)
        one = torch.finfo(dtype).eps * x.abs().double()
        move = torch.randint(-1, 2, (K,), generator=g, device=DEV).double()
        x = (x.double() + move * one).to(dtype).clamp(-amax, amax)
        x[K // 2] = -amax
        rows.append(x)
    x = torch.stack(rows)
    _same_rows(I.quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [24, 1000, 4096])
def test_rows_of_extreme_sizes(dtype, K):
    """Rows of zeros, of the type's smallest numbers, of its largest."""
    I, _ = _ops()
    x = _randn(7, K, seed=1).double()
    t = torch.finfo(dtype)
    x[0] = 0
    x[1] *= 0
    x[1, 3] = t.smallest_normal * 2.0 ** -5          # a subnormal alone
    x[2] *= t.smallest_normal
    x[3] = x[3] / x[3].abs().max() * t.max
    x[4] = x[4] / x[4].abs().max() * t.smallest_normal * 4
    x[5] = x[5].abs() + 1e-3
    x = x.to(dtype)
    _same_rows(I.quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K", [40, 333, 4096])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_that_are_not_numbers(dtype, K, bad):
    I, _ = _ops()
    x = _randn(3, K, seed=2, dtype=dtype)
    x[1, K - 3] = bad
    q, s = I.quantize_rows(x)
    assert torch.isnan(s[1]) and not q[1].any()
    keep = torch.tensor([0, 2], device=DEV)
    _same_rows((q[keep], s[keep]), x[keep])
    w = _weight(9, K)
    y = I.linear_int8(x, w)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[keep]).all()


def test_rows_of_other_layouts():
    I, _ = _ops()
    big = _randn(9, 3000, seed=3, dtype=BF)
    for x in (big[:, :2048], big[:, 3:1003], big[::2, 8:1032], big[4:5, 1:2], big.view(3, 3, 3000)):
        _same_rows(I.quantize_rows(x), x)
    q, s = torch.zeros(9, 3000, dtype=torch.int8, device=DEV), torch.zeros(9, device=DEV)
    got = I.quantize_rows(big, out=(q, s))
    assert got[0] is q and got[1] is s
    _same_rows(got, big)
    q, s = I.quantize_rows(big[:0])
    assert q.shape == (0, 3000) and s.shape == (0,)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,K", [(3, 64), (2, 100), (5, 4096), (1, 14336), (2, 40000)])
def test_rows_behind_a_norm(dtype, M, K):
    """The ratio of an element to the row's largest is off by four roundings and the quotient by two: values may differ by one where the quotient in 64 bits lies that near the
    middle of two."""
    I, _ = _ops()
    x, g = _randn(M, K, seed=4, dtype=dtype, scale=2.0), _randn(K, seed=6, dtype=dtype)
    q, s = I.quantize_rows(x, norm_w=g, eps=1e-5)
    xd = x.double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g.double()
    amax = h.abs().amax(-1, keepdim=True)
    t = 127.0 * h / amax
    near = (t - t.floor() - 0.5).abs() < 127.0 * 8 * O.U
    off = (q.double() - t.round()).abs()
    assert bool((off <= near).all())
    # the mean: chains of at most 160 additions of one thread and 13 between threads, under a root; then six roundings
    assert bool(((s.double() / (amax[:, 0] / 127.0) - 1).abs() <= (0.5 * 173 + 8) * O.U).all())


# --------------------------------------------------------------------------- linear layers
SIZES = [(1, 1, 1), (1, 8, 16), (2, 17, 3), (1, 4096, 4096), (3, 130, 127), (4, 1000, 128), (5, 6144, 512), (8, 64, 1001), (9, 100, 4096), (16, 2048, 2048), (17, 250, 640), (33, 4096, 1024),
         (64, 129, 2048), (100, 28672, 256), (128, 512, 4096), (129, 1000, 1000), (200, 4096, 4096), (256, 260, 14336), (257, 1024, 512), (333, 6144, 384), (600, 130, 2064), (1025, 640, 1111),
         (2048, 2048, 2048), (7, 4096, 14336), (48, 1024, 8192), (600, 1, 64), (700, 7, 100), (1030, 2, 8), (513, 300, 1), (300, 512, 2048),
         (512, 1024, 4096), (3, 8, 131072), (140, 20000, 256), (8, 2048, 2048), (2, 30000, 1000)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear(M, N, K, dtype):
    I, K_ = _ops()
    x, w = _randn(M, K, seed=M, dtype=dtype), _weight(N, K, seed=N)
    q, s = O.rows(x)
    y = O.products(q, s, w.values, w.scales)
    off, want = O.bound(y, dtype)
    for resident in (False, True):
        _check(I.linear_int8(x, w, resident=resident), off, want)
    r = _randn(M, N, seed=9, dtype=dtype)
    off, want = O.bound(y, dtype, residual=r)
    _check(I.linear_int8(x, w, residual=r, mode=K_.RESIDUAL), off, want)
    if N % 2 == 0:
        off, want = O.bound_gated(y, dtype)
        _check(I.linear_int8(x, w, mode=K_.SWIGLU), off, want)


@pytest.mark.parametrize("M,N,K", [(1, 512, 256), (6, 100, 72), (40, 136, 200), (300, 258, 640)])
def test_linear_of_other_types(M, N, K):
    I, K_ = _ops()
    x, w = _randn(M, K, seed=M, dtype=HF), _weight(N, K, seed=N)
    y = O.products(*O.rows(x), w.values, w.scales)
    off, want = O.bound(y, HF)
    _check(I.linear_int8(x, w), off, want)
    off, want = O.bound_gated(y, F32)
    _check(I.linear_int8(x.to(HF), w, mode=K_.SWIGLU, out_f32=True), off, want)
    xb = x.to(BF)
    y = O.products(*O.rows(xb), w.values, w.scales)
    off, want = O.bound(y, F32)
    got = I.linear_int8(xb, w, out_f32=True)
    assert got.dtype is F32
    _check(got, off, want)


@pytest.mark.parametrize("M", [1, 3, 8, 20, 300])
@pytest.mark.parametrize("N,K", [(96, 64), (250, 4096), (128, 1500)])
def test_linear_behind_a_norm(M, N, K):
    I, _ = _ops()
    x, g, w = _randn(M, K, seed=M, dtype=BF, scale=2.0), _randn(K, seed=7, dtype=BF), _weight(N, K, seed=N)
    xd = x.double()
    h = xd / (xd.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g.double()
    amax = h.abs().amax(-1, keepdim=True)
    t = 127.0 * h / amax
    near = ((t - t.floor() - 0.5).abs() < 127.0 * 8 * O.U).double()
    s = amax[:, 0] / 127.0
    y = O.products(t.round(), s, w.values, w.scales)
    extra = (near @ w.values.double().abs().t()) * s[:, None] * w.scales.double() + (0.5 * 173 + 8) * O.U * y.abs()
    off, want = O.bound(y, BF, extra=extra)
    _check(I.linear_int8(x, w, norm_w=g, eps=1e-5), off, want)


@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_largest_sums(M):
    """Every product 127 * 127, and the longest K: sums of 2.1e9 stay in 32 bits."""
    I, _ = _ops()
    K = I.MAX_K
    x = torch.ones(M, K, dtype=BF, device=DEV)
    x[-1] = -1
    v = torch.full((6, K), 127, dtype=torch.int8, device=DEV)
    v[1] = -127
    w = I.Int8Weight(v, torch.full((6,), 2.0 ** -9, device=DEV))
    y = O.products(*O.rows(x), v, w.scales)
    off, want = O.bound(y, F32)
    _check(I.linear_int8(x, w, out_f32=True), off, want)


@pytest.mark.parametrize("M", [2, 6, 24, 290])
def test_rows_do_not_meet(M):
    """Rows of zeros and rows that are not numbers leave their neighbours alone; the result of a row does not depend on the rows beside it."""
    I, _ = _ops()
    x, w = _randn(M, 512, seed=1, dtype=BF), _weight(300, 512)
    alone = I.linear_int8(x, w)
    x[0] = 0
    x[M // 2, 5] = float("nan")
    y = I.linear_int8(x, w)
    assert not y[0].any() and torch.isnan(y[M // 2]).all()
    keep = [i for i in range(M) if i not in (0, M // 2)]
    assert torch.equal(y[keep], alone[keep])


@pytest.mark.parametrize("M", [1, 5, 8, 48, 260])
def test_layouts_of_x_and_results(M):
    I, K_ = _ops()
    wide = _randn(M, 2000, seed=3, dtype=BF)
    w = _weight(260, 640)
    for x in (wide[:, 16:656], wide[:, 5:645]):
        y = O.products(*O.rows(x), w.values, w.scales)
        off, want = O.bound(y, BF)
        _check(I.linear_int8(x, w), off, want)
        room = torch.full((M * 260 + 8,), 7.0, dtype=BF, device=DEV)
        for at in (1, 4):                                            # results on and off their ordinary boundary, with room around them
            room.fill_(7.0)
            out = room[at:at + M * 260].view(M, 260)
            assert I.linear_int8(x, w, out=out) is out
            _check(out, off, want)
            assert bool((room[:at] == 7).all()) and bool((room[at + M * 260:] == 7).all())
        r = _randn(M, 260, seed=8, dtype=BF)
        off, want = O.bound(y, BF, residual=r)
        _check(I.linear_int8(x, w, residual=r, mode=K_.RESIDUAL, out=r), off, want)      # in place on the residual


def test_one_row_of_any_pitch_and_no_rows():
    I, K_ = _ops()
    w = _weight(64, 48)
    x = _randn(4, 100, seed=2, dtype=BF)[2:3, :48]
    off, want = O.bound(O.products(*O.rows(x), w.values, w.scales), BF)
    _check(I.linear_int8(x, w), off, want)
    assert I.linear_int8(x[:0], w).shape == (0, 64)
    assert I.linear_int8(x[:0], w, mode=K_.SWIGLU).shape == (0, 32)
    three = _randn(2, 3, 48, seed=4, dtype=BF)
    assert torch.equal(I.linear_int8(three, w), I.linear_int8(three.view(6, 48), w))


@pytest.mark.parametrize("M", [1, 6, 64, 300])
def test_linear_through_the_framework(M):
    """kernels.linear takes an Int8Weight as it takes a matrix."""
    I, K_ = _ops()
    x, w = _randn(M, 512, seed=M, dtype=BF), _weight(384, 512)
    g, r = _randn(512, seed=5, dtype=BF), _randn(M, 384, seed=6, dtype=BF)
    assert torch.equal(K_.linear(x, w), I.linear_int8(x, w))
    assert torch.equal(K_.linear(x, w, norm_w=g, eps=1e-6, mode=K_.SWIGLU), I.linear_int8(x, w, norm_w=g, eps=1e-6, mode=K_.SWIGLU))
    assert torch.equal(K_.linear(x, w, residual=r, mode=K_.RESIDUAL), I.linear_int8(x, w, residual=r, mode=K_.RESIDUAL))
    assert K_.linear(x, w, out_f32=True).dtype is F32


# --------------------------------------------------------------------------- experts
def _expert_case(counts, M, seed=0, lead=0, behind=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(counts) + lead + behind
    rows = torch.randint(0, M, (T,), generator=g, device=DEV, dtype=torch.int32)
    offsets = torch.tensor([lead] + counts).cumsum(0).to(torch.int32).to(DEV)
    return rows, offsets, T


def _expert_check(x, w, rows, offsets, T, mode, dtype, out):
    I, K_ = _ops()
    q, s = O.rows(x)
    ends = offsets.tolist()
    for e in range(w.experts):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        at = rows[a:b].long() if rows is not None else torch.arange(a, b, device=DEV)
        y = O.products(q[at], s[at], w.values[e], w.scales[e])
        off, want = O.bound_gated(y, dtype) if mode == K_.SWIGLU else O.bound(y, dtype)
        _check(out[a:b], off, want)
    assert bool((out[:ends[0]] == 3).all()) and bool((out[ends[-1]:] == 3).all())      # rows of no expert: as they were


COUNTS = [[1], [4, 0, 0, 3], [0, 0, 5], [16, 1, 15, 17, 0, 33], [1] * 40, [0] * 9 + [200], [130, 128, 127, 0, 1], [300, 5, 257, 256], [1000, 3, 900, 40], [7] * 100, [600, 700, 500]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}e{sum(c)}")
@pytest.mark.parametrize("N,K", [(256, 128), (130, 1001), (96, 520), (1024, 1024)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_experts(counts, N, K, dtype):
    I, K_ = _ops()
    M = 50
    x, w = _randn(M, K, seed=1, dtype=dtype), _weight(len(counts), N, K, seed=2)
    rows, offsets, T = _expert_case(counts, M, lead=2, behind=3)
    for mode in (K_.PLAIN, K_.SWIGLU):
        out = torch.full((T, N // 2 if mode == K_.SWIGLU else N), 3.0, dtype=dtype, device=DEV)
        assert I.expert_linear_int8(x, w, offsets, rows=rows, mode=mode, out=out) is out
        _expert_check(x, w, rows, offsets, T, mode, dtype, out)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("E", [1, 3, 32, 300, 1024])
@pytest.mark.parametrize("N,K", [(18, 40), (130, 1001), (256, 4096), (34, 16384)])
def test_few_pairs(N, K, E, dtype):
    """A token's experts and a few tokens': each row with its expert, wherever among the experts that is; some rows of none."""
    I, K_ = _ops()
    x, w = _randn(5, K, seed=1, dtype=dtype), _weight(E, N, K, seed=2)
    g = torch.Generator().manual_seed(E)
    for lead, pairs, behind in ((0, 1, 0), (1, 2, 0), (0, 4, 1), (2, 3, 3), (0, 8, 0), (0, 0, 3)):
        T = lead + pairs + behind
        counts = torch.bincount(torch.randint(0, E, (pairs,), generator=g), minlength=E)
        offsets = (lead + torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])).to(torch.int32).to(DEV)
        rows = torch.randint(0, 5, (T,), generator=g).to(torch.int32).to(DEV)
        for mode in (K_.PLAIN, K_.SWIGLU):
            out = torch.full((T, N // 2 if mode == K_.SWIGLU else N), 3.0, dtype=dtype, device=DEV)
            I.expert_linear_int8(x, w, offsets, rows=rows, mode=mode, out=out)
            _expert_check(x, w, rows, offsets, T, mode, dtype, out)
            again = torch.zeros(T + 30, out.shape[1], dtype=dtype, device=DEV)        # with rows behind them another kernel runs: the same bits
            I.expert_linear_int8(x, w, offsets, rows=torch.cat([rows, rows.new_zeros(30)]), mode=mode, out=again)
            assert torch.equal(again[lead:lead + pairs], out[lead:lead + pairs])
            none = I.expert_linear_int8(x[:0], w, offsets, rows=rows, mode=mode)[lead:lead + pairs]
            assert not none.any()
    strided = _randn(5, 2 * K + 1, seed=4, dtype=dtype)[:, 1:K + 1]                  # rows off any boundary
    offsets = torch.full((E + 1,), 5, dtype=torch.int32, device=DEV)
    offsets[0] = 0
    _expert_check(strided, w, None, offsets, 5, K_.PLAIN, dtype, I.expert_linear_int8(strided, w, offsets))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("E", [1, 3, 32, 1024])
@pytest.mark.parametrize("N,K", [(18, 40), (130, 1001), (256, 4096), (34, 16384)])
def test_choices_without_an_order(N, K, E, dtype):
    I, K_ = _ops()
    w = _weight(E, N, K, seed=2)
    g = torch.Generator().manual_seed(E)
    for M, top in ((1, 1), (1, 4), (2, 3), (8, 1), (1, 8), (0, 2)):
        x = _randn(M, K + 3, seed=M, dtype=dtype)[:, :K]
        choice = torch.randint(0, E, (M, top), generator=g).to(torch.int32)
        if M > 1:
            choice[1, 0] = -1 if top > 1 else E
        choice = choice.to(DEV)
        q, s = O.rows(x) if M else (None, None)
        pos, rows, offsets = I.expert_order(choice, E)
        for mode in (K_.PLAIN, K_.SWIGLU):
            for f32 in (False, True):
                out = I.choice_linear_int8(x, w, choice, mode=mode, out_f32=f32)
                assert out.dtype is (F32 if f32 else dtype) and tuple(out.shape) == (M * top, N // 2 if mode == K_.SWIGLU else N)
                for i, e in enumerate(choice.reshape(-1).tolist()):
                    if not 0 <= e < E:
                        assert not out[i].any()
                        continue
                    y = O.products(q[i // top:i // top + 1], s[i // top:i // top + 1], w.values[e], w.scales[e])
                    off, want = O.bound_gated(y, out.dtype) if mode == K_.SWIGLU else O.bound(y, out.dtype)
                    _check(out[i:i + 1], off, want)
                if M:
                    ordered = I.expert_linear_int8(x, w, offsets, rows=rows, mode=mode, out_f32=f32)      # the same bits
                    there = pos >= 0
                    assert torch.equal(out[there], ordered[pos[there].long()])


def test_experts_without_an_index_and_of_other_types():
    I, K_ = _ops()
    counts = [5, 0, 70, 30]
    for dtype, f32 in ((HF, False), (BF, True)):
        x, w = _randn(105, 264, seed=3, dtype=dtype), _weight(4, 120, 264)
        offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(DEV)
        out = I.expert_linear_int8(x, w, offsets, out_f32=f32)
        assert out.dtype is (F32 if f32 else dtype)
        _expert_check(x, w, None, offsets, 105, K_.PLAIN, out.dtype, out)


def test_an_index_that_is_not_there_is_zeros():
    I, K_ = _ops()
    x, w = _randn(6, 64, seed=1, dtype=BF), _weight(2, 32, 64)
    rows = torch.tensor([0, -1, 5, 6, 1 << 30, 2], dtype=torch.int32, device=DEV)
    offsets = torch.tensor([0, 4, 6], dtype=torch.int32, device=DEV)
    y = I.expert_linear_int8(x, w, offsets, rows=rows)
    z = I.expert_linear_int8(x, w, offsets, rows=rows.clamp(0, 5))
    there = torch.tensor([0, 2, 5], device=DEV)
    assert torch.equal(y[there], z[there]) and not y[[1, 3, 4]].any()


def test_offsets_beyond_the_rows_stay_inside():
    I, _ = _ops()
    x, w = _randn(20, 64, seed=1, dtype=BF), _weight(3, 32, 64)
    room = torch.full((40, 32), 3.0, dtype=BF, device=DEV)
    out = room[10:30]
    I.expert_linear_int8(x, w, torch.tensor([-5, 7, 1000, 2000], dtype=torch.int32, device=DEV), out=out)
    fine = I.expert_linear_int8(x, w, torch.tensor([0, 7, 20, 20], dtype=torch.int32, device=DEV))
    assert torch.equal(out, fine) and bool((room[:10] == 3).all()) and bool((room[30:] == 3).all())


def test_many_experts():
    I, K_ = _ops()
    E = I.MAX_EXPERTS
    counts = [(7 * e) % 5 for e in range(E)]
    x, w = _randn(64, 32, seed=1, dtype=BF), _weight(E, 16, 32)
    rows, offsets, T = _expert_case(counts, 64)
    out = I.expert_linear_int8(x, w, offsets, rows=rows)
    _expert_check(x, w, rows, offsets, T, K_.PLAIN, BF, out)


@pytest.mark.parametrize("M,top,E", [(1, 1, 1), (1, 4, 32), (3, 8, 8), (200, 2, 8), (1000, 4, 64), (5000, 4, 128), (17, 3, 1000)])
def test_order(M, top, E):
    I, _ = _ops()
    g = torch.Generator().manual_seed(M)
    idx = torch.stack([torch.randperm(E, generator=g)[:top] for _ in range(M)]).to(torch.int32)
    if M > 2:
        idx[1, 0], idx[2, -1] = -1, E + 5                         # choices that are no expert's
    pos, rows, offsets = (t.cpu() for t in I.expert_order(idx.to(DEV), E))
    flat = idx.reshape(-1)
    good = (flat >= 0) & (flat < E)
    assert torch.equal(offsets.long(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(flat[good].long(), minlength=E).cumsum(0)]))
    assert bool((pos[~good] == -1).all()) and pos[good].unique().numel() == int(good.sum())
    assert torch.equal(rows[pos[good].long()].long(), torch.arange(M * top)[good] // top)
    expert = torch.searchsorted(offsets.long(), pos[good].long(), right=True) - 1
    assert torch.equal(expert, flat[good].long())
    assert bool((rows[int(offsets[-1]):] == -1).all())


# --------------------------------------------------------------------------- together
@pytest.mark.parametrize("M", [1, 7, 60, 700])
def test_a_mixture_of_experts(M):
    """Router's choice -> order -> gate | up of every expert -> down -> weighted sum, against 64 bits with the stages' own values."""
    I, K_ = _ops()
    W, ff, E, top = 256, 192, 8, 3
    x = _randn(M, W, seed=1, dtype=BF)
    up, down = _weight(E, 2 * ff, W, seed=2), _weight(E, W, ff, seed=3)
    idx = _randn(M, E, seed=4).topk(top, -1).indices.to(torch.int32)
    wt = _randn(M, top, seed=5).abs()
    pos, rows, offsets = I.expert_order(idx, E)
    t = I.expert_linear_int8(x, up, offsets, rows=rows, mode=K_.SWIGLU)
    y = I.expert_linear_int8(t, down, offsets, out_f32=True)
    got = (y[pos.long()].view(M, top, W) * wt[..., None]).sum(1)
    q, s = O.rows(x)
    want = torch.zeros(M, W, dtype=torch.float64, device=DEV)
    off = torch.zeros_like(want)
    for c in range(top):
        for e in range(E):
            m = (idx[:, c] == e).nonzero()[:, 0]
            if not m.numel():
                continue
            p = pos.view(M, top)[m, c].long()
            b, h = O.bound_gated(O.products(q[m], s[m], up.values[e], up.scales[e]), BF)
            _check(t[p], b, h)
            b, z = O.bound(O.products(*O.rows(t[p]), down.values[e], down.scales[e]), F32)
            want[m] += wt[m, c, None].double() * z
            off[m] += wt[m, c, None].double() * (b + 4 * O.U * z.abs())
    _check(got, off, want)


@pytest.mark.parametrize("M", [1, 4, 30, 300])
def test_captured_and_replayed(M):
    I, K_ = _ops()
    x, w, w2 = _randn(M, 512, seed=1, dtype=BF), _weight(1024, 512), _weight(512, 512, seed=4)
    r = _randn(M, 512, seed=2, dtype=BF)

    def layer():
        return I.linear_int8(I.linear_int8(x, w, mode=K_.SWIGLU, resident=True), w2, residual=r, mode=K_.RESIDUAL, resident=True)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer()
    for seed in (5, 6):
        x.copy_(_randn(M, 512, seed=seed, dtype=BF))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, layer())


def test_two_streams_at_once():
    I, _ = _ops()
    w = _weight(2048, 1024)
    xs = [_randn(m, 1024, seed=m, dtype=BF) for m in (1, 40, 3, 300)]
    want = [I.linear_int8(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [None] * len(xs)
    for _ in range(5):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i] = I.linear_int8(x, w, resident=True)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("M", [1, 16, 200, 600])
def test_weights_quantised_directly_before(M):
    """The library's own kernel writes the weights, the product follows at once."""
    I, _ = _ops()
    x = _randn(M, 4096, seed=1, dtype=BF)
    for seed in range(4):
        w16 = _randn(4096, 4096, seed=seed, dtype=BF)
        y = I.linear_int8(x, I.Int8Weight.of(w16))
        q, s = O.rows(w16)
        off, want = O.bound(O.products(*O.rows(x), q, s), BF)
        _check(y, off, want)


def test_repeated_calls_give_the_same_bits():
    I, K_ = _ops()
    for M in (1, 5, 16, 64, 200, 600):
        x, w = _randn(M, 2048, seed=M, dtype=BF), _weight(1000, 2048)
        first = I.linear_int8(x, w, mode=K_.SWIGLU)
        for _ in range(3):
            assert torch.equal(I.linear_int8(x, w, mode=K_.SWIGLU), first)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,K", [(256, 512), (1000, 2048), (130, 72)])
def test_every_kernel_gives_a_row_the_same_bits(N, K, dtype):
    """Sums are exact and what follows them is one chain of fp32 operations: the rows beside it, and with them the kernel, change nothing."""
    I, K_ = _ops()
    x, w = _randn(700, K, seed=1, dtype=dtype), _weight(N, K)
    for mode in (K_.PLAIN, K_.SWIGLU):
        full = I.linear_int8(x, w, mode=mode)
        for M in (1, 2, 4, 8, 9, 16, 40, 64, 128, 130, 256, 300, 512, 600):
            assert torch.equal(I.linear_int8(x[:M], w, mode=mode), full[:M])
        e = I.Int8Weight(w.values[None], w.scales[None])
        for M in (1, 30, 700):
            off = torch.tensor([0, M], dtype=torch.int32, device=DEV)
            assert torch.equal(I.expert_linear_int8(x[:M], e, off, mode=mode), full[:M])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,N,K", [(1, 33, 64), (3, 2048, 512), (20, 130, 1001), (100, 4096, 2048), (300, 6144, 2080), (700, 514, 640), (9, 1, 8)])
def test_squared_relu(M, N, K, dtype):
    I, K_ = _ops()
    x, w = _randn(M, K, seed=M, dtype=dtype), _weight(N, K, seed=N)
    y = O.products(*O.rows(x), w.values, w.scales)
    off, want = O.bound_relu2(y, dtype)
    got = I.linear_int8(x, w, mode=I.RELU2)
    _check(got, off, want)
    assert torch.equal(K_.linear(x, w, mode=I.RELU2), got)
    e = I.Int8Weight(w.values[None], w.scales[None])
    assert torch.equal(I.expert_linear_int8(x, e, torch.tensor([0, M], dtype=torch.int32, device=DEV), mode=I.RELU2), got)
    assert torch.equal(I.choice_linear_int8(x[:1], e, torch.zeros(1, 3, dtype=torch.int32, device=DEV), mode=I.RELU2), got[:1].expand(3, -1))
    x[M // 2, K // 2] = float("nan")
    got = I.linear_int8(x, w, mode=I.RELU2)
    assert bool(got[M // 2].isnan().all()) and int(got.isnan().sum()) == N


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,K", [(200, 2500), (1000, 2056), (2100, 4100), (4096, 2048), (6200, 2064), (4500, 6400), (16380, 2080), (130, 70)])
def test_however_a_product_is_cut(N, K, dtype):
    """Pieces of rows and parts of K depend on the sizes; a row's results do not."""
    I, K_ = _ops()
    x, w, r = _randn(520, K, seed=3, dtype=dtype), _weight(N, K), _randn(520, N, seed=4, dtype=dtype)
    plain, more = I.linear_int8(x, w), I.linear_int8(x, w, mode=K_.RESIDUAL, residual=r)
    off, want = O.bound(O.products(*O.rows(x), w.values, w.scales), dtype)
    _check(plain, off, want)
    for M in (1, 2, 7, 16, 48, 64, 65, 80, 81, 97, 112, 128, 129, 144, 176, 177, 225, 256, 257, 336, 337, 384, 385, 449, 512):
        assert torch.equal(I.linear_int8(x[:M], w), plain[:M])
        assert torch.equal(I.linear_int8(x[:M], w, mode=K_.RESIDUAL, residual=r[:M]), more[:M])


@pytest.mark.parametrize("N,K", [(100, 4096), (163, 11374), (1000, 2056), (2048, 2048), (4608, 2100)])
def test_many_rows_of_few_features(N, K):
    I, K_ = _ops()
    x, w, r = _randn(1500, K, seed=3, dtype=BF), _weight(N, K), _randn(1500, N, seed=4, dtype=BF)
    off, want = O.bound(O.products(*O.rows(x), w.values, w.scales), BF, residual=r)
    for M in (513, 700, 1500):
        got = I.linear_int8(x[:M], w, mode=K_.RESIDUAL, residual=r[:M])
        _check(got, off[:M], want[:M])
        assert torch.equal(got, torch.cat([I.linear_int8(x[i:min(i + 60, M)], w, mode=K_.RESIDUAL, residual=r[i:min(i + 60, M)]) for i in range(0, M, 60)]))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,N,K", [(700, 1001, 200), (1030, 2502, 72), (601, 1034, 1000), (300, 35, 256), (1000, 4, 64), (530, 259, 130)])
def test_results_off_the_boundary(M, N, K, dtype):
    """Rows of results and residuals that begin anywhere: odd ones, and those on four bytes."""
    I, K_ = _ops()
    x, w, r = _randn(M, K, seed=3, dtype=dtype), _weight(N, K), _randn(M, N, seed=4, dtype=dtype)
    y = O.products(*O.rows(x), w.values, w.scales)
    room = torch.full((M * N + 9,), 3.0, dtype=dtype, device=DEV)
    for shift in (1, 2):
        out = room[shift:shift + M * N].view(M, N)
        off, want = O.bound(y, dtype, residual=r)
        I.linear_int8(x, w, mode=K_.RESIDUAL, residual=r, out=out)
        _check(out, off, want)
        out.copy_(r)
        I.linear_int8(x, w, mode=K_.RESIDUAL, residual=out, out=out)                  # in place
        _check(out, off, want)
        off, want = O.bound(y, dtype)
        I.linear_int8(x, w, out=out)
        _check(out, off, want)
        assert bool((room[:shift] == 3).all()) and bool((room[shift + M * N:] == 3).all())
        room.fill_(3.0)
    if N % 2 == 0:
        off, want = O.bound_gated(y, dtype)
        _check(I.linear_int8(x, w, mode=K_.SWIGLU), off, want)


@pytest.mark.parametrize("counts,N", [([600, 700, 500], 1024), ([900, 0, 1100], 2050)])
def test_gathered_rows_of_pairs(counts, N):
    """Many rows of few tokens: every token is brought to 8 bits once and gathered; indices that are not there give zeros, rows of no expert stay."""
    I, K_ = _ops()
    M, K, T = 70, 520, sum(counts) + 9
    x, w = _randn(M, K, seed=1, dtype=BF), _weight(len(counts), N, K, seed=2)
    rows = torch.randint(0, M, (T,), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(3))
    offsets = torch.tensor([4] + counts).cumsum(0).to(torch.int32).to(DEV)
    bad = torch.tensor([5, 300, 617, 1500], device=DEV)
    for mode in (K_.PLAIN, K_.SWIGLU):
        out = torch.full((T, N // 2 if mode == K_.SWIGLU else N), 3.0, dtype=BF, device=DEV)
        I.expert_linear_int8(x, w, offsets, rows=rows, mode=mode, out=out)
        _expert_check(x, w, rows, offsets, T, mode, BF, out)
        gone = rows.clone()
        gone[bad] = torch.tensor([-1, M, -(1 << 31), (1 << 31) - 1], dtype=torch.int32, device=DEV)
        got = I.expert_linear_int8(x, w, offsets, rows=gone, mode=mode)
        keep = torch.ones(T, dtype=torch.bool, device=DEV)
        keep[bad], keep[:4], keep[-5:] = False, False, False
        assert not got[bad].any() and torch.equal(got[keep], out[keep])


def test_many_experts_of_many_rows():
    I, K_ = _ops()
    E = 300
    counts = [(37 * e) % 401 for e in range(E)]
    x, w = _randn(64, 32, seed=1, dtype=BF), _weight(E, 32, 32)
    rows, offsets, T = _expert_case(counts, 64, lead=1, behind=2)
    out = torch.full((T, 32), 3.0, dtype=BF, device=DEV)
    I.expert_linear_int8(x, w, offsets, rows=rows, out=out)
    q, s = O.rows(x)
    ids = torch.repeat_interleave(torch.arange(E, device=DEV), torch.tensor(counts, device=DEV))
    m = rows[1:T - 2].long()
    y = torch.einsum("tk,tnk->tn", q[m], w.values.double()[ids]) * s.double()[m, None] * w.scales.double()[ids]
    _check(out[1:T - 2], *O.bound(y, BF))
    assert bool((out[0] == 3).all()) and bool((out[T - 2:] == 3).all())


def test_an_order_written_directly_before():
    """Offsets and rows of a router's choice, at once used: they are read ahead of the wait for the activations."""
    I, _ = _ops()
    x, w = _randn(600, 256, seed=1, dtype=BF), _weight(16, 640, 256)
    for M in (3, 40, 600):
        for seed in range(4):
            idx = _randn(M, 16, seed=seed).topk(4, -1).indices.to(torch.int32)
            pos, rows, offsets = I.expert_order(idx, 16)
            y = I.expert_linear_int8(x[:M], w, offsets, rows=rows)[pos.long()]
            torch.cuda.synchronize()
            for e in range(16):
                at = (idx.reshape(-1) == e).nonzero()[:, 0]
                if at.numel():
                    one = I.Int8Weight(w.values[e], w.scales[e])
                    assert torch.equal(y[at], I.linear_int8(x[at // 4].contiguous(), one))


# --------------------------------------------------------------------------- places beyond 2^31
def test_rows_beyond_2_31():
    I, _ = _ops()
    M, K = 140000, 16384
    x = torch.empty(M, K, dtype=BF, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    q, s = I.quantize_rows(x)
    at = torch.tensor([0, 131071, 131072, 139999], device=DEV)
    _same_rows((q[at], s[at]), x[at])


@pytest.mark.parametrize("M,N,K", [(70000, 32768, 64), (120, 20_000_000, 112)])
def test_results_and_weights_beyond_2_31(M, N, K):
    I, _ = _ops()
    x = _randn(M, K, seed=1, dtype=BF)
    w = I.Int8Weight(_values(N, K), torch.full((N,), 1e-3, device=DEV))
    y = I.linear_int8(x, w)
    rows, cols = torch.tensor([0, M // 2, M - 1], device=DEV), torch.tensor([0, 1, N // 2, N - 2, N - 1], device=DEV)
    off, want = O.bound(O.products(*O.rows(x[rows]), w.values[cols], w.scales[cols]), BF)
    _check(y[rows][:, cols], off, want)


def test_experts_beyond_2_31():
    I, K_ = _ops()
    E, N, K = 40, 30000, 2048
    x = _randn(64, K, seed=1, dtype=BF)
    w = I.Int8Weight(_values(E, N, K), torch.full((E, N), 1e-3, device=DEV))
    rows, offsets, T = _expert_case([3] * E, 64)
    y = I.expert_linear_int8(x, w, offsets, rows=rows)
    q, s = O.rows(x)
    for e in (0, 35, 39):
        m = rows[3 * e:3 * e + 3].long()
        _check(y[3 * e:3 * e + 3], *O.bound(O.products(q[m], s[m], w.values[e], w.scales[e]), BF))
