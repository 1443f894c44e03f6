"""How the functions of 8-bit layers call the library: on the CPU, with a stand-in for its entry points."""
import copy
import io
import weakref

import pytest
import torch

from jax_llama_b200.ops import int8 as I


class OnGpu(torch.Tensor):
    """A tensor of the CPU that says it is on cuda:0, and remembers the workspaces that were made from it."""

    made = []

    is_cuda = True

    def get_device(self):
        return 0

    def new_empty(self, *args, **kw):
        t = super().new_empty(*args, **kw)
        if t.dtype is torch.uint8:
            OnGpu.made.append(weakref.ref(t))
        return t


class Library:
    """Entry points that look at their arguments and launch nothing."""

    def __init__(self):
        self.calls = []

    def jl_linear_int8_scratch_bytes(self, M, N, K):
        return 1024

    def jl_experts_int8_scratch_bytes(self, T, N, K):
        return 2048

    def _called(self, name, args):
        held = [t() for t in OnGpu.made]
        assert len(held) == 1 and held[0] is not None, f"{name}: its workspace is gone"
        assert held[0].data_ptr() in args and held[0].numel() in args
        self.calls.append((name, args))
        return 0

    def jl_linear_int8(self, *args):
        return self._called("linear", args)

    def jl_experts_int8(self, *args):
        return self._called("experts", args)


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    OnGpu.made = []
    monkeypatch.setattr(I._lib, "lib", lambda: lib)
    monkeypatch.setattr(I, "_here", lambda dev, who: None)
    monkeypatch.setattr(I, "_stream", lambda: 0)
    return lib


def on_gpu(t):
    return t.as_subclass(OnGpu)


def weight(*shape):
    w = I.Int8Weight(torch.ones(shape, dtype=torch.int8), torch.ones(shape[:-1]))
    object.__setattr__(w, "dev", 0)
    return w


def test_the_workspace_of_a_layer_lives_until_the_call_is_over(library):
    I.linear_int8(on_gpu(torch.randn(300, 64)), weight(32, 64))
    assert [n for n, _ in library.calls] == ["linear"]


def test_the_workspace_of_experts_lives_until_the_call_is_over(library):
    x = on_gpu(torch.randn(30, 64))
    I.expert_linear_int8(x, weight(2, 32, 64), on_gpu(torch.tensor([0, 10, 30], dtype=torch.int32)))
    assert [n for n, _ in library.calls] == ["experts"]


def test_a_row_that_is_not_there_is_zeros_beside_rows_that_are_no_numbers():
    """An index that x does not have, where the rows that x does have hold NaN or infinities."""
    w = I.Int8Weight(torch.ones(2, 6, 16, dtype=torch.int8), torch.ones(2, 6))
    x = torch.full((3, 16), float("nan"))
    x[1] = 2.0
    x[2, 5] = float("inf")
    y = I.expert_linear_int8(x, w, torch.tensor([0, 3, 5], dtype=torch.int32), rows=torch.tensor([-1, 1, 3, 99, 0], dtype=torch.int32))
    assert not y[[0, 2, 3]].any() and torch.isfinite(y[1]).all() and torch.isnan(y[4]).all()


def test_rows_longer_than_they_may_be(monkeypatch):
    """A number of columns beyond 32 bits would reach the library cut short."""
    from jax_llama_b200.ops import _lib
    assert I.MAX_COLUMNS == 1 << 30
    monkeypatch.setattr(I, "MAX_COLUMNS", 7)
    with pytest.raises(ValueError, match="rows of 8 numbers"):
        I.quantize_rows(torch.zeros(3, 8))
    K = (1 << 30) + 8                                           # (refused by the library ahead of any use of the device)
    assert _lib.lib().jl_int8_rows(0, 0, 1, K, K, 0, 1, 0, 1e-5, 0, K, 0, 0) != 0


@pytest.mark.parametrize("M", [2, 128, 200, 3000])
def test_weights_through_the_framework_are_parameters_at_any_number_of_rows(library, M):
    """kernels.linear says that weights in 8 bits may be read ahead; linear_int8 reads them in turn unless it is told."""
    from jax_llama_b200.ops import kernels as K
    w = weight(32, 64)
    x = on_gpu(torch.randn(M, 64))
    assert "at any number of rows" in " ".join(K.linear.__doc__.split())
    for call, resident in ((lambda: K.linear(x, w), True), (lambda: I.linear_int8(x, w), False)):
        OnGpu.made = []
        call()
        assert library.calls[-1][1][-3] is resident


@pytest.mark.parametrize("shape", [(4, 16), (3, 6, 20)])
def test_copies_of_weights_have_their_own_addresses(shape):
    """What a call hands to the library are addresses: those of a copy, or of weights that were stored and loaded, are not the first one's."""
    w = I.Int8Weight.of(torch.randn(shape))
    room = io.BytesIO()
    torch.save(w, room)
    room.seek(0)
    for other in (copy.deepcopy(w), torch.load(room, weights_only=False)):
        assert torch.equal(other.values, w.values) and torch.equal(other.scales, w.scales) and (other.n, other.k, other.pitch, other.experts) == (w.n, w.k, w.pitch, w.experts)
        assert other.values.data_ptr() != w.values.data_ptr()
        assert other._held[0] == (other.values.data_ptr(), other.pitch, other.scales.data_ptr(), other.n)
        assert other.values.stride(-2) == other.pitch and other.values.data_ptr() % 16 == 0


def test_fields_of_weights_are_not_assigned():
    w = I.Int8Weight.of(torch.randn(4, 16))
    for name in ("values", "scales", "k", "_held"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name))
    w.values.zero_()                                            # (written into, they are what calls read)
    assert not I.linear_int8(torch.randn(2, 16), w).any()
