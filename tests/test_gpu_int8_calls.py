"""8-bit layers called by several threads, and with an allocator that gives memory back in the stream's order."""
import os
import subprocess
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_llama_b200.ops import int8 as I                                        # noqa: E402
from jax_llama_b200.ops import kernels as K                                     # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16)


def _weight(*shape, seed=0):
    return I.Int8Weight.of(_randn(*shape, seed=seed))


@pytest.mark.parametrize("M", [1, 40, 300, 900])
def test_threads_of_one_stream(M):
    """The default stream is every thread's: workspaces and results of calls that are issued between one another's launches."""
    w, e = _weight(1024, 512), _weight(8, 256, 512, seed=1)
    xs = [_randn(M, 512, seed=s) for s in range(6)]
    orders = [I.expert_order(torch.randint(0, 8, (M, 2), generator=torch.Generator().manual_seed(s)).to(torch.int32).cuda(), 8) for s in range(6)]
    g = _randn(512, seed=9)

    def work(i):
        pos, rows, offsets = orders[i]
        return I.linear_int8(xs[i], w, norm_w=g, mode=K.SWIGLU), I.expert_linear_int8(xs[i], e, offsets, rows=rows), I.linear_int8(xs[i], w)

    want = [work(i) for i in range(6)]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(6)

    def thread(i):
        start.wait()
        got = [work(i) for _ in range(40)]
        for a in got:
            if not all(torch.equal(p, q) for p, q in zip(a, want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_memory_given_back_in_the_streams_order():
    """torch's cudaMallocAsync backend: what a call let go of ahead of its launches would be free, or another's, while they run."""
    code = """
import torch
from jax_llama_b200.ops import int8 as I
from tests import int8_oracle as O
g = torch.Generator(device='cuda').manual_seed(0)
w16 = torch.randn(512, 1024, generator=g, device='cuda').bfloat16()
w, q = I.Int8Weight.of(w16), O.rows(w16)
for M in (40, 300, 2000):
    x = torch.randn(M, 1024, generator=g, device='cuda').bfloat16()
    off, want = O.bound(O.products(*O.rows(x), *q), torch.bfloat16)
    for _ in range(5):
        assert bool(((I.linear_int8(x, w).double() - want).abs() <= off).all())
    e = I.Int8Weight(w.values[None], w.scales[None])
    ends = torch.tensor([0, M], dtype=torch.int32, device='cuda')
    for _ in range(5):
        assert bool(((I.expert_linear_int8(x, e, ends).double() - want).abs() <= off).all())
print('same', torch.cuda.get_allocator_backend())
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT, env=dict(os.environ, PYTORCH_CUDA_ALLOC_CONF="backend:cudaMallocAsync"))
    assert r.returncode == 0 and "same cudaMallocAsync" in r.stdout, r.stderr[-1500:]
