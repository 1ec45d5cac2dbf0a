"""Lists that come and go: what they hold on the device, with calls in flight, and with captured ones (needs an MI355X)."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend
from test_gpu_adamw import List, cfg_of, log

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def free():
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


def test_closed_lists_hold_no_memory(be):
    """A thousand lists one after another, each of 50 KB of tables and more: 16 MB at most, as one or two of them."""
    lst, norm = List([4 << 20, 100], 32), torch.zeros(1, device="cuda")
    keep = None
    for k in range(1000):
        opt = lst.optimizer(be)
        if k % 100 == 0:
            opt.grad_norm_async(norm)
        opt.close()
        if k == 0:
            be.synchronize()
            keep = free()
    be.synchronize()
    assert keep - free() < 16 << 20


@pytest.mark.parametrize("bits", [32, 8])
def test_lists_in_the_place_of_others(be, bits):
    """Each of several sizes, made behind others that were closed, steps as the definition says."""
    for k, sizes in enumerate([[5000], [3, 70000, 40], [300] * 300, [1], [], [2000, 2000], [5000], [100000], [17] * 900]):
        log(f"list {bits} {k}")
        lst = List(sizes, bits, seed=k)
        opt = lst.optimizer(be)
        cfg, before = cfg_of(lst), lst.host()
        torch.cuda.synchronize()
        opt.step_async(lr=1e-3)
        opt.close()  # with the step still in flight
        other = List([777, 5], bits, seed=k)
        oc, ob, second = cfg_of(other), other.host(), other.optimizer(be)
        second.step_async(lr=1e-3)
        be.synchronize()
        lst.check(before, cfg), other.check(ob, oc)
        second.close()


def test_a_captured_list_keeps_its_tables(be):
    """Its handle is closed and lists of its size are made and used before the graph is replayed."""
    a, b = List([5000, 300], 32), List([5000, 300], 32)
    oa, ob = a.optimizer(be), b.optimizer(be)
    na, nb, lr = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.full((1,), 1e-3, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(s.cuda_stream)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            oa.grad_norm_async(na)
            oa.step_async(lr=lr, grad_norm=na, max_norm=0.5)
        oa.close()
        for k in range(3):
            c = List([5000, 300], 32, seed=k)
            oc = c.optimizer(be)
            cfg, before = cfg_of(c), c.host()
            oc.step_async(lr=1e-3)
            be.synchronize()
            c.check(before, cfg)
            oc.close()
            with torch.cuda.stream(s):
                g.replay()
            torch.cuda.synchronize()
            ob.grad_norm_async(nb)
            ob.step_async(lr=lr, grad_norm=nb, max_norm=0.5)
            be.synchronize()
            assert torch.equal(na, nb) and int(a.step) == int(b.step)
            for x, y in zip(a.p + a.m + a.v, b.p + b.m + b.v):
                assert torch.equal(x, y)
        del g
    finally:
        torch.cuda.synchronize()
        be.set_stream(None)


def test_a_list_closed_behind_many_steps(be):
    """Some milliseconds of steps in flight when the handle goes and others take their tables in its place: all of the steps are its own."""
    n, steps = 8 << 20, 100
    g = torch.randn(n, device="cuda")
    got = []
    for kept in (True, False):
        p, step = torch.zeros(n, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
        m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        q, h = torch.ones(n - 5000, device="cuda"), torch.ones(n - 5000, device="cuda")
        torch.cuda.synchronize()
        opt = be.adamw([p], [g], m=[m], v=[v], step=step)
        for _ in range(steps):
            opt.step_async(lr=1e-3)
        if not kept:
            opt.close()
        r = be.adamw([q], [h], m=[torch.zeros_like(q)], v=[torch.zeros_like(q)], step=torch.zeros_like(step))
        torch.cuda.synchronize()
        r.step_async(lr=1e-3)
        be.synchronize()
        got.append([p, m, v, step, q, r.m[0], r.v[0]])
        opt.close(), r.close()
    assert int(got[1][3]) == steps
    assert all(torch.equal(a, b) for a, b in zip(*got))
