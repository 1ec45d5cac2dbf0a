"""The RMS norm of rows and its backward pass against the definition in 64 bits (needs an MI355X).

Tolerances, u = 2^-24: a row's sum of squares over d terms is off by at most (d/64 + 8) u relative (a lane's share in a chain,
then a tree), r by half of that and a few roundings: er = (d/64 + 16) u.  y: three more roundings.  dx: the sum of a x is off by
er sum |a x|, so dx by r (8 u + er) |a| + |x| r^3 (2 er + er) mean |a x|.  dg: a chain over at most `rows` rows, its terms off
by er.  Outputs are rounded once: half a step (2^-8 |y| for bf16, u |y| for fp32)."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd._lib import AdnError, ADN_E_CAPACITY, ADN_E_INVALID
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def make(rows, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 13 + d)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    size = torch.pow(10.0, 4 * torch.rand((rows, 1), device="cuda", generator=g) - 2)
    return (rnd(rows, d) * size).to(dtype), rnd(rows, d).to(dtype), rnd(d) * 0.3 + 1


def reference(x, dy, gain, eps, dtype):
    rows, d = x.shape
    step = 2.0 ** -8 if dtype == BF16 else U
    er = (d / 64 + 16) * U
    X, D = x.double(), dy.double()
    g = torch.ones(d, device="cuda", dtype=torch.float64) if gain is None else gain.double()
    r = 1 / torch.sqrt((X * X).mean(1, keepdim=True) + eps)
    a = D * g
    ref = dict(y=X * r * g, dx=r * (a - X * r * r * (a * X).mean(1, keepdim=True)), dg=(D * X * r).sum(0))
    mag = (a * X).abs().mean(1, keepdim=True)
    tol = dict(y=(er + 4 * U) * ref["y"].abs() + step * ref["y"].abs(),
               dx=r * (8 * U + er) * a.abs() + 3 * er * X.abs() * r ** 3 * mag + 8 * U * X.abs() * r ** 3 * mag + step * ref["dx"].abs(),
               dg=(er + (rows + 8) * U) * (D * X * r).abs().sum(0) + U * ref["dg"].abs())
    return ref, tol


def run(be, x, dy, gain, eps, dx=True, dg=True):
    out = dict(y=torch.full_like(x, 7.0))
    if dx:
        out["dx"] = torch.full_like(x, 7.0)
    if dg:
        out["dg"] = torch.full((x.shape[1],), 7.0, device="cuda")
    torch.cuda.synchronize()
    be.rms_norm_async(x, out["y"], gain=gain, eps=eps)
    be.rms_norm_backward_async(x, dy, gain=gain, eps=eps, outputs={k: v for k, v in out.items() if k != "y"})
    be.synchronize()
    return out


def check(out, ref, tol):
    for k, v in out.items():
        err = (v.double() - ref[k]).abs()
        bad = ~(err <= tol[k] + 1e-300)
        assert not bad.any(), f"{k}: {int(bad.sum())} beyond the tolerance, worst {float(err[bad].max())} at {torch.nonzero(bad)[0].tolist()}"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 64), (5, 63), (4, 65), (7, 128), (2, 257), (24, 512), (600, 512), (33, 513),
                                    (9, 1000), (6, 1024), (130, 1025), (5, 2047), (3000, 2048), (4, 2049), (3, 4096), (700, 5001),
                                    (2, 8192), (2049, 96), (16385, 8)])
def test_against_definition(be, rows, d, dtype):
    log(f"norm {rows} x {d} {dtype}")
    x, dy, gain = make(rows, d, dtype)
    gain = None if rows % 5 == 0 else gain
    check(run(be, x, dy, gain, 1e-5), *reference(x, dy, gain, 1e-5, dtype))


@pytest.mark.parametrize("eps", [0.0, 1e-5, 3.0])
def test_eps_and_rows_of_zeros(be, eps):
    x, dy, gain = make(9, 100, F32)
    if eps:
        x[4] = 0
    check(run(be, x, dy, gain, eps), *reference(x, dy, gain, eps, F32))


@pytest.mark.parametrize("dx,dg", [(True, False), (False, True)])
def test_outputs_apart(be, dx, dg):
    x, dy, gain = make(77, 320, F32)
    both = run(be, x, dy, gain, 1e-5)
    one = run(be, x, dy, gain, 1e-5, dx, dg)
    for k, v in one.items():
        assert torch.equal(v, both[k])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("offset,extra", [(1, 3), (8, 8), (0, 1)])
def test_strides_and_alignment(be, offset, extra, dtype):
    """Results of rows at a stride within the tolerance, nothing written between them."""
    rows, d = 37, 200
    x, dy, gain = make(rows, d, dtype)

    def spaced(t):
        store = torch.full((offset + rows * (d + extra),), 5.0, device="cuda", dtype=t.dtype)
        v = store[offset:].view(rows, d + extra)[:, :d]
        v.copy_(t)
        return v, store
    xs, dys = spaced(x)[0], spaced(dy)[0]
    y, ys = spaced(torch.zeros_like(x))
    dx, dxs = spaced(torch.zeros_like(x))
    dg = torch.zeros(d, device="cuda")
    torch.cuda.synchronize()
    be.rms_norm_async(xs, y, gain=gain)
    be.rms_norm_backward_async(xs, dys, gain=gain, outputs=dict(dx=dx, dg=dg))
    be.synchronize()
    check(dict(y=y, dx=dx, dg=dg), *reference(x, dy, gain, 1e-5, dtype))
    for store in (ys, dxs):
        gaps = store[offset:].view(rows, d + extra)[:, d:]
        assert torch.equal(gaps, torch.full_like(gaps, 5.0)) and (store[:offset] == 5.0).all()


def test_bad_rows_stay_their_own(be):
    x, dy, gain = make(50, 130, F32)
    clean = run(be, x, dy, gain, 1e-5)
    x[3, 2], x[8, 1] = float("nan"), float("inf")
    out = run(be, x, dy, gain, 1e-5)
    ok = torch.ones(50, dtype=torch.bool, device="cuda")
    ok[[3, 8]] = False
    assert torch.equal(out["y"][ok], clean["y"][ok]) and torch.equal(out["dx"][ok], clean["dx"][ok])
    assert torch.isnan(out["y"][3]).all()


def test_empty_batch(be):
    e = torch.empty((0, 70), device="cuda")
    dg = torch.full((70,), 7.0, device="cuda")
    be.rms_norm_async(e, torch.empty_like(e))
    be.rms_norm_backward_async(e, e, outputs=dict(dx=torch.empty_like(e), dg=dg))
    be.rms_norm_backward_async(e, e, outputs=dict(dx=torch.empty_like(e)))
    be.synchronize()
    assert (dg == 0).all()


def test_gradients_against_differences(be):
    """Central differences of sum(c y) along random directions, formed from the framework's own y.  With c and the direction of
    order one, an element of y is off by its tolerance, and a third derivative of at most 16 |c| a row per unit step."""
    rows, d, h = 20, 96, 2.0 ** -6
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, d), device="cuda", generator=g)
    c = torch.randn((rows, d), device="cuda", generator=g)
    gain = torch.rand(d, device="cuda", generator=g) + 0.5
    out = run(be, x, c, gain, 1e-5)
    _, tol = reference(x, c, gain, 1e-5, F32)
    for which, grad in (("x", "dx"), ("gain", "dg")):
        u = torch.randn(x.shape if which == "x" else gain.shape, device="cuda", generator=g)
        u = u / u.norm()
        val = []
        for sgn in (1, -1):
            y = torch.empty_like(x)
            xs, gs = (x + sgn * h * u, gain) if which == "x" else (x, gain + sgn * h * u)
            torch.cuda.synchronize()
            be.rms_norm_async(xs, y, gain=gs)
            be.synchronize()
            val.append((y.double() * c.double()).sum())
        diff, got = float((val[0] - val[1]) / (2 * h)), float((out[grad].double() * u.double()).sum())
        # inputs x +- h u are themselves rounded: U |x| a component, through |dx| <= r |a|
        slack = float((tol["y"] * c.double().abs()).sum()) / h + 16 * h * h + 4 * U / h * float((out["dx"].double().abs() * x.double().abs()).sum())
        assert abs(diff - got) <= slack, (which, diff, got, slack)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_same_bits_again_and_in_a_graph(dtype):
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    x, dy, gain = make(900, 256, dtype)
    out = run(b, x, dy, gain, 1e-5)
    ref = {k: v.clone() for k, v in out.items()}
    again = run(b, x, dy, gain, 1e-5)
    assert all(torch.equal(again[k], ref[k]) for k in ref)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        b.rms_norm_async(x, out["y"], gain=gain)
        b.rms_norm_backward_async(x, dy, gain=gain, outputs=dict(dx=out["dx"], dg=out["dg"]))
    bx, bdy, bgain = make(3000, 2048, dtype)
    for rep in range(3):
        for v in out.values():
            v.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], ref[k]) for k in ref), rep
        run(b, bx, bdy, bgain, 1e-5)
    b.close()


def test_capture_before_the_workspace_is_there():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    x, dy, gain = make(30, 64, F32)
    dg = torch.zeros(64, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(AdnError) as ei:
            b.rms_norm_backward_async(x, dy, gain=gain, outputs=dict(dg=dg))
        dg.zero_()
    assert ei.value.code == ADN_E_CAPACITY
    b.close()


def test_refusals(be):
    x, dy, gain = make(8, 64, F32)
    y = torch.empty_like(x)

    def refused(match, f):
        with pytest.raises(AdnError, match=match) as ei:
            f()
        assert ei.value.code == ADN_E_INVALID
    refused("expected", lambda: be.rms_norm_async(x.half(), y.half()))
    refused("other matrices", lambda: be.rms_norm_async(x, y.bfloat16()))
    refused("shape", lambda: be.rms_norm_async(x, y[:, :60]))
    refused("context's GPU", lambda: be.rms_norm_async(x.cpu(), y))
    refused("gain", lambda: be.rms_norm_async(x, y, gain=gain[:60]))
    refused("eps", lambda: be.rms_norm_async(x, y, eps=-1.0))
    refused("eps", lambda: be.rms_norm_async(x, y, eps=float("nan")))
    refused("stride", lambda: be.rms_norm_async(x[:1].expand(8, 64), y))
    refused("d must be", lambda: be.rms_norm_async(torch.zeros((1, 8193), device="cuda"), torch.zeros((1, 8193), device="cuda")))
    many = torch.zeros(((1 << 24) + 1, 1), device="cuda")
    refused("number of rows", lambda: be.rms_norm_async(many, torch.empty_like(many)))
    refused("no output", lambda: be.rms_norm_backward_async(x, dy, outputs={}))
    refused("unknown", lambda: be.rms_norm_backward_async(x, dy, outputs=dict(dgain=gain)))
    refused("shape", lambda: be.rms_norm_backward_async(x, dy[:4], outputs=dict(dx=y)))
    be.synchronize()
