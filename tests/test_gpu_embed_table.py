"""The scaled embedding lookup and the table's gradient against the definition in 64 bits (needs an MI355X).

Tolerances, u = 2^-24: the lookup is one product, then one rounding to the type (half a step: 2^-8 for bf16, u for fp32).  A
gradient row is a fp32 sum of m rows in a fixed order, at most m additions: m u sum |dout|, times the scale, rounded once."""
import numpy as np
import pytest
import torch

from aideen_amd import synth
from aideen_amd._lib import AdnError, ADN_E_CAPACITY, ADN_E_INVALID, ADN_E_NO_WEIGHTS
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


def tokens_of(kind, n, V, seed=0):
    r = np.random.default_rng(seed + n + V)
    if kind == "zipf":
        t = np.minimum(r.zipf(1.3, n) - 1, V - 1)
    elif kind == "one":
        t = np.full(n, V // 2)
    elif kind == "runs":  # rows whose counts end at, before and after the chunks' edges
        t = np.repeat(np.arange(V), 31 + np.arange(V) % 4)[:n]
        t = np.concatenate([t, r.integers(0, V, n - len(t))])
    elif kind == "ends":
        t = np.where(r.random(n) < 0.5, 0, V - 1)
    else:
        t = r.integers(0, V, n)
    t = t.astype(np.int32)
    if kind == "padded":
        t[r.random(n) < 0.3] = -1
    return torch.from_numpy(t).cuda()


def make(n, d, V, dtype, kind="uniform", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n * 3 + d)
    return (torch.randn((V, d), device="cuda", generator=g).to(dtype), torch.randn((n, d), device="cuda", generator=g).to(dtype),
            tokens_of(kind, n, V, seed))


def reference(table, dout, toks, scale, dtype):
    step = 2.0 ** -8 if dtype == BF16 else U
    V, d = table.shape
    keep = torch.nonzero((toks >= 0) & (toks < V))[:, 0]
    t = toks[keep].long()
    out = torch.zeros((len(toks), d), device="cuda", dtype=torch.float64)
    out[keep] = table.double()[t] * scale
    tg = torch.zeros((V, d), dtype=torch.float64, device="cuda").index_add_(0, t, dout.double()[keep]) * scale
    mag = torch.zeros((V, d), dtype=torch.float64, device="cuda").index_add_(0, t, dout.double()[keep].abs()) * abs(scale)
    m = torch.bincount(t, minlength=V).double()[:, None]
    # the scale itself is a fp32 number
    return dict(out=out, dtable=tg), dict(out=(step + 2 * U) * out.abs(), dtable=(m + 2) * U * mag + step * tg.abs())


def run(be, table, dout, toks, scale):
    out = dict(out=torch.full_like(dout, 7.0), dtable=torch.full_like(table, 7.0))
    torch.cuda.synchronize()
    be.embed_lookup_async(toks, out["out"], table=table, scale=scale)
    be.embed_grad_async(dout, toks, out["dtable"], scale=scale)
    be.synchronize()
    return out


def check(out, ref, tol):
    for k, v in out.items():
        err = (v.double() - ref[k]).abs()
        bad = ~(err <= tol[k] + 1e-300)
        assert not bad.any(), f"{k}: {int(bad.sum())} beyond the tolerance, worst {float(err[bad].max())} at {torch.nonzero(bad)[0].tolist()}"


CASES = [(1, 1, 1, "uniform"), (1, 64, 50257, "uniform"), (2, 7, 3, "uniform"), (31, 64, 10, "zipf"), (32, 65, 10, "one"), (33, 128, 2, "ends"),
         (64, 192, 65, "uniform"), (65, 33, 1000, "padded"), (255, 512, 300, "zipf"), (257, 100, 256, "uniform"), (2047, 64, 255, "zipf"),
         (2049, 64, 257, "zipf"), (4097, 96, 70000, "uniform"), (5000, 64, 100, "runs"), (8192, 72, 50257, "zipf"), (9001, 48, 65, "uniform"),
         (20000, 32, 7, "one"), (33000, 16, 65535, "zipf"), (33000, 16, 65536, "padded"), (70001, 8, 300, "zipf"), (300, 2048, 500, "zipf"),
         (100, 8192, 20, "zipf"), (3000, 4, 1 << 24, "uniform"), (2048, 64, 50257, "one"), (16384, 64, 1024, "padded"), (1023, 64, 40, "zipf"),
         (1024, 130, 50257, "padded"), (1025, 64, 40, "zipf"), (1000, 64, 3, "one"), (4095, 64, 700, "zipf"), (4096, 48, 50257, "padded"), (4096, 2048, 9, "one"), (513, 64, 20, "zipf"),
         (140001, 8, 300, "zipf"), (131072, 8, 2000, "ends"),
         (131073, 8, 70001, "padded"), (2952, 2048, 512, "zipf"), (2000, 520, 9, "zipf"), (100, 1000, 6, "uniform"), (500, 8192, 31, "zipf")]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,d,V,kind", CASES)
def test_against_definition(be, n, d, V, kind, dtype):
    log(f"embedding {n} x {d} of {V} {kind} {dtype}")
    table, dout, toks = make(n, d, V, dtype, kind)
    scale = 1.0 if n % 2 else 8.0 / 3.0
    scale = float(np.float32(scale))
    check(run(be, table, dout, toks, scale), *reference(table, dout, toks, scale, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [137, 4300])
@pytest.mark.parametrize("offset,extra", [(1, 3), (8, 8), (0, 1)])
def test_strides_and_alignment(be, offset, extra, n, dtype):
    d, V = 200, 90
    table, dout, toks = make(n, d, V, dtype, "zipf")
    tight = run(be, table, dout, toks, 0.5)

    def spaced(t):
        r = t.shape[0]
        store = torch.full((offset + r * (d + extra),), 5.0, device="cuda", dtype=t.dtype)
        v = store[offset:].view(r, d + extra)[:, :d]
        v.copy_(t)
        return v, store
    out, os_ = spaced(torch.zeros_like(dout))
    dt, dts = spaced(torch.zeros_like(table))
    torch.cuda.synchronize()
    be.embed_lookup_async(toks, out, table=spaced(table)[0], scale=0.5)
    be.embed_grad_async(spaced(dout)[0], toks, dt, scale=0.5)
    be.synchronize()
    assert torch.equal(out, tight["out"]) and torch.equal(dt, tight["dtable"])
    for store, r in ((os_, n), (dts, V)):
        gaps = store[offset:].view(r, d + extra)[:, d:]
        assert torch.equal(gaps, torch.full_like(gaps, 5.0)) and (store[:offset] == 5.0).all()


@pytest.mark.parametrize("n", [50, 5000])
def test_positions_without_a_token_are_not_read(be, n):
    table, dout, toks = make(n, 64, 200, F32, "padded")
    dout[toks < 0] = float("nan")
    out = run(be, table, dout, toks, 1.0)
    assert torch.isfinite(out["out"]).all() and torch.isfinite(out["dtable"]).all()
    toks[:] = -1
    out = run(be, table, dout, toks, 1.0)
    assert (out["out"] == 0).all() and (out["dtable"] == 0).all()


def test_bad_values_stay_in_their_rows(be):
    table, dout, toks = make(300, 64, 50, F32, "zipf")
    dout[7, 3] = float("inf")
    table[int(toks[9])] = float("nan")
    out = run(be, table, dout, toks, 1.0)
    t = int(toks[7])
    assert torch.isinf(out["dtable"][t, 3]) and int((~torch.isfinite(out["dtable"])).sum()) == 1
    bad = torch.isnan(out["out"]).all(1)
    assert torch.equal(bad, toks == toks[9])


@pytest.mark.parametrize("n", [40, 4000, 4500])
def test_token_beyond_the_table_is_reported(be, n):
    table, dout, toks = make(n, 64, 50, F32)
    toks[5] = 50
    toks[6] = 2147483647
    for f in (lambda o: be.embed_lookup_async(toks, o["out"], table=table), lambda o: be.embed_grad_async(dout, toks, o["dtable"])):
        out = dict(out=torch.full_like(dout, 7.0), dtable=torch.full_like(table, 7.0))
        torch.cuda.synchronize()
        f(out)
        with pytest.raises(AdnError, match="outside"):
            be.synchronize()
        ref, tol = reference(table, dout, toks, 1.0, F32)
        for k, v in out.items():
            if not (v == 7.0).all():
                check({k: v}, ref, tol)
    be.synchronize()


def test_empty_batch(be):
    table, _, _ = make(1, 64, 300, F32)
    e, t = torch.empty((0, 64), device="cuda"), torch.empty(0, device="cuda", dtype=torch.int32)
    dt = torch.full_like(table, 7.0)
    be.embed_lookup_async(t, torch.empty_like(e), table=table)
    be.embed_grad_async(e, t, dt)
    be.synchronize()
    assert (dt == 0).all()


def test_uploaded_table():
    mc = synth.ModelConfig(d=128, H=2, V=515, N=1, flags=0)
    w = synth.make_token_sensitive_weights(mc, seed=3)
    b = GpuDeqBackend(mc, 1, 8)
    toks = tokens_of("padded", 100, 515)
    out = torch.full((100, 128), 7.0, device="cuda")
    with pytest.raises(AdnError) as ei:
        b.embed_lookup_async(toks, out)
    assert ei.value.code == ADN_E_NO_WEIGHTS
    b.upload_weights(w)
    torch.cuda.synchronize()
    b.embed_lookup_async(toks, out, scale=2.0)
    b.synchronize()
    ref = torch.from_numpy(w["embed"]).cuda()[toks.clamp(min=0).long()] * 2.0
    ref[toks < 0] = 0
    assert torch.equal(out, ref)
    b.close()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,V", [(300, 700), (12000, 50257)])
def test_same_bits_again_and_in_a_graph(n, V, dtype):
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    table, dout, toks = make(n, 64, V, dtype, "zipf")
    out = run(b, table, dout, toks, 1.5)
    ref = {k: v.clone() for k, v in out.items()}
    again = run(b, table, dout, toks, 1.5)
    assert all(torch.equal(again[k], ref[k]) for k in ref)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        b.embed_lookup_async(toks, out["out"], table=table, scale=1.5)
        b.embed_grad_async(dout, toks, out["dtable"], scale=1.5)
    big = make(3 * n, 128, V, dtype, "uniform")
    for rep in range(3):
        for v in out.values():
            v.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], ref[k]) for k in ref), rep
        run(b, *big, 1.0)
    b.close()


def test_capture_before_the_workspace_is_there():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    table, dout, toks = make(5000, 64, 90, F32)  # sorted: up to 4096 positions need no workspace
    out = torch.zeros_like(table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(AdnError) as ei:
            b.embed_grad_async(dout, toks, out)
        out.zero_()
    assert ei.value.code == ADN_E_CAPACITY
    b.close()


def test_refusals(be):
    table, dout, toks = make(8, 64, 50, F32)
    out, dt = torch.empty_like(dout), torch.empty_like(table)

    def refused(match, f):
        with pytest.raises(AdnError, match=match) as ei:
            f()
        assert ei.value.code == ADN_E_INVALID
    refused("expected", lambda: be.embed_lookup_async(toks, out.half(), table=table.half()))
    refused("other matrices", lambda: be.embed_lookup_async(toks, out, table=table.bfloat16()))
    refused("torch.int32", lambda: be.embed_lookup_async(toks.long(), out, table=table))
    refused("elements", lambda: be.embed_lookup_async(toks[:5], out, table=table))
    refused("shape", lambda: be.embed_lookup_async(toks, out, table=table[:, :32]))
    refused("context's GPU", lambda: be.embed_lookup_async(toks, out, table=table.cpu()))
    refused("context's GPU", lambda: be.embed_grad_async(dout, toks.cpu(), dt))
    refused("vocab", lambda: be.embed_grad_async(dout, toks, dt[:0]))
    refused("other matrices", lambda: be.embed_grad_async(dout, toks, dt.bfloat16()))
    refused("stride", lambda: be.embed_grad_async(dout[:1].expand(8, 64), toks, dt))
    be.synchronize()
