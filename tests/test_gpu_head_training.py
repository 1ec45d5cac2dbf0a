"""The head's training operators run together, as a training step uses them (needs an MI355X): embedding rows -> forward ->
norm -> loss and its gradients -> norm's backward pass -> adjoint -> the table's gradient, on one stream without a wait in
between, against the same chain in 64 bits from the forward's own pooled rows and the adjoint's own source gradient.

Tolerances: the loss's logits are off by the norm's and the product's rounding, 2^-18 of sum |x w| at most; every gradient is a
sum of products of values that far off, so it is held to 2^-14 of the same sum over magnitudes (rows of the batch that have no
target contribute exactly nothing)."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
REL = 2.0 ** -14


def log(msg):
    print(msg, flush=True)


def norm64(x, g, eps):
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return x * r * g, r


@pytest.mark.parametrize("B,T,d,H,V", [(1, 1, 64, 2, 300), (2, 13, 128, 4, 777), (3, 177, 192, 3, 2100), (4, 100, 512, 8, 5000)])
def test_training_step(B, T, d, H, V):
    log(f"training step {B} x {T} d={d} V={V}")
    mc = synth.ModelConfig(d=d, H=H, V=V, N=1, flags=0, max_iters=6, eps=0.0)
    w = synth.make_token_sensitive_weights(mc, seed=2)
    be = GpuDeqBackend(mc, B, T)
    be.upload_weights(w)
    dev = {k: torch.from_numpy(w[k]).cuda() for k in ("embed", "lm_w", "lm_b", "lm_g")}
    n = B * T
    g = torch.Generator(device="cuda").manual_seed(n)
    toks = torch.randint(0, V, (n,), device="cuda", generator=g, dtype=torch.int32)
    tgt = torch.randint(0, V, (n,), device="cuda", generator=g, dtype=torch.int32)
    if n > 1:  # the tail of the last sequence is padding
        tgt[-(T // 3 + 1):] = -1
    counted = tgt >= 0
    up = counted.float() / counted.sum()
    f = lambda *s: torch.full(s, 7.0, device="cuda")  # noqa: E731
    s_in, pooled, y = f(B, T, d), f(B, T, d), f(n, d)
    loss, lse, dy, dw, db = f(n), f(n), f(n, d), f(V, d), f(V)
    dpool, dg, src, dE = f(n, d), f(d), f(n, d), f(V, d)
    torch.cuda.synchronize()
    be.embed_lookup_async(toks, s_in.view(n, d))
    be.forward_async(s_in=s_in, outputs=dict(pooled=pooled))
    be.rms_norm_async(pooled.view(n, d), y, gain=dev["lm_g"])
    be.lm_loss_async(y, tgt, w=dev["lm_w"], bias=dev["lm_b"], dloss=up, outputs=dict(loss=loss, lse=lse, dx=dy, dw=dw, db=db))
    be.rms_norm_backward_async(pooled.view(n, d), dy, gain=dev["lm_g"], outputs=dict(dx=dpool, dg=dg))
    be.adjoint_async(n, dpool, 2, 0.7, None, src)
    be.embed_grad_async(src, toks, dE)
    be.synchronize()
    assert torch.equal(s_in.view(n, d), dev["embed"][toks.long()])
    # the head from the forward's pooled rows, in 64 bits
    p, gn, W = pooled.view(n, d).double(), dev["lm_g"].double(), dev["lm_w"].double()
    Y, r = norm64(p, gn, 1e-5)
    z = torch.mm(Y, W.t().contiguous()) + dev["lm_b"].double()
    L = torch.logsumexp(z, 1)
    t = tgt.long().clamp(min=0)
    c, u = counted.double(), up.double()
    hot = torch.zeros_like(z)
    hot[torch.arange(n), t] = 1
    dz = (torch.exp(z - L[:, None]) - hot) * u[:, None]
    az = (torch.exp(z - L[:, None]) + hot) * u[:, None]
    A = torch.mm(Y.abs(), W.abs().t().contiguous()).amax(1)

    def near(got, ref, tol, what):
        err = (got.double() - ref).abs()
        assert (err <= tol).all(), f"{what}: {float((err - tol).max())} beyond, worst {float(err.max())}"
    near(loss, (L - z.gather(1, t[:, None])[:, 0]) * c, (2.0 ** -16 * A + 2.0 ** -14), "loss")
    near(lse, L * c, 2.0 ** -16 * A + 2.0 ** -14, "lse")
    dY = torch.mm(dz, W)
    mY = torch.mm(az, W.abs())
    near(dy, dY, REL * (1 + A[:, None]) * mY + 1e-12, "dx")
    near(dw, torch.mm(dz.t().contiguous(), Y), REL * (1 + float(A.max())) * torch.mm(az.t().contiguous(), Y.abs()) + 1e-12, "dw")
    near(db, dz.sum(0), REL * (1 + float(A.max())) * az.sum(0) + 1e-12, "db")
    # the norm's backward pass from the loss's own dx
    D = dy.double()
    a = D * gn
    near(dpool, r * (a - p * r * r * (a * p).mean(1, keepdim=True)),
         2.0 ** -16 * r * (a.abs() + p.abs() * r * r * (a * p).abs().mean(1, keepdim=True)) + 1e-12, "dpool")
    near(dg, (D * p * r).sum(0), 2.0 ** -14 * (D * p * r).abs().sum(0) + 1e-12, "dg")
    assert torch.equal(dpool[~counted], torch.zeros_like(dpool[~counted]))
    # the table's gradient from the adjoint's own source gradient
    ref = torch.zeros((V, d), device="cuda", dtype=torch.float64).index_add_(0, toks.long(), src.double())
    mag = torch.zeros((V, d), device="cuda", dtype=torch.float64).index_add_(0, toks.long(), src.double().abs())
    near(dE, ref, (n + 2) * 2.0 ** -24 * mag, "dE")
    be.close()


def test_training_step_in_a_graph():
    """The head's part of a step captured as one graph and replayed with other work in between: the eager step's bits."""
    n, d, V = 600, 256, 5000
    be = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    toks = torch.randint(-1, V, (n,), device="cuda", generator=g, dtype=torch.int32)
    tgt = torch.randint(-1, V, (n,), device="cuda", generator=g, dtype=torch.int32)
    table, w, gain, up = rnd(V, d), rnd(V, d) * 0.1, rnd(d) * 0.1 + 1, torch.full((n,), 1.0 / n, device="cuda")
    o = {k: torch.empty(s, device="cuda") for k, s in dict(x=(n, d), y=(n, d), loss=(n,), dy=(n, d), dw=(V, d), dx=(n, d), dg=(d,),
                                                           dE=(V, d)).items()}

    def step():
        be.embed_lookup_async(toks, o["x"], table=table, scale=d ** 0.5)
        be.rms_norm_async(o["x"], o["y"], gain=gain)
        be.lm_loss_async(o["y"], tgt, w=w, dloss=up, outputs=dict(loss=o["loss"], dx=o["dy"], dw=o["dw"]))
        be.rms_norm_backward_async(o["x"], o["dy"], gain=gain, outputs=dict(dx=o["dx"], dg=o["dg"]))
        be.embed_grad_async(o["dx"], toks, o["dE"], scale=d ** 0.5)
    torch.cuda.synchronize()
    step()
    be.synchronize()
    ref = {k: v.clone() for k, v in o.items()}
    assert all(torch.isfinite(v).all() for v in ref.values())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for rep in range(4):
        for v in o.values():
            v.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o[k], ref[k]) for k in ref), rep
        assert float((torch.ones(1 << 20, device="cuda") * 2).sum()) == 2.0 ** 21
        if rep == 1:
            step()
            be.synchronize()
            assert all(torch.equal(o[k], ref[k]) for k in ref)
    be.close()
