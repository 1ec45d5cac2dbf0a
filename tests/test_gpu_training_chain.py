"""A training step of a residual block between the embedding and the head, every operator on the framework's kernels: lookup, the
block (a matrix product), its norms, the loss with its gradients, the way back, the table's gradient, clipping and the AdamW step
(needs an MI355X).

Gradients against automatic differentiation in 64 bits: each operator's outputs are within 2^-17 of their norm (operands of the loss
keep 21 bits, the others are fp32), eight of them in a row and a block's product between them: 2^-13 of a gradient's norm.  The step
itself against its formula from the gradients that it was given, as in the optimizer's own tests."""
import numpy as np
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROWS, D, VOCAB = 96, 128, 300


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def exact_gradients(w, tokens, targets, keep, scale):
    p = {k: v.detach().double().requires_grad_() for k, v in w.items()}
    x = p["table"][tokens.long()]
    f = x @ p["block"].t()
    n = f / torch.sqrt(f.square().mean(1, keepdim=True) + 1e-6) * p["post"]
    z = keep * x + scale * p["gate"] * n
    y = z / torch.sqrt(z.square().mean(1, keepdim=True) + 1e-6) * p["pre"]
    loss = torch.nn.functional.cross_entropy(y @ p["head"].t() + p["bias"], targets.long())
    return dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(be, bits):
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    w = dict(table=rnd(VOCAB, D) * 0.3, block=rnd(D, D) * D ** -0.5, post=1 + 0.1 * rnd(D), gate=0.5 + 0.1 * rnd(D), pre=1 + 0.1 * rnd(D),
             head=rnd(VOCAB, D) * 0.2, bias=rnd(VOCAB) * 0.05)
    grad = {k: torch.zeros_like(v) for k, v in w.items()}
    keep, scale, lr, max_norm = 0.3, 0.7, 1e-2, 0.25
    decay = [0.0 if v.dim() == 1 else 0.1 for v in w.values()]
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    x, f, z, y, dy, dx, df = (new(ROWS, D) for _ in range(7))
    loss, lse, norm = new(ROWS), new(ROWS), new(1)
    dloss = torch.full((ROWS,), 1.0 / ROWS, device="cuda")
    copies = [torch.zeros_like(v, dtype=torch.bfloat16) for v in w.values()]
    opt = be.adamw(list(w.values()), list(grad.values()), state_bits=bits, weight_decay=decay, copies=copies, seed=1)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(stream.cuda_stream)
    block = dict(gate=w["gate"], post_gain=w["post"], pre_gain=w["pre"], keep=keep, scale=scale, eps=1e-6)
    try:
        for k in range(3):
            tokens = torch.randint(0, VOCAB, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
            targets = torch.randint(0, VOCAB, (ROWS,), device="cuda", generator=g, dtype=torch.int32)
            want = exact_gradients(w, tokens, targets, keep, scale)
            before = {n: v.clone() for n, v in w.items()}
            state = [(m.float().clone(), v.float().clone(), None if bits == 32 else (a.clone(), b.clone()))
                     for m, v, a, b in zip(opt.m, opt.v, opt.m_scale, opt.v_scale)]
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                be.embed_lookup_async(tokens, x, table=w["table"])
                torch.mm(x, w["block"].t(), out=f)
                be.residual_norm_async(x, f, outputs=dict(z=z, y=y), **block)
                be.lm_loss_async(y, targets, w=w["head"], bias=w["bias"], dloss=dloss, outputs=dict(loss=loss, lse=lse, dx=dy, dw=grad["head"], db=grad["bias"]))
                be.residual_norm_backward_async(z, f, dy=dy, outputs=dict(dx=dx, df=df, dgate=grad["gate"], dpost_gain=grad["post"], dpre_gain=grad["pre"]), **block)
                torch.mm(df.t(), x, out=grad["block"])
                dx.addmm_(df, w["block"])
                be.embed_grad_async(dx, tokens, grad["table"])
                opt.grad_norm_async(norm)
                opt.step_async(lr=lr, grad_norm=norm, max_norm=max_norm)
            torch.cuda.synchronize()
            for n in w:
                err = float((grad[n].double() - want[n]).norm() / want[n].norm())
                assert err <= 2.0 ** -13, (k, n, err)
            total = float(torch.stack([v.double().square().sum() for v in grad.values()]).sum().sqrt())
            assert abs(float(norm) - total) <= 2 * U * total
            coef, t = min(1.0, max_norm / (float(norm) + 1e-6)), k + 1
            assert int(opt.step[0]) == t
            for (n, v), (m0, v0, scales), wd, c in zip(w.items(), state, decay, copies):
                a = lambda q: q.double().cpu().numpy().ravel()  # noqa: E731
                gr, m0, v0 = a(grad[n]) * coef, a(m0), a(v0)
                if scales is not None:
                    m0, v0 = (q * np.repeat(a(s), 256)[:q.size] for q, s in zip((m0, v0), scales))
                m1, v1, p0 = 0.9 * m0 + (1 - 0.9) * gr, 0.999 * v0 + (1 - 0.999) * gr * gr, a(before[n])
                away = m1 / (1 - 0.9 ** t) / (np.sqrt(v1 / (1 - 0.999 ** t)) + 1e-8)
                den = (1 - 0.9 ** t) * (np.sqrt(v1 / (1 - 0.999 ** t)) + 1e-8)
                p1 = p0 - lr * (away + wd * p0)
                tol = lr * (36 * U * np.abs(away) + 6 * U * (np.abs(0.9 * m0) + np.abs(0.1 * gr)) / den + 6 * U * np.abs(wd * p0)) + 2 * U * (np.abs(p0) + np.abs(p1))
                assert (np.abs(a(v) - p1) <= tol + 1e-45).all(), (k, n)
                assert torch.equal(c, v.to(torch.bfloat16))
    finally:
        torch.cuda.synchronize()
        be.set_stream(None)
