"""That the roundings of the vocabulary cross entropy's gradients have no common sign, and how right its sums are (needs an
MI355X)."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    yield b
    b.close()


def loss(be, s, what=("dx", "dw", "db", "loss", "lse")):
    rows, d = s["x"].shape
    V = s["w"].shape[0]
    shape = dict(loss=(rows,), lse=(rows,), dx=(rows, d), dw=(V, d), db=(V,))
    out = {k: torch.full(shape[k], 7.0, device="cuda", dtype=s["x"].dtype if k in ("dx", "dw") else F32) for k in what}
    torch.cuda.synchronize()
    be.lm_loss_async(s["x"], s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], outputs=out)
    be.synchronize()
    return out


@pytest.mark.parametrize("counted,V,spread", [(425, 3000, 1.0), (600, 1500, 0.05), (531, 5003, 0.02), (425, 100, 0.02), (130, 2500, 0.05)])
def test_roundings_have_no_common_sign(be, counted, V, spread):
    """bf16 gradients of a mean over the rows (dloss = 1 / n, alike for all), probabilities nearly alike too: their error has no
    part in the direction of the gradient itself.

    That part, sum(err y) / sum(y y), adds independent roundings: the output's, uniform over a step of 2^-8 to 2^-7 of |y| (1.4
    x 2^-8 in the mean of squares, a standard deviation of that / sqrt(12)), and those of x dloss and dz to 11 bits, an eighth
    of it each.  Five such deviations are 6 x 1.25 x 2^-8 / sqrt(12); 2^-15 for what is common: fp32 exponentials and logits."""
    print(f"mean signed error {counted} x 128 x {V}", flush=True)
    rows, d = counted + counted // 4, 128
    g = torch.Generator(device="cuda").manual_seed(counted)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    s = dict(x=rnd(rows, d).to(BF16), w=(rnd(V, d) * spread / d ** 0.5).to(BF16), bias=None)
    t = torch.randint(0, V, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[torch.randperm(rows, device="cuda", generator=g)[:rows - counted]] = -1
    s["targets"], s["dloss"] = t, torch.full((rows,), 1.0 / counted, device="cuda")
    out = loss(be, s, ("dx", "dw"))
    keep = torch.nonzero(t >= 0)[:, 0]
    x, w, gg = s["x"].double()[keep], s["w"].double(), s["dloss"].double()[keep][:, None]
    dz = torch.softmax(torch.mm(x, w.t().contiguous()), 1)
    dz[torch.arange(counted, device="cuda"), t.long()[keep]] -= 1.0
    ref = dict(dw=torch.mm((dz * gg).t().contiguous(), x), dx=torch.zeros((rows, d), dtype=torch.float64, device="cuda"))
    ref["dx"][keep] = torch.mm(dz * gg, w)
    for k, y in ref.items():
        part = float(((out[k].double() - y) * y).sum() / (y * y).sum())
        dev = 1.25 * 2.0 ** -8 / 12 ** 0.5 * float(y.pow(4).sum().sqrt() / (y * y).sum())
        assert abs(part) <= 6 * dev + 2.0 ** -15, f"{k}: {part:.2e} of the gradient against {6 * dev + 2.0 ** -15:.2e}"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", [(1, 64, 50257), (7, 96, 65), (30, 64, 9001), (64, 128, 50257), (100, 60, 200), (130, 64, 3001),
                                      (300, 96, 50257), (2000, 64, 1030)])
@pytest.mark.parametrize("grads", [True, False])
def test_sum_of_exponentials(be, rows, d, V, dtype, grads):
    """Rows of zeros: every logit is its bias, so lse shows the sum's own error.  A term is off by 2^-22 (the hardware's
    exponential) and by 3 u of its exponent's size (the conversion to units of log 2); the sum is at most 2^7 additions deep; lse
    is rounded twice more, in units of log 2 and in natural ones."""
    print(f"sum {rows} x {d} x {V} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V)
    s = dict(x=torch.zeros((rows, d), device="cuda", dtype=dtype), w=torch.randn((V, d), device="cuda", generator=g).to(dtype),
             bias=None, dloss=None, targets=torch.randint(0, V, (rows,), device="cuda", generator=g, dtype=torch.int32))
    for bias in (None, torch.randn(V, device="cuda", generator=g)):
        s["bias"] = bias
        out = loss(be, s, ("loss", "lse", "dx") if grads else ("loss", "lse"))
        z = torch.zeros(V, dtype=torch.float64, device="cuda") if bias is None else bias.double()
        lse = torch.logsumexp(z, 0)
        most = float(z.abs().max())
        tol = 2.0 ** -22 + 3 * U * most + 2.0 ** 7 * U + 4 * U * float(lse.abs())
        assert ((out["lse"].double() - lse).abs() <= tol).all(), (float((out["lse"].double() - lse).abs().max()), tol)
        ref = lse - z[s["targets"].long()]
        assert ((out["loss"].double() - ref).abs() <= tol + 4 * U * most + U * ref.abs()).all()
