"""What the vocabulary cross entropy's gradients keep of small probabilities, and that its roundings have no common sign (needs
an MI355X).

Tolerances, with u = 2^-24, A_iv = sum_k |x_ik w_vk|:
  z      2^-20 A (operands of 21 bits at least, three of four products) + d u A (the sum) + 2^-36 max|w| sum|x| (w's resolution)
         + 3 u |z| (bias, conversion to units of log 2, rounding);
  p      relative: z's error, the largest of its row for lse, 2^-16 for the sum of exponentials (at most 2^8 additions deep) and
         the exponentials themselves, 3 u |lse|;
  dz     rounded to 21 bits (fp32 calls) or 11 (bf16 calls, half a step 2^-12); half the smallest step, of dloss: fp16's 2^-24
         under a scale of 2^14, times at most 2 (dz / dloss is stored over a factor in [1, 2)), 2^-38, and 2^-16 of that for an
         entry whose largest value is below 2^-16 (fp32 calls), 2^-24 of that below 2^-24;
  dW     sum over the rows of that error times |x|, operands 2^-20 and x's own planes 2^-35 of the largest |x dloss| (bf16 calls:
         x dloss rounded to 11 bits), a chain of at most `rows` fp32 additions; the output's half step.
"""
import math

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


def peaked(rows, d, V, dtype, seed):
    """A trained head: a quarter of the entries (at most 200) share nearly all probability, the others have 1e-12 to 1e-6, and
    change by up to e^6 from one block of 128 rows to the next.  The last row's target is one of those, the others' are not."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    often = max(1, min(V // 4, 200))
    x, w = rnd(rows, d), rnd(V, d) * (0.5 / d ** 0.5)
    bias = math.log(often) - 13.8 - 13.8 * torch.rand(V, device="cuda", generator=g)
    bias[:often] = 0.3 * rnd(often)
    x[:, 0] = 4.0 * (torch.arange(rows, device="cuda") // 128 % 2)
    w[:, 0] = torch.where(torch.arange(V, device="cuda") % 2 == 0, 1.5, -1.5)
    w[:often, 0] = 0.0
    t = torch.randint(0, often, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[rows - 1] = V - 1
    t[rows // 3] = -1
    return dict(x=x.to(dtype), w=w.to(dtype), bias=bias, targets=t, dloss=torch.full((rows,), 1.0 / (rows - 1), device="cuda")), often


SHAPES = [(65, 96, 1200), (70, 100, 256), (130, 64, 700), (300, 64, 2000), (300, 192, 250), (600, 72, 900), (531, 512, 3000),
          (2100, 96, 130), (300, 64, 50257), (5000, 64, 9000), (1030, 1024, 5000), (3000, 2048, 1000),
          (9000, 2048, 12000), (64, 64, 900), (3, 64, 900)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", SHAPES)
def test_gradients_of_rare_entries(be, rows, d, V, dtype):
    """Each row of dW is right at its own size, however small."""
    print(f"rare entries {rows} x {d} x {V} {dtype}", flush=True)
    s, often = peaked(rows, d, V, dtype, rows + V)
    out = loss(be, s)
    keep = torch.nonzero(s["targets"] >= 0)[:, 0]
    x, w, t, g = s["x"].double()[keep], s["w"].double(), s["targets"].long()[keep], s["dloss"].double()[keep][:, None]
    z = torch.mm(x, w.t().contiguous()) + s["bias"].double()
    tz = (2.0 ** -20 + d * U) * torch.mm(x.abs(), w.abs().t().contiguous()) + 3 * U * z.abs()
    tz += 2.0 ** -36 * float(w.abs().max()) * x.abs().sum(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    dz = p.clone()
    dz[torch.arange(len(keep), device="cuda"), t] -= 1.0
    assert 1e-16 < float(p[:, often:].min()) and float(p[:, often:].max()) < 1e-2
    bf = dtype == BF16
    e = p * (tz + tz.amax(1, keepdim=True) + 2.0 ** -16 + 3 * U * lse.abs()) + (2.0 ** -12 if bf else 2.0 ** -21) * dz.abs()
    top = dz.abs().amax(0, keepdim=True)
    e += torch.where(top >= (2.0 ** -24 if bf else 2.0 ** -16), 2.0 ** -38, torch.where(top >= 2.0 ** -24, 2.0 ** -54, 2.0 ** -62))
    xg = (x * g).abs()
    wide = xg * ((2.0 ** -12 if bf else 0.0) + 2.0 ** -20 + rows * U) + 2.0 ** -35 * xg.max()
    ref = torch.mm((dz * g).t().contiguous(), x)
    tol = torch.mm(e.t().contiguous(), xg) + torch.mm(dz.abs().t().contiguous(), wide) + (2.0 ** -8 if bf else U) * ref.abs()
    err = (out["dw"].double() - ref).abs()
    worst = (err / tol).amax()
    ref_dw, tol_dw = ref, tol
    assert (err <= tol).all(), f"dw: {int((err > tol).sum())} elements beyond, worst {float(worst)} of the tolerance"
    ref = (dz * g).sum(0)
    assert ((out["db"].double() - ref).abs() <= (e * g).sum(0) + rows * U * (dz.abs() * g).sum(0)).all()
    assert ((loss(be, s, ("dw",))["dw"].double() - ref_dw).abs() <= tol_dw).all()  # by itself


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", [(300, 64, 2000), (300, 192, 250), (5000, 64, 9000)])
def test_rows_and_calls_apart(be, rows, d, V, dtype):
    """Beside rare entries too: equal calls give equal bits, and a row matters to no other row's loss and dx."""
    s, _ = peaked(rows, d, V, dtype, rows)
    out = loss(be, s)
    again = loss(be, s)
    assert all(torch.equal(out[k], again[k]) for k in out)
    s["x"][7] = float("nan")  # takes its values out of its entries' largest
    s["x"][rows - 2] *= 30
    s["dloss"][40] = 1e6
    s["targets"][60] = V - 2
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[[7, 40, 60, rows - 2]] = False
    other = loss(be, s)
    for k in ("loss", "lse", "dx"):
        assert torch.equal(other[k][rest], out[k][rest]), k


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
