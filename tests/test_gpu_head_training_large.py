"""The training operators where offsets pass 32 bits (needs an MI355X): tables and rows of more than 2^31 elements, and a few
rows at strides beyond it.  Results are checked where offsets are largest, in 64 bits.

Tolerances: bf16 outputs are off by half a step (2^-8 of the value at most) and by the fp32 sums below them.  A logit adds 1024
exact products with partial sums below 8: 1024 x 2^-24 x 8 = 2^-11.  A sum of exponentials is at most 2048 additions deep (2^-13
relative), so lse is off by 2^-11 + 2^-13, an exponential by 2^-10 and the exponent's own rounding in relative terms, and dz is
rounded to 11 bits besides."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    yield b
    b.close()
    torch.cuda.empty_cache()


def near(got, ref, tol, what):
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), f"{what}: worst {float(err.max())}, {float((err - tol).max())} beyond"


def test_norm_of_many_rows(be):
    n, d = (1 << 21) + 5, 1024
    print(f"norm {n} x {d}", flush=True)
    x = torch.randn((n, d), device="cuda", dtype=BF16)
    dy = torch.randn((n, d), device="cuda", dtype=BF16)
    y, dx, dg = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(d, device="cuda")
    torch.cuda.synchronize()
    be.rms_norm_async(x, y)
    be.rms_norm_backward_async(x, dy, outputs=dict(dx=dx, dg=dg))
    be.synchronize()
    at = torch.tensor([0, 1, n // 2, n - 1000, n - 2, n - 1], device="cuda")
    X, A = x[at].double(), dy[at].double()
    r = 1 / torch.sqrt((X * X).mean(1, keepdim=True) + 1e-5)
    near(y[at], X * r, 2.0 ** -8 * (X * r).abs() + 2.0 ** -18 * X.abs(), "y")
    ref = r * (A - X * r * r * (A * X).mean(1, keepdim=True))
    near(dx[at], ref, 2.0 ** -8 * ref.abs() + 2.0 ** -16 * r * (A.abs() + X.abs() * r), "dx")
    total, size = torch.zeros(d, device="cuda", dtype=torch.float64), torch.zeros(d, device="cuda", dtype=torch.float64)
    for i in range(0, n, 1 << 17):
        X, A = x[i:i + (1 << 17)].double(), dy[i:i + (1 << 17)].double()
        t = A * X / torch.sqrt((X * X).mean(1, keepdim=True) + 1e-5)
        total += t.sum(0)
        size += t.abs().sum(0)
    # each of 512 blocks' 4 teams adds n / 2048 = 1025 rows one after another, then 2048 sums: 2^-24 a step
    near(dg, total, (1025 + 2048 + 8) * 2.0 ** -24 * size, "dg")


def test_table_of_many_rows(be):
    V, d, n = (1 << 21) + 9, 1024, 9000
    print(f"table {V} x {d}", flush=True)
    table = torch.randn((V, d), device="cuda", dtype=BF16)
    toks = torch.randint(0, V, (n,), device="cuda", dtype=torch.int32)
    toks[:4] = torch.tensor([V - 1, V - 2, 0, V - 1], device="cuda", dtype=torch.int32)
    out, dt = torch.zeros((n, d), device="cuda", dtype=BF16), torch.full_like(table, 7.0)
    torch.cuda.synchronize()
    be.embed_lookup_async(toks, out, table=table)
    be.synchronize()
    assert torch.equal(out, table[toks.long()])
    for m in (n, 3000):  # sorted, and in one launch
        dt.fill_(7.0)
        torch.cuda.synchronize()
        be.embed_grad_async(out[:m], toks[:m], dt)
        be.synchronize()
        seen = torch.zeros(V, device="cuda", dtype=torch.bool)
        seen[toks[:m].long()] = True
        for i in range(0, V, 1 << 19):
            assert (dt[i:i + (1 << 19)][~seen[i:i + (1 << 19)]] == 0).all()
        uniq, inv = torch.unique(toks[:m], return_inverse=True)
        ref = torch.zeros((len(uniq), d), device="cuda", dtype=torch.float64).index_add_(0, inv, out[:m].double())
        mag = torch.zeros_like(ref).index_add_(0, inv, out[:m].double().abs())
        near(dt[uniq.long()], ref, 2.0 ** -8 * ref.abs() + 2.0 ** -20 * mag, f"dtable of {m}")


@pytest.mark.parametrize("rows", [2, 20])
def test_loss_of_a_large_vocabulary(be, rows):
    V, d = (1 << 21) + 9, 1024
    print(f"loss {rows} x {d} of {V}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = torch.randn((V, d), device="cuda", dtype=BF16, generator=g)
    x = (torch.randn((rows, d), device="cuda", generator=g) / 32).to(BF16)
    t = torch.randint(0, V, (rows,), device="cuda", dtype=torch.int32, generator=g)
    t[0], t[1] = V - 1, V - 9
    out = dict(loss=torch.zeros(rows, device="cuda"), lse=torch.zeros(rows, device="cuda"), dx=torch.zeros_like(x),
               dw=torch.full_like(w, 7.0), db=torch.full((V,), 7.0, device="cuda"))
    torch.cuda.synchronize()
    be.lm_loss_async(x, t, w=w, outputs=out)
    be.synchronize()
    z = torch.empty((rows, V), device="cuda", dtype=torch.float64)
    step, X = 1 << 18, x.double()
    for i in range(0, V, step):
        z[:, i:i + step] = torch.mm(X, w[i:i + step].double().t().contiguous())
    assert float(z.abs().max()) < 8
    lse = torch.logsumexp(z, 1)
    near(out["lse"], lse, 2.0 ** -11 + 2.0 ** -13, "lse")
    near(out["loss"], lse - z.gather(1, t.long()[:, None])[:, 0], 2.0 ** -10 + 2.0 ** -13, "loss")
    dz = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(dz).scatter_(1, t.long()[:, None], 1.0)
    e = (2.0 ** -10 + 2.0 ** -12 + 2.0 ** -11) * dz + 2.0 ** -11 * hot + 2.0 ** -36  # of |dz|: exponentials, 11 bits, its smallest step
    dz -= hot
    dx, tol = torch.zeros((rows, d), device="cuda", dtype=torch.float64), torch.zeros((rows, d), device="cuda", dtype=torch.float64)
    for i in range(0, V, step):
        W = w[i:i + step].double()
        dx += torch.mm(dz[:, i:i + step].contiguous(), W)
        tol += torch.mm((e[:, i:i + step] + 2.0 ** -12 * dz[:, i:i + step].abs()).contiguous(), W.abs())
    near(out["dx"], dx, tol + 2.0 ** -8 * dx.abs(), "dx")
    near(out["db"], dz.sum(0), e.sum(0), "db")
    at = torch.cat([t.long(), torch.arange(V - 700, V, device="cuda"), torch.randint(0, V, (500,), device="cuda")])
    D, E = dz[:, at].t().contiguous(), e[:, at].t().contiguous()
    dw = torch.mm(D, X)
    near(out["dw"][at], dw, torch.mm(E + 2.0 ** -20 * D.abs(), X.abs()) + 2.0 ** -8 * dw.abs(), "dw")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_far_apart(be, dtype):
    """Strides past 2^31 elements: the same bits as tight rows."""
    d, rows, V, stride = 72, 3, 400, (1 << 31) + 24
    print(f"strides of {stride} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, d), device="cuda", generator=g).to(dtype)
    w = torch.randn((V, d), device="cuda", generator=g).to(dtype)
    t = torch.tensor([0, 7, V - 1], device="cuda", dtype=torch.int32)

    def far():
        return torch.empty(2 * stride + d, device="cuda", dtype=dtype).as_strided((rows, d), (stride, 1))
    fx, fy = far(), far()
    fx.copy_(x)
    tight, y = dict(dx=torch.zeros_like(x), dw=torch.zeros_like(w)), torch.zeros_like(x)
    for xs, dx, nm in ((x, tight["dx"], y), (fx, fy, fy)):
        got = dict(dx=dx, dw=torch.zeros_like(w))
        torch.cuda.synchronize()
        be.lm_loss_async(xs, t, w=w, outputs=got)
        be.synchronize()
        if xs is x:
            tight["dw"] = got["dw"]
        else:
            assert torch.equal(fy, tight["dx"]) and torch.equal(got["dw"], tight["dw"])
        be.rms_norm_async(xs, nm)
        be.synchronize()
    assert torch.equal(fy, y)
    dx, dt = torch.zeros_like(x), torch.zeros((50, d), device="cuda", dtype=dtype)
    torch.cuda.synchronize()
    be.rms_norm_backward_async(x, x, outputs=dict(dx=dx))
    be.rms_norm_backward_async(fx, fx, outputs=dict(dx=fy))
    be.synchronize()
    assert torch.equal(fy, dx)
    toks = torch.tensor([2, 0, 2], device="cuda", dtype=torch.int32)
    near_t, far_t = torch.zeros((3, d), device="cuda", dtype=dtype), far()
    torch.cuda.synchronize()
    be.embed_lookup_async(toks, fy, table=fx, scale=2.0)
    be.embed_grad_async(x, toks, near_t)
    be.embed_grad_async(fx, toks, far_t)
    be.embed_grad_async(fx, toks, dt)
    be.synchronize()
    assert torch.equal(fy, (x[toks.long()].float() * 2).to(dtype))
    assert torch.equal(far_t, near_t) and torch.equal(dt[:3], near_t) and (dt[3:] == 0).all()
