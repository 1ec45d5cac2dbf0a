"""The training operators at sizes whose launches would pass 2^32 threads in one grid (needs an MI355X with 150 GB of it free).

Tolerances.  Losses: logits of at most 32 exact products (bf16) with partial sums below 2^4, 32 x 2^-24 x 2^4 = 2^-15, and the
conversion to units of log 2, 3 x 2^-24 x 2^4; a sum of exponentials is at most 2^9 additions deep, 2^-15; lse (below 2^5) is
rounded twice, 2^-18.  Norm: bf16 outputs by half a step, 2^-8, the fp32 sum of 2049 squares before by 2^-13 at most."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture()
def be():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("less than 150 GB of the GPU's memory are free")
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    yield b
    b.close()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d", [8, 32])
def test_losses_of_many_rows_and_entries(be, d):
    """2^20 rows against 2^19 entries are 2^24 tiles of 128 x 256 logits, from planes of w (d = 8) and from w as it is."""
    rows, V = 1 << 20, (1 << 19) + 5
    print(f"losses {rows} x {d} x {V}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(d)
    x = (torch.randn((rows, d), device="cuda", generator=g) / d ** 0.5).to(BF16)
    w = torch.randn((V, d), device="cuda", generator=g).to(BF16)
    t = torch.randint(0, V, (rows,), device="cuda", generator=g, dtype=torch.int32)
    t[0], t[1], t[rows - 1] = V - 1, 0, V - 1
    out = dict(loss=torch.full((rows,), 7.0, device="cuda"), lse=torch.full((rows,), 7.0, device="cuda"))
    torch.cuda.synchronize()
    be.lm_loss_async(x, t, w=w, outputs=out)
    be.synchronize()
    at = torch.cat([torch.arange(0, 20, device="cuda"), torch.arange(rows - 20, rows, device="cuda"),
                    torch.randint(0, rows, (60,), device="cuda", generator=g)])
    z = torch.mm(x[at].double(), w.double().t().contiguous())
    assert float(z.abs().max()) < 16
    lse = torch.logsumexp(z, 1)
    tol = 2.0 ** -15 + 2.0 ** -18 + 2.0 ** -15 + 2.0 ** -18
    assert ((out["lse"][at].double() - lse).abs() <= tol).all(), float((out["lse"][at].double() - lse).abs().max())
    ref = lse - z.gather(1, t[at].long()[:, None])[:, 0]
    assert ((out["loss"][at].double() - ref).abs() <= 2 * tol).all(), float((out["loss"][at].double() - ref).abs().max())
    assert torch.isfinite(out["loss"]).all() and (out["lse"] > 8).all()


def test_norm_of_many_long_rows(be):
    """2^24 rows of a block each."""
    rows, d = 1 << 24, 2049
    print(f"norm {rows} x {d}", flush=True)
    x, y = torch.empty((rows, d), device="cuda", dtype=BF16), torch.empty((rows, d), device="cuda", dtype=BF16)
    part = torch.randn((1 << 18, d), device="cuda", dtype=BF16)
    for i in range(0, rows, 1 << 18):
        x[i:i + (1 << 18)] = part * (1 + i / rows)
    y[::4099].fill_(7)
    torch.cuda.synchronize()
    be.rms_norm_async(x, y)
    be.synchronize()
    for i in (0, (1 << 23) - 300, 1 << 23, rows - 300):
        X = x[i:i + 300].double()
        ref = X / torch.sqrt((X * X).mean(1, keepdim=True) + 1e-5)
        assert ((y[i:i + 300].double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -12) * ref.abs() + 1e-30).all(), i
    X = x[::4099].double()
    ref = X / torch.sqrt((X * X).mean(1, keepdim=True) + 1e-5)
    assert ((y[::4099].double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -12) * ref.abs() + 1e-30).all()
