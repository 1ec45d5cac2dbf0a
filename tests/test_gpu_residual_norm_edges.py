"""The residual norms where an input has no say in an output, and column sums that are exact (needs an MI355X)."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
GATES = ["none", "channel", "row", "element"]


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def gate_of(kind, rows, d, dtype, g):
    shape = {"none": None, "channel": (d,), "row": (rows, 1), "element": (rows, d)}[kind]
    return None if shape is None else torch.randn(shape, device="cuda", generator=g).to(dtype if kind == "element" else F32)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("d", [64, 100, 600, 2048, 5000])
def test_without_the_norm_df_does_not_depend_on_f(be, d, gate, dtype):
    """df = scale s D there: an infinite or undefined f changes none of its bits, nor dx's."""
    rows = 9
    log(f"df without the norm {rows} x {d} {gate} {dtype}")
    g = torch.Generator(device="cuda").manual_seed(d)
    f, z, dz, dy = (torch.randn((rows, d), device="cuda", generator=g).to(dtype) for _ in range(4))
    s = gate_of(gate, rows, d, dtype, g)
    got = []
    for bad in (False, True):
        h = f.clone()
        if bad:
            h[2, 3], h[4, d - 1], h[4, 0], h[7] = float("inf"), float("nan"), -float("inf"), float("inf")
        out = dict(dx=torch.zeros_like(f), df=torch.zeros_like(f))
        torch.cuda.synchronize()
        be.residual_norm_backward_async(z, h, dz=dz, dy=dy, gate=s, post_norm=False, keep=0.3, scale=0.7, outputs=out)
        be.synchronize()
        got.append(out)
    for k in ("dx", "df"):
        assert bool(torch.isfinite(got[0][k]).all())
        assert torch.equal(got[1][k], got[0][k]), k
