"""The residual norms' column sums where they are exact: a lost, doubled or misplaced row shows, however many there are (needs an MI355X).

z and f are +-1 and eps is 0, so that both reciprocal roots are 1 (d is a power of two: sums of ones times 1 / d).  dy z is +q, -q
in neighbouring columns and pre_gain is the same in both, so that mean(a z) is 0 and D = dz + dy pre_gain.  All factors are
small integers or powers of two: every product and every partial sum is a multiple of 2^-3 below 2^20, exact in fp32 in any order."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def inputs(rows, d, dtype, gate, seed=0):
    g = torch.Generator(device="cuda").manual_seed(rows + d + seed)
    sign = lambda *s: (torch.randint(0, 2, s, device="cuda", generator=g) * 2 - 1).float()  # noqa: E731
    whole = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, device="cuda", generator=g).float()  # noqa: E731
    power = lambda *s: torch.pow(2.0, whole(-1, 0, *s).float())  # noqa: E731
    z, f, dz = sign(rows, d), sign(rows, d), whole(-2, 2, rows, d)
    q = whole(-2, 2, rows, d // 2)
    dy = torch.stack([q, -q], 2).reshape(rows, d) * z
    t = dict(z=z, f=f, dz=dz, dy=dy, post_gain=power(d), pre_gain=power(d // 2).repeat_interleave(2))
    shape = {"none": None, "channel": (d,), "row": (rows, 1), "element": (rows, d)}[gate]
    t["gate"] = None if shape is None else power(*shape) * sign(*shape)
    t = {k: v.to(dtype) if k in ("z", "f", "dz", "dy") or (k == "gate" and gate == "element") else v for k, v in t.items()}
    return t


def expected(t, keep, scale):
    """In 64 bits, where all of it is exact."""
    z, f, dz, dy, gp, gq = (t[k].double() for k in ("z", "f", "dz", "dy", "post_gain", "pre_gain"))
    s = 1.0 if t["gate"] is None else t["gate"].double()
    D = dz + dy * gq
    out = dict(dpre_gain=(dy * z).sum(0), dpost_gain=(scale * D * s * f).sum(0), dx=keep * D)
    if t["gate"] is not None:
        dg = scale * D * f * gp
        out["dgate"] = dg.sum(0) if t["gate"].dim() == 1 else dg.sum(1, keepdim=True) if t["gate"].shape[1] == 1 else dg
    return out


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", ["none", "channel", "row", "element"])
@pytest.mark.parametrize("rows,d", [(1, 64), (3, 8), (100003, 8), (2047, 64), (50000, 512), (65536, 256), (511, 1024), (20011, 1024), (40000, 2048),
                                    (2049, 4096), (513, 8192), (5003, 8192)])
def test_exact(be, rows, d, gate, dtype):
    log(f"columns {rows} x {d} {gate} {dtype}")
    t = inputs(rows, d, dtype, gate)
    keep, scale = 0.5, 2.0
    names = ["dx", "dpost_gain", "dpre_gain"] + (["dgate"] if gate != "none" else [])
    like = dict(dx=t["f"], dgate=t["gate"], dpost_gain=t["post_gain"], dpre_gain=t["pre_gain"])
    out = {k: torch.full_like(like[k], 7.0) for k in names}
    torch.cuda.synchronize()
    be.residual_norm_backward_async(t["z"], t["f"], dz=t["dz"], dy=t["dy"], gate=t["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"],
                                    keep=keep, scale=scale, eps=0.0, outputs=out)
    be.synchronize()
    want = expected(t, keep, scale)
    for k in names:
        bad = out[k].double() != want[k]
        assert not bad.any(), f"{k}: {int(bad.sum())} of {bad.numel()} differ, first at {torch.nonzero(bad)[0].tolist()}"


@pytest.mark.parametrize("rows,d", [(30011, 512), (10007, 2048)])
def test_exact_off_the_alignment(be, rows, d):
    """By single elements."""
    t = inputs(rows, d, F32, "channel", 1)
    off = {}
    for k in ("z", "f", "dz", "dy"):
        off[k] = torch.empty(rows * d + 1, device="cuda")[1:].view(rows, d)
        off[k].copy_(t[k])
    out = {k: torch.full((d,), 7.0, device="cuda") for k in ("dpost_gain", "dpre_gain", "dgate")}
    torch.cuda.synchronize()
    be.residual_norm_backward_async(off["z"], off["f"], dz=off["dz"], dy=off["dy"], gate=t["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"],
                                    scale=2.0, eps=0.0, outputs=out)
    be.synchronize()
    want = expected(t, 1.0, 2.0)
    assert all(torch.equal(out[k].double(), want[k]) for k in out)


@pytest.mark.parametrize("lost", [0, 12345, 49999])
def test_a_lost_row_would_show(lost):
    """In the oracle: without one row each sum is another in most columns."""
    t = inputs(50000, 512, F32, "channel")
    whole = expected(t, 0.5, 2.0)
    short = expected({k: torch.cat([v[:lost], v[lost + 1:]]) if v.dim() == 2 else v for k, v in t.items()}, 0.5, 2.0)
    for k in ("dgate", "dpost_gain", "dpre_gain"):
        assert float((whole[k] != short[k]).float().mean()) > 0.5


def test_exact_at_the_most_rows(be):
    """2^24 rows, of which one in 64 has a gradient: sums of at most 2^20."""
    rows, d = 1 << 24, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    f = (torch.randint(0, 2, (rows, d), device="cuda", generator=g) * 2 - 1).float()
    dz = torch.zeros((rows, d), device="cuda")
    dz[5::64] = torch.randint(1, 3, (rows // 64, d), device="cuda", generator=g).float()
    gate, gain = torch.full((rows, 1), 0.5, device="cuda"), torch.ones(d, device="cuda")
    out = dict(dpost_gain=torch.full((d,), 7.0, device="cuda"), df=torch.full_like(f, 7.0), dgate=torch.full_like(gate, 7.0))
    torch.cuda.synchronize()
    be.residual_norm_backward_async(None, f, dz=dz, gate=gate, post_gain=gain, scale=2.0, eps=0.0, outputs=out)
    be.synchronize()
    D, h = dz.double(), f.double()
    assert torch.equal(out["dpost_gain"].double(), (D * h).sum(0))
    assert torch.equal(out["dgate"].double(), 2 * (D * h).sum(1, keepdim=True))
    assert torch.equal(out["df"].double(), D - h * (D * h).mean(1, keepdim=True))
