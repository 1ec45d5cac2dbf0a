"""The vocabulary cross entropy and its gradients (adn_lm_loss_async) against the definition in 64 bits (needs an MI355X).

Tolerances, with A_iv = sum_k |x_ik w_vk| and u = 2^-24 (half a step of fp32):
  logits   operands carried with at least 21 bits (two fp16 halves, or bf16 values as they are), three products kept of
           four: 2^-20 A; the fp32 sum over d: d u A.  tz = (2^-20 + d u) max A.
  lse      2 tz (every logit off by at most tz, and the reference's own shift), the exponentials and their sum in fp32 with
           at most 2^9 additions in a chain: 2^-14, and the rounding of the result, 2 u |lse|.
  dz       p = exp(z - lse) is off by (3 tz + 2^-14) p; rounded to 21 bits (fp32 call) or one fp16 value (bf16 call, half a
           step 2^-11), with a floor of 2^-36 of the largest |dloss| (fp16's smallest step under the scale).
  products sum over K terms of |dz| |w| (|x|), operands 2^-20, a chain of at most K fp32 additions: K u.
  outputs  rounded once: half a step, 2^-8 |y| for bf16, u |y| for fp32.
"""
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


def make(rows, d, V, dtype=F32, bias=False, pad=0.0, dloss="mean", seed=0, spread=1.7):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + d * 17 + V)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x = rnd(rows, d).to(dtype)
    w = (rnd(V, d) * (spread / d ** 0.5)).to(dtype)
    b = rnd(V) * 0.3 if bias else None
    t = torch.randint(0, V, (rows,), device="cuda", generator=g, dtype=torch.int32)
    if pad:
        t[torch.rand(rows, device="cuda", generator=g) < pad] = -1
    if dloss == "mean":
        up = torch.full((rows,), 1.0 / rows, device="cuda")
    elif dloss == "mixed":  # signs, zeros and six orders of magnitude
        up = rnd(rows) * torch.pow(10.0, -6 * torch.rand(rows, device="cuda", generator=g))
        up[::5] = 0.0
    else:
        up = None
    return dict(x=x, w=w, bias=b, targets=t, dloss=up)


def buffers(s, what=("loss", "lse", "dx", "dw", "db"), fill=7.0):
    rows, d = s["x"].shape
    V = s["w"].shape[0]
    shape = dict(loss=(rows,), lse=(rows,), dx=(rows, d), dw=(V, d), db=(V,))
    return {k: torch.full(shape[k], fill, device="cuda", dtype=s["x"].dtype if k in ("dx", "dw") else F32) for k in what}


def call(be, s, out):
    torch.cuda.synchronize()
    be.lm_loss_async(s["x"], s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], outputs=out)
    be.synchronize()
    return out


def reference(s):
    """Results and tolerances in 64 bits; rows without a target are left out before anything is formed."""
    keep = torch.nonzero(s["targets"] >= 0)[:, 0]
    rows, d = s["x"].shape
    V = s["w"].shape[0]
    x, w, t = s["x"].double()[keep], s["w"].double(), s["targets"].long()[keep]
    g = torch.ones(rows, device="cuda", dtype=torch.float64) if s["dloss"] is None else s["dloss"].double()
    g = g[keep][:, None]
    z = torch.mm(x, w.t().contiguous())
    if s["bias"] is not None:
        z = z + s["bias"].double()
    lse = torch.logsumexp(z, 1)
    hot = torch.zeros_like(z)
    hot[torch.arange(len(keep)), t] = 1.0
    dz = torch.exp(z - lse[:, None]) - hot
    ref, tol = {}, {}
    A = torch.mm(x.abs(), w.abs().t().contiguous()).amax(1) if len(keep) and V else torch.zeros(len(keep), device="cuda")
    zb = s["bias"].double().abs().clamp(max=1e30).where(s["bias"].double().isfinite(), torch.zeros(())
                                                        .double().cuda()) if s["bias"] is not None else None
    tz = (2.0 ** -20 + d * U) * A + (2 * U * (z.where(z.isfinite() & (z.abs() < 1e30), torch.zeros_like(z)).abs().amax(1))
                                     if len(keep) else 0)
    del zb

    def spread_rows(v):
        out = torch.zeros(rows, dtype=torch.float64, device="cuda")
        out[keep] = v
        return out
    lt = 2 * tz + 2.0 ** -14 + 2 * U * lse.abs()
    ref["lse"], tol["lse"] = spread_rows(lse), spread_rows(lt)
    ref["loss"], tol["loss"] = spread_rows(lse - z[torch.arange(len(keep)), t]), spread_rows(lt + tz)
    bf = s["x"].dtype == BF16
    dP = 2.0 ** -11 if bf else 2.0 ** -20
    out_step = 2.0 ** -8 if bf else U
    p = torch.exp(z - lse[:, None])
    floor = 2.0 ** -36 * float(g.abs().max()) if len(keep) else 0.0
    # |dz| and its error: the exponential's relative error and the halves' rounding
    e_dz = g.abs() * ((3 * tz[:, None] + 2.0 ** -14) * p + dP * dz.abs()) + floor
    a_dz = g.abs() * dz.abs()
    dzg = g * dz
    ref["dx"] = torch.zeros((rows, d), dtype=torch.float64, device="cuda")
    tol["dx"] = torch.zeros_like(ref["dx"])
    ref["dx"][keep] = torch.mm(dzg, w)
    tol["dx"][keep] = torch.mm(e_dz + (2.0 ** -20 + V * U) * a_dz, w.abs()) + out_step * ref["dx"][keep].abs()
    ref["dw"] = torch.mm(dzg.t().contiguous(), x)
    tol["dw"] = torch.mm((e_dz + (2.0 ** -20 + rows * U) * a_dz).t().contiguous(), x.abs()) + out_step * ref["dw"].abs()
    ref["db"] = dzg.sum(0)
    tol["db"] = (e_dz + rows * U * a_dz).sum(0) + U * ref["db"].abs()
    return ref, tol


def check(out, ref, tol, what):
    for k, v in out.items():
        err = (v.double() - ref[k]).abs()
        bad = ~(err <= tol[k] + 1e-300)
        assert not bad.any(), (f"{what}: {k}: {int(bad.sum())} of {bad.numel()} beyond the tolerance, worst error "
                               f"{float(err[bad].max())} against {float(tol[k][bad].max())}, first at {torch.nonzero(bad)[0].tolist()}")


SHAPES = [
    # rows, d, vocab: one of each, the tiles' edges, odd and prime sizes
    (1, 1, 1), (1, 1, 2), (3, 7, 5), (1, 64, 300), (1, 512, 4099), (2, 33, 257), (16, 128, 1000), (17, 64, 255),
    (31, 100, 2100), (32, 256, 512), (33, 192, 65), (63, 16, 129), (64, 64, 64), (65, 31, 1023), (100, 320, 700),
    (127, 512, 256), (128, 192, 65), (129, 48, 3001), (255, 512, 1025), (257, 130, 777), (300, 1024, 513),
    (531, 96, 2049), (40, 2048, 900), (1025, 64, 97), (70, 4100, 50),
    # up to 64 rows: as many as fit a wave's lanes, in 128-byte pieces of W, and of other widths
    (7, 100, 300), (6, 33, 4000), (8, 500, 1001), (5, 64, 100), (64, 2048, 600), (33, 160, 3001), (9, 8192, 130), (64, 32, 2066),
    (256, 100, 256), (199, 64, 250), (257, 64, 250), (2100, 96, 130), (11001, 256, 128),
    # logits kept or formed again, on tiles of every size
    (65, 512, 300), (1000, 352, 5000), (2000, 640, 2100), (130, 1024, 900), (600, 2048, 3000), (400, 64, 4000), (5000, 64, 1500),
    (48, 4096, 1000), (50, 1056, 700), (64, 64, 64 * 1030 + 1), (5, 128, 20000), (63, 8192, 2000),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", SHAPES)
def test_against_definition(be, rows, d, V, dtype):
    log(f"loss {rows} x {d} x {V} {dtype}")
    s = make(rows, d, V, dtype, bias=V % 2 == 1, pad=0.2 if rows % 2 else 0.0, dloss="mixed" if rows % 3 == 0 else "mean")
    out = call(be, s, buffers(s))
    check(out, *reference(s), (rows, d, V))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 1500])
def test_large_vocabulary(be, rows, dtype):
    """The repository's vocabulary; 1500 rows are more than one piece of it."""
    log(f"loss {rows} x 64 x 50257 {dtype}")
    s = make(rows, 64, 50257, dtype, bias=True, pad=0.1 if rows > 1 else 0)
    out = call(be, s, buffers(s))
    check(out, *reference(s), rows)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", [(300, 64, 50257), (5000, 64, 50257), (257, 512, 20011), (700, 192, 30011), (3001, 256, 9973),
                                      (1300, 1536, 4001), (1 << 20, 16, 65), (200001, 40, 600)])
def test_large_tiles_and_many_pieces(be, rows, d, V, dtype):
    """Grids of more than a round of the chip, whose tiles are the large ones; 5000 rows take several pieces of the vocabulary, of
    which the last is the smaller, and add dx up over them."""
    log(f"loss {rows} x {d} x {V} {dtype}")
    s = make(rows, d, V, dtype, bias=True, pad=0.1)
    out = call(be, s, buffers(s))
    check(out, *reference(s), rows)


@pytest.mark.parametrize("rows", [3, 20, 200])
def test_row_without_any_entry(be, rows):
    """A bias of -inf everywhere leaves no entry: nothing is a number, and the next call is as ever."""
    s = make(rows, 64, 700, bias=True)
    keep = s["bias"].clone()
    s["bias"][:] = float("-inf")
    out = call(be, s, buffers(s))
    assert torch.isnan(out["loss"]).all() and torch.isnan(out["dx"]).all() and torch.isnan(out["dw"]).all()
    assert (out["lse"] == float("-inf")).all()
    s["bias"] = keep
    check(call(be, s, buffers(s)), *reference(s), rows)


def test_two_contexts_side_by_side():
    """Two contexts on two streams, their calls enqueued without a wait in between."""
    both = []
    for seed in (1, 2):
        b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
        st = torch.cuda.Stream()
        b.set_stream(st.cuda_stream)
        s = make(400, 256, 6000, bias=True, seed=seed)
        both.append((b, s, buffers(s), st))
    torch.cuda.synchronize()
    for _ in range(3):
        for b, s, out, _st in both:
            b.lm_loss_async(s["x"], s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], outputs=out)
    for b, s, out, _st in both:
        b.synchronize()
        check(out, *reference(s), "two contexts")
    for b, *_ in both:
        b.close()


@pytest.mark.parametrize("what", [("loss",), ("lse",), ("dx",), ("dw",), ("db",), ("loss", "dx"), ("dw", "lse")])
@pytest.mark.parametrize("rows", [5, 150])
def test_outputs_apart(be, what, rows):
    """Each output wanted by itself is the one that comes with all of them."""
    s = make(rows, 96, 700, bias=True, dloss=None)
    full = call(be, s, buffers(s))
    some = call(be, s, buffers(s, what))
    for k in what:
        assert torch.equal(some[k], full[k]), k
    check(full, *reference(s), rows)


@pytest.mark.parametrize("rows", [1, 6, 200, 600])
def test_no_row_has_a_target(be, rows):
    s = make(rows, 64, 500)
    s["targets"][:] = -1
    s["x"][:] = float("nan")
    out = call(be, s, buffers(s))
    for k, v in out.items():
        assert torch.equal(v, torch.zeros_like(v)), k


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [9, 300])
def test_padded_rows_are_not_read(be, rows, dtype):
    """NaN, inf and large values in rows without a target, and their dloss, change no bit of the rest."""
    s = make(rows, 128, 999, dtype, pad=0.4)
    gone = s["targets"] < 0
    s["x"][gone] = 0
    clean = {k: v.clone() for k, v in call(be, s, buffers(s)).items()}
    s["x"][gone] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30], device="cuda").repeat(32).to(dtype)
    s["dloss"][gone] = float("nan")
    s["targets"][gone] = -2147483648
    out = call(be, s, buffers(s))
    for k, v in out.items():
        assert torch.equal(v, clean[k]), k
    s["x"][gone] = 0
    s["dloss"][gone] = 0
    check(out, *reference(s), rows)


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(F32).min])
@pytest.mark.parametrize("rows", [4, 20, 130])
def test_entries_out_of_the_vocabulary(be, rows, low):
    """A bias of -inf or the lowest value takes entries out, whole tiles of them too."""
    s = make(rows, 64, 1500, bias=True)
    s["bias"][10:40] = low
    s["bias"][256:1024] = low
    s["targets"][:] = torch.arange(rows, device="cuda", dtype=torch.int32) % 10
    out = call(be, s, buffers(s))
    check(out, *reference(s), low)
    assert torch.equal(out["dw"][256:1024], torch.zeros_like(out["dw"][256:1024]))
    assert torch.equal(out["db"][10:40], torch.zeros_like(out["db"][10:40]))


@pytest.mark.parametrize("rows", [3, 20, 140])
def test_bad_rows_stay_their_own(be, rows):
    """A row of NaN or inf has a loss and a dx that are no numbers; the other rows' are as without it."""
    s = make(rows, 128, 600)
    clean = {k: v.clone() for k, v in call(be, s, buffers(s)).items()}
    s["x"][1, 5] = float("nan")
    s["x"][2, 7] = float("inf")
    out = call(be, s, buffers(s))
    ok = torch.ones(rows, dtype=torch.bool, device="cuda")
    ok[1:3] = False
    for k in ("loss", "lse", "dx"):
        assert torch.equal(out[k][ok], clean[k][ok]), k
        assert not torch.isfinite(out[k][~ok]).any() or k == "dx"
    assert torch.isnan(out["loss"][1:3]).all() and torch.isnan(out["dx"][1:3]).any(1).all()
    assert torch.isnan(out["dw"]).any()


@pytest.mark.parametrize("rows", [8, 260])
def test_rows_of_unlike_size(be, rows):
    """Rows from 1e-6 to 1e3 of the usual size: each row's results at its own scale; one row of zeros."""
    s = make(rows, 128, 800)
    s["x"] *= torch.pow(10.0, torch.linspace(-6, 1, rows, device="cuda"))[:, None]
    s["x"][1] = 0
    out = call(be, s, buffers(s))
    check(out, *reference(s), rows)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 20, 200])
def test_sharp_rows(be, rows, dtype):
    """Logits up to thousands: softmax weights of one and of zero, losses of zero and of thousands."""
    s = make(rows, 64, 900, dtype, spread=300.0)
    best = torch.mm(s["x"].double(), s["w"].double().t().contiguous()).argmax(1).int()
    s["targets"][::2] = best[::2]
    out = call(be, s, buffers(s))
    check(out, *reference(s), rows)


@pytest.mark.parametrize("scale", [1e-20, 1e15])
@pytest.mark.parametrize("rows,V", [(4, 400), (150, 400), (600, 400), (40, 1500)])
def test_weights_of_any_size(be, rows, V, scale):
    """Operands far from 1: a head of 1e-20 (or 1e15) with rows of the inverse size."""
    s = make(rows, 64, V, dloss=None)
    s["w"] *= scale
    s["w"][5] = 0
    s["x"] /= scale
    out = call(be, s, buffers(s))
    check(out, *reference(s), scale)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["large row", "zeros in the sample", "small sample", "small weights", "as the sample"])
@pytest.mark.parametrize("grads", [True, False])
def test_weights_unlike_their_sample(be, grads, kind, dtype):
    """A large W's scale comes from one row in 32: rows that it does not fit, and samples that say nothing."""
    s = make(100, 256, 70000, dtype, bias=True, pad=0.1)
    w = s["w"]
    if kind == "large row":
        w[17] *= 1000
        w[19999] *= 100
    elif kind == "zeros in the sample":
        w[::32] = 0
        w *= 2.0 ** -60
        s["x"] *= 2.0 ** 60
    elif kind == "small sample":
        w[::32] *= 2.0 ** -20
    elif kind == "small weights":
        w *= 2.0 ** -70
        w[5] *= 2.0 ** -20
        s["x"] *= 2.0 ** 70
    else:
        w[1::32] *= 7
    out = call(be, s, buffers(s) if grads else buffers(s, ("loss", "lse")))
    ref, tol = reference(s)
    check(out, ref, tol, kind)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [5, 21, 133, 600])
@pytest.mark.parametrize("offset,extra", [(0, 8), (1, 3), (8, 0)])
def test_strides_and_alignment(be, rows, offset, extra, dtype):
    """Rows at a stride, bases off 16 bytes: same bits as tight rows, nothing written between them."""
    d, V = 72, 333
    s = make(rows, d, V, dtype, bias=True)
    tight = call(be, s, buffers(s))

    def spaced(t):
        n, m = t.shape
        store = torch.full((offset + n * (m + extra),), 5.0, device="cuda", dtype=t.dtype)
        v = store[offset:].view(n, m + extra)[:, :m]
        v.copy_(t)
        return v, store
    loose = dict(s, x=spaced(s["x"])[0], w=spaced(s["w"])[0])
    out = buffers(s)
    out["dx"], dxs = spaced(out["dx"])
    out["dw"], dws = spaced(out["dw"])
    call(be, loose, out)
    for k in tight:
        assert torch.equal(out[k], tight[k]), k
    for store, n in ((dxs, rows), (dws, V)):
        gaps = store[offset:].view(n, d + extra)[:, d:]
        assert torch.equal(gaps, torch.full_like(gaps, 5.0)) and (store[:offset] == 5.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [11, 64])
def test_strides_of_up_to_64_rows(be, rows, dtype):
    """As above where W's rows stand on 16 bytes and the other matrices anywhere."""
    d, V = 192, 1333
    s = make(rows, d, V, dtype, bias=True, pad=0.2)
    tight = call(be, s, buffers(s))

    def spaced(t, offset, extra):
        n, m = t.shape
        store = torch.full((offset + n * (m + extra),), 5.0, device="cuda", dtype=t.dtype)
        v = store[offset:].view(n, m + extra)[:, :m]
        v.copy_(t)
        return v, store
    for o, e in ((1, 3), (8, 8), (0, 2)):
        loose = dict(s, x=spaced(s["x"], o, e)[0], w=spaced(s["w"], 8, 24)[0])
        out = buffers(s)
        out["dx"], dxs = spaced(out["dx"], o, e)
        out["dw"], dws = spaced(out["dw"], o, e)
        call(be, loose, out)
        for k in tight:
            assert torch.equal(out[k], tight[k]), (k, o, e)
        for store, n in ((dxs, rows), (dws, V)):
            gaps = store[o:].view(n, d + e)[:, d:]
            assert torch.equal(gaps, torch.full_like(gaps, 5.0)) and (store[:o] == 5.0).all()


@pytest.mark.parametrize("rows,V", [(4, 200), (70, 200), (600, 200), (30, 2000)])
def test_target_beyond_the_vocabulary_is_reported(be, rows, V):
    s = make(rows, 64, V)
    clean = dict(s, targets=s["targets"].clone())
    clean["targets"][3] = -1
    ref = call(be, clean, buffers(s))
    s["targets"][3] = V
    out = buffers(s)
    be.lm_loss_async(s["x"], s["targets"], w=s["w"], dloss=s["dloss"], outputs=out)
    with pytest.raises(AdnError, match="outside"):
        be.synchronize()
    for k in ref:
        assert torch.equal(out[k], ref[k]), k
    be.synchronize()  # reported once


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V,offset,extra", [(70, 96, 700, 0, 0), (70, 96, 700, 8, 16), (70, 96, 700, 1, 3), (530, 100, 1500, 0, 4),
                                                   (33, 64, 257, 4, 1), (260, 512, 5003, 0, 0), (20, 64, 3000, 8, 8),
                                                   (64, 256, 1111, 0, 0)])
def test_losses_alone(be, rows, d, V, offset, extra, dtype):
    """Without gradients W is read as it stands where its rows allow it: any stride and base."""
    s = make(rows, d, V, dtype, bias=True, pad=0.1)
    store = torch.full((offset + V * (d + extra),), float("nan"), device="cuda", dtype=dtype)
    w = store[offset:].view(V, d + extra)[:, :d]
    w.copy_(s["w"])
    out = call(be, dict(s, w=w), buffers(s, ("loss", "lse")))
    ref, tol = reference(s)
    check(out, ref, tol, (rows, d, V, offset, extra))


def test_empty_batch(be):
    s = make(1, 64, 300)
    out = buffers(s)
    e = torch.empty((0, 64), device="cuda")
    be.lm_loss_async(e, torch.empty(0, device="cuda", dtype=torch.int32), w=s["w"],
                     outputs=dict(loss=torch.empty(0, device="cuda"), dx=torch.empty_like(e), dw=out["dw"], db=out["db"]))
    be.synchronize()
    assert (out["dw"] == 0).all() and (out["db"] == 0).all()


@pytest.mark.parametrize("rows", [3, 20, 90, 600])
def test_uploaded_head(rows):
    """w None: the context's lm_w and lm_b."""
    mc = synth.ModelConfig(d=128, H=2, V=515, N=1, flags=0)
    wts = synth.make_token_sensitive_weights(mc, seed=3)
    b = GpuDeqBackend(mc, 1, 8)
    s = make(rows, 128, 515)
    s["w"], s["bias"] = torch.from_numpy(wts["lm_w"]).cuda(), torch.from_numpy(wts["lm_b"]).cuda()
    with pytest.raises(AdnError) as ei:
        b.lm_loss_async(s["x"], s["targets"], outputs=buffers(s))
    assert ei.value.code == ADN_E_NO_WEIGHTS
    b.upload_weights(wts)
    ref = call(b, s, buffers(s))
    out = buffers(s)
    b.lm_loss_async(s["x"], s["targets"], dloss=s["dloss"], outputs=out)
    b.synchronize()
    for k in ref:
        assert torch.equal(out[k], ref[k]), k
    with pytest.raises(AdnError, match="context's head"):
        b.lm_loss_async(s["x"][:, :64], s["targets"], outputs=dict(loss=out["loss"]))
    b.close()


@pytest.mark.parametrize("rows", [4, 200, 600])
def test_gradients_against_differences(be, rows):
    """Central differences of the losses' sum along random directions.  A step h of a direction of unit size changes each
    logit by about h; the difference's own error is the loss's (2 tol / 2h a row) and the third derivative's, at most h^2 a
    row for directions that move logits by about one."""
    s = make(rows, 64, 500, bias=True, dloss=None)
    out = call(be, s, buffers(s))
    _, tol = reference(s)
    h = 2.0 ** -6
    g = torch.Generator(device="cuda").manual_seed(5)
    for name, grad in (("x", "dx"), ("w", "dw"), ("bias", "db")):
        u = torch.randn(s[name].shape, device="cuda", generator=g)
        u = u / u.norm() * (rows ** 0.5 if name == "x" else 1.0)
        sides = []
        for sign in (1, -1):
            m = dict(s, **{name: s[name] + sign * h * u})
            sides.append(call(be, m, buffers(s, ("loss",)))["loss"].double().sum())
        diff = float((sides[0] - sides[1]) / (2 * h))
        got = float((out[grad].double() * u.double()).sum())
        slack = float(tol["loss"].sum()) / h + h * h * rows * 8 + 1e-6 * abs(got)
        assert abs(diff - got) <= slack, (name, diff, got, slack)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d,V", [(1, 512, 5000), (30, 128, 2000), (300, 192, 3000), (100, 512, 40000)])
def test_same_bits_again_and_in_a_graph(be, rows, d, V, dtype):
    """Equal calls give equal bits; a captured call replayed with other work and a larger call (which grows the workspace)
    in between does too."""
    s = make(rows, d, V, dtype, bias=True, pad=0.1 if rows > 1 else 0)
    b = GpuDeqBackend(be.model, 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    out = call(b, s, buffers(s))
    ref = {k: v.clone() for k, v in out.items()}
    call(b, s, out)
    assert all(torch.equal(out[k], ref[k]) for k in ref)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        b.lm_loss_async(s["x"], s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], outputs=out)
    big = make(2 * rows + 40, d, 2 * V + 300, dtype)
    for rep in range(3):
        for v in out.values():
            v.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], ref[k]) for k in ref), rep
        call(b, big, buffers(big))
        assert float((torch.ones(1 << 20, device="cuda") * 2).sum()) == 2.0 ** 21
    b.close()


def test_capture_before_the_workspace_is_there():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    stream = torch.cuda.Stream()
    b.set_stream(stream.cuda_stream)
    s = make(64, 64, 300)
    out = buffers(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(AdnError) as ei:
            b.lm_loss_async(s["x"], s["targets"], w=s["w"], outputs=out)
        out["loss"].zero_()
    assert ei.value.code == ADN_E_CAPACITY
    torch.cuda.synchronize()
    check(call(b, s, out), *reference(s), "after the refusal")
    b.close()


def test_refusals(be):
    """Each is refused on the host, before anything is launched."""
    s = make(8, 64, 300, bias=True)
    ok = buffers(s)

    def refused(match=None, code=ADN_E_INVALID, outputs=None, **kw):
        a = dict(x=s["x"], targets=s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], **{})
        a.update(kw)
        with pytest.raises(AdnError, match=match) as ei:
            be.lm_loss_async(a.pop("x"), a.pop("targets"), outputs=ok if outputs is None else outputs, **a)
        assert ei.value.code == code
    refused("no output", outputs={})
    refused("unknown outputs", outputs=dict(logits=ok["loss"]))
    refused("expected", x=s["x"].half())
    refused("other matrices", w=s["w"].bfloat16())
    refused("context's GPU", x=s["x"].cpu())
    refused("context's GPU", targets=s["targets"].cpu())
    refused("torch.int32", targets=s["targets"].long())
    refused("shape", w=s["w"][:, :63])
    refused("adjacent", x=s["x"].t().contiguous().t())
    refused("stride", x=s["x"][:1].expand(8, 64))
    refused("bias", bias=s["bias"][:-1])
    refused("dloss", dloss=s["dloss"].double())
    refused("shape", outputs=dict(dx=ok["dw"]))
    refused("other matrices", outputs=dict(dx=ok["dx"].bfloat16()))
    refused("d must be", x=torch.zeros((2, 8193), device="cuda"), targets=s["targets"][:2], dloss=s["dloss"][:2],
            w=torch.zeros((300, 8193), device="cuda"), outputs=dict(loss=ok["loss"][:2]))
    many = (1 << 20) + 1
    refused("number of rows", x=torch.zeros((many, 1), device="cuda"), targets=torch.zeros(many, device="cuda", dtype=torch.int32),
            w=torch.zeros((300, 1), device="cuda"), dloss=None, outputs=dict(loss=torch.zeros(many, device="cuda")))
    refused("vocab", w=torch.zeros(((1 << 24) + 1, 1), device="cuda"), bias=None, x=s["x"][:, :1].contiguous(), outputs=dict(loss=ok["loss"]))
    refused("vocab", w=s["w"][:0], bias=None, outputs=dict(loss=ok["loss"]))
    be.synchronize()
