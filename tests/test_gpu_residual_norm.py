"""The norms around a residual block, forward and backward, against the definition in 64 bits (needs an MI355X).

Tolerances, u = 2^-24.  A row's sum of d products: a lane adds at most d/64 + 16 of them in a chain, then a tree of 6 and up to 8 waves:
es = (d/64 + 32) u of the sum of magnitudes; a reciprocal root has half of that and 6 u: er = es.  The gate: exp, a sum, a
reciprocal, a product: eg = 8 u relative, its slope 12 u.  n = f rf gp s scale: (er + eg + 8 u) |n|; z: that, u |keep x| and u |z|; y: the row's
sum of squares of z moves by 2 |z| dz: r by r^3 mean(|z| dz), so |y| (er + 4 u) + dz r gq + |z| gq r^3 mean(|z| dz).
Backward, D: es of mean |a z| and 3 er of it for r^3, and (8 u + er) of each term; its error dD goes on linearly: dx keep dD, dgate |scale n| dD,
b = scale s gp D and df as D from a, with mean |b f|.  Column sums: the terms' errors, and a chain over at most `rows` rows:
(rows + 40) u of the sum of magnitudes.  Outputs are rounded once: half a step (2^-8 for bf16, u for fp32)."""
import pytest
import torch

from aideen_amd import _lib, synth
from aideen_amd._lib import ADN_E_CAPACITY, ADN_E_INVALID, AdnError
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
GATES = ["none", "channel", "row", "element"]


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def make(rows, d, dtype, gate="none", sigmoid=False, post=True, pre=True, seed=0, gains=True):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 13 + d)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    size = lambda: torch.pow(10.0, 2 * torch.rand((rows, 1), device="cuda", generator=g) - 1)  # noqa: E731
    t = dict(x=(rnd(rows, d) * size()).to(dtype), f=(rnd(rows, d) * size()).to(dtype), z=(rnd(rows, d) * size()).to(dtype),
             dz=rnd(rows, d).to(dtype), dy=rnd(rows, d).to(dtype) if pre else None)
    shape = {"none": None, "channel": (d,), "row": (rows, 1), "element": (rows, d)}[gate]
    t["gate"] = None if shape is None else rnd(*shape) * (4 if sigmoid else 1)
    if gate == "element":
        t["gate"] = t["gate"].to(dtype)
    t["post_gain"] = rnd(d) * 0.3 + 1 if post and gains else None
    t["pre_gain"] = rnd(d) * 0.3 + 1 if pre and gains else None
    t["kw"] = dict(gate_sigmoid=sigmoid, post_norm=post, keep=0.3, scale=0.7, eps=1e-5)
    return t


def reference(t, dtype, pre=True):
    D_ = lambda v: None if v is None else v.double()  # noqa: E731
    x, f, z, dz, dy, gate, gp, gq = (D_(t[k]) for k in ("x", "f", "z", "dz", "dy", "gate", "post_gain", "pre_gain"))
    kw = t["kw"]
    rows, d = f.shape
    keep, scale, eps = kw["keep"], kw["scale"], kw["eps"]
    step = 2.0 ** -8 if dtype == BF16 else U
    es = (d / 64 + 32) * U
    one = torch.ones(d, device="cuda", dtype=torch.float64)
    gp, gq = one if gp is None else gp, one if gq is None else gq
    s, slope = (one, one) if gate is None else (gate, torch.ones_like(gate))
    if kw["gate_sigmoid"]:
        s = torch.sigmoid(gate)
        slope = s * torch.sigmoid(-gate)
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    rf = 1 / torch.sqrt(mean(f * f) + eps) if kw["post_norm"] else torch.ones((rows, 1), device="cuda", dtype=torch.float64)
    er = es if kw["post_norm"] else 0.0
    n = f * rf * gp
    ref, tol = {}, {}
    zz = keep * x + scale * s * n
    dzz = (er + 16 * U) * (scale * s * n).abs() + 2 * U * (keep * x).abs() + U * zz.abs()
    rz = 1 / torch.sqrt(mean(zz * zz) + eps)
    ref["z"], tol["z"] = zz, dzz + step * zz.abs()
    y = zz * rz * gq
    ref["y"] = y
    tol["y"] = (es + 4 * U) * y.abs() + dzz * (rz * gq).abs() + (zz * gq).abs() * rz ** 3 * mean(zz.abs() * dzz) + step * y.abs()
    # backward, from the given z
    D, dD = dz if dz is not None else torch.zeros_like(f), torch.zeros_like(f)
    if dy is not None:
        r = 1 / torch.sqrt(mean(z * z) + eps)
        a, m, mag = dy * gq, mean(dy * gq * z), mean((dy * gq * z).abs())
        D = D + r * (a - z * r * r * m)
        dD = (8 * U + es) * (r * a).abs() + z.abs() * r ** 3 * mag * (es + 3 * es + 8 * U)
        ref["dpre_gain"] = (dy * z * r).sum(0)
        tol["dpre_gain"] = (es + (rows + 40) * U) * (dy * z * r).abs().sum(0) + U * ref["dpre_gain"].abs()
    dD = dD + 2 * U * D.abs()
    ref["dx"], tol["dx"] = keep * D, keep * dD + 2 * U * (keep * D).abs() + step * (keep * D).abs()
    dg = scale * D * n * slope
    ddg = (scale * n * slope).abs() * dD + (er + 32 * U) * dg.abs()
    if gate is not None:
        if gate.dim() == 1:
            ref["dgate"], tol["dgate"] = dg.sum(0), ddg.sum(0) + (rows + 40) * U * dg.abs().sum(0)
        elif gate.shape[1] == 1 and (d > 1 or t["gate"].dtype != t["f"].dtype):
            ref["dgate"], tol["dgate"] = dg.sum(1, keepdim=True), (ddg + es * dg.abs()).sum(1, keepdim=True)
        else:
            ref["dgate"], tol["dgate"] = dg, ddg + step * dg.abs()
    dn = scale * D * s
    ddn = (scale * s).abs() * dD + 16 * U * dn.abs()
    if kw["post_norm"]:
        ref["dpost_gain"] = (dn * f * rf).sum(0)
        tol["dpost_gain"] = (ddn * (f * rf).abs()).sum(0) + (er + (rows + 48) * U) * (dn * f * rf).abs().sum(0)
        b, db = dn * gp, ddn * gp.abs() + 2 * U * (dn * gp).abs()
        m, mag = mean(b * f), mean((b * f).abs())
        ref["df"] = rf * (b - f * rf * rf * m)
        tol["df"] = rf * db + (8 * U + es) * (rf * b).abs() + f.abs() * rf ** 3 * (mag * (4 * es + 8 * U) + mean(db * f.abs()))
    else:
        ref["df"], tol["df"] = dn, ddn
    tol["df"] = tol["df"] + step * ref["df"].abs()
    return ref, tol


def outputs(t, names, fill=7.0):
    like = dict(z=t["f"], y=t["f"], dx=t["f"], df=t["f"], dgate=t["gate"])
    d = t["f"].shape[1]
    return {k: torch.full_like(like[k], fill) if k in like else torch.full((d,), fill, device="cuda") for k in names}


def names_of(t, pre=True):
    fwd = ["z"] + (["y"] if pre else [])
    back = ["dx", "df"] + (["dgate"] if t["gate"] is not None else []) + (["dpost_gain"] if t["kw"]["post_norm"] else [])
    return fwd, back + (["dpre_gain"] if t["dy"] is not None else [])


def run(be, t, fwd, back):
    of, ob = outputs(t, fwd), outputs(t, back)
    torch.cuda.synchronize()
    pre = "y" in fwd
    if fwd:
        be.residual_norm_async(t["x"], t["f"], outputs=of, gate=t["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"] if pre else None, **t["kw"])
    if back:
        be.residual_norm_backward_async(t["z"], t["f"], outputs=ob, dz=t["dz"], dy=t["dy"], gate=t["gate"], post_gain=t["post_gain"],
                                        pre_gain=t["pre_gain"] if t["dy"] is not None else None, **t["kw"])
    be.synchronize()
    return {**of, **ob}


def check(out, ref, tol):
    for k, v in out.items():
        err = (v.double() - ref[k]).abs()
        bad = ~(err <= tol[k] + 1e-300)
        assert not bad.any(), f"{k}: {int(bad.sum())} of {bad.numel()} beyond the tolerance, worst {float((err / tol[k])[bad].max())} of it at {torch.nonzero(bad)[0].tolist()}"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("i,rows,d", [(i, *s) for i, s in enumerate(
    [(1, 1), (3, 2), (1, 64), (5, 63), (4, 65), (7, 128), (2, 257), (24, 512), (600, 512), (33, 513), (9, 1000), (6, 1024), (130, 1025),
     (5, 2047), (3000, 2048), (4, 2049), (3, 4096), (700, 5001), (2, 8192), (2049, 96), (16385, 8), (40, 7)])])
def test_against_definition(be, i, rows, d, dtype):
    for j, gate in enumerate(GATES):
        sigmoid = gate != "none" and (i + j) % 2 == 0
        log(f"residual {rows} x {d} {dtype} {gate} {sigmoid}")
        t = make(rows, d, dtype, gate, sigmoid, post=(i + j) % 4 != 3, gains=i % 5 != 2)
        check(run(be, t, *names_of(t)), *reference(t, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("post,pre,dz", [(True, False, True), (False, False, True), (True, True, False), (False, True, False)])
def test_parts(be, gate, post, pre, dz, dtype):
    """Without the norm behind, without the norm before, without a gradient by other ways."""
    t = make(70, 320, dtype, gate, gate == "row", post, pre)
    if not dz:
        t["dz"] = None
    if not pre:
        t["z"] = None
    ref, tol = reference(t, dtype)
    check(run(be, t, *names_of(t, pre)), ref, tol)


@pytest.mark.parametrize("d", [1000, 2048, 5000])
@pytest.mark.parametrize("post,pre", [(True, False), (False, True), (False, False)])
def test_wide_rows_with_one_sum_each(be, d, post, pre):
    """Rows of several waves, many a block, with one reduction a row (or none): the waves' sums have places of their own from row to row."""
    t = make(6000, d, F32, "none", False, post, pre)
    if not pre:
        t["z"] = None
    check(run(be, t, *names_of(t, pre)), *reference(t, F32))


@pytest.mark.parametrize("gate", GATES)
def test_outputs_apart(be, gate):
    t = make(77, 320, F32, gate, True and gate != "none")
    fwd, back = names_of(t)
    whole = run(be, t, fwd, back)
    for k in fwd:
        assert torch.equal(run(be, t, [k], [])[k], whole[k])
    for k in back:
        assert torch.equal(run(be, t, [], [k])[k], whole[k]), k


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("offset,extra", [(1, 3), (8, 8), (0, 1)])
@pytest.mark.parametrize("gate", ["channel", "element"])
def test_strides_and_alignment(be, offset, extra, dtype, gate):
    """Results of rows at a stride within the tolerance, nothing written between them."""
    rows, d = 37, 200
    t = make(rows, d, dtype, gate)
    ref, tol = reference(t, dtype)
    stores = []

    def spaced(v):
        store = torch.full((offset + rows * (d + extra),), 5.0, device="cuda", dtype=v.dtype)
        w = store[offset:].view(rows, d + extra)[:, :d]
        w.copy_(v)
        stores.append((store, w))
        return w
    u = dict(t)
    for k in ("x", "f", "z", "dz", "dy"):
        u[k] = spaced(t[k])
    if gate == "element":
        u["gate"] = spaced(t["gate"])
    names = ["z", "y", "dx", "df", "dgate", "dpost_gain", "dpre_gain"]
    out = {k: spaced(torch.zeros_like(t["f"])) if k in ("z", "y", "dx", "df") or (k == "dgate" and gate == "element") else torch.zeros(d, device="cuda")
           for k in names}
    torch.cuda.synchronize()
    kw = dict(gate=u["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"], **t["kw"])
    be.residual_norm_async(u["x"], u["f"], outputs={k: out[k] for k in names[:2]}, **kw)
    be.residual_norm_backward_async(u["z"], u["f"], dz=u["dz"], dy=u["dy"], outputs={k: out[k] for k in names[2:]}, **kw)
    be.synchronize()
    check(out, ref, tol)
    for store, w in stores:
        w.fill_(5.0)
        assert bool((store == 5.0).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,d", [(50, 512), (9, 2048), (5, 77)])
def test_in_place(be, rows, d, dtype):
    """z in x's place and dx in dz's give the bits that they have elsewhere."""
    t = make(rows, d, dtype, "channel")
    out = run(be, t, *names_of(t))
    x, dz = t["x"].clone(), t["dz"].clone()
    torch.cuda.synchronize()
    kw = dict(gate=t["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"], **t["kw"])
    be.residual_norm_async(x, t["f"], outputs=dict(z=x), **{**kw, "pre_gain": None})
    be.residual_norm_backward_async(t["z"], t["f"], dz=dz, dy=t["dy"], outputs=dict(dx=dz), **kw)
    be.synchronize()
    assert torch.equal(x, out["z"]) and torch.equal(dz, out["dx"])


def test_rows_of_zeros_and_gates_at_the_ends(be):
    """A block that gives nothing; logits so far out that the gate is 0 or 1 and its slope 0."""
    t = make(9, 100, F32, "element", True)
    t["f"][4] = 0
    t["gate"][:, 0], t["gate"][:, 1], t["gate"][:, 2], t["gate"][:, 3] = 200.0, -200.0, float("inf"), -float("inf")
    ref, tol = reference(t, F32)
    out = run(be, t, *names_of(t))
    check(out, ref, {k: v + 1e-38 for k, v in tol.items()})
    assert float(out["dgate"][:, 2:4].abs().max()) == 0.0


def test_a_row_that_is_not_a_number_stays_alone(be):
    for d in (512, 2048):
        t = make(40, d, F32, "element")
        clean = run(be, t, *names_of(t))
        t["f"][7, 3] = float("nan")
        t["z"][9, 5] = float("inf")
        out = run(be, t, *names_of(t))
        keep = [i for i in range(40) if i not in (7, 9)]
        for k in ("z", "y", "dx", "df", "dgate"):
            assert torch.equal(out[k][keep], clean[k][keep]), k
        assert bool(torch.isnan(out["z"][7]).any()) and bool(torch.isnan(out["df"][7]).all())


def test_gradients_against_differences(be):
    """<dz, z> + <dy, y> moves along a direction as the gradients say: central differences of the kernels' own forward, whose steps
    of 2^-7 leave 2^-14 times third derivatives (a few units), and whose roundings leave 2^-24 / 2^-7 of sums of 640 terms of a few units."""
    rows, d, h = 5, 128, 2.0 ** -7
    for gate in GATES:
        t = make(rows, d, F32, gate, gate != "none")
        t["x"], t["f"] = t["x"].clamp(-2, 2), t["f"].clamp(-2, 2) + 0.5
        g = torch.Generator(device="cuda").manual_seed(5)

        def forward(u):
            out = outputs(u, ["z", "y"])
            torch.cuda.synchronize()
            be.residual_norm_async(u["x"], u["f"], outputs=out, gate=u["gate"], post_gain=u["post_gain"], pre_gain=u["pre_gain"], **u["kw"])
            be.synchronize()
            return out
        t["z"] = forward(t)["z"]
        grads = run(be, t, [], names_of(t)[1])
        for k, dk in (("x", "dx"), ("f", "df"), ("gate", "dgate"), ("post_gain", "dpost_gain"), ("pre_gain", "dpre_gain")):
            if t[k] is None:
                continue
            v = torch.randn(t[k].shape, device="cuda", generator=g)
            value = []
            for sign in (1, -1):
                o = forward({**t, k: t[k] + sign * h * v})
                value.append(float((o["z"].double() * t["dz"].double()).sum() + (o["y"].double() * t["dy"].double()).sum()))
            want = float((grads[dk].double() * v.double()).sum())
            scale = float((grads[dk].double() * v.double()).abs().sum())
            assert abs((value[0] - value[1]) / (2 * h) - want) <= 4e-3 * scale + 0.02, (gate, k)


def test_equal_calls_give_equal_bits(be):
    t = make(3000, 512, BF16, "channel", True)
    a, b = run(be, t, *names_of(t)), run(be, t, *names_of(t))
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_captured(be):
    """Forward and backward in one graph, replayed on new inputs between eager calls of the same context."""
    t = make(100, 512, F32, "channel")
    fwd, back = names_of(t)
    run(be, t, fwd, back)  # the workspace
    of, ob = outputs(t, fwd), outputs(t, back)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(s.cuda_stream)
    try:
        g = torch.cuda.CUDAGraph()
        kw = dict(gate=t["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"], **t["kw"])
        with torch.cuda.graph(g, stream=s):
            be.residual_norm_async(t["x"], t["f"], outputs=of, **kw)
            be.residual_norm_backward_async(of["z"], t["f"], dz=t["dz"], dy=t["dy"], outputs=ob, **kw)
        for k in range(3):
            t["x"].mul_(-1.5), t["f"].add_(0.25)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                g.replay()
            torch.cuda.synchronize()
            got = {n: v.clone() for n, v in {**of, **ob}.items()}
            want = run(be, {**t, "z": of["z"]}, fwd, back)
            assert all(torch.equal(got[n], want[n]) for n in want), k
        del g
    finally:
        torch.cuda.synchronize()
        be.set_stream(None)


def test_a_workspace_that_would_grow_under_capture_is_refused():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    t = make(100, 512, F32)
    ob = outputs(t, ["dpre_gain"])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    b.set_stream(s.cuda_stream)
    g, refused = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(g, stream=s):
        try:
            b.residual_norm_backward_async(t["z"], t["f"], dy=t["dy"], pre_gain=t["pre_gain"], outputs=ob)
        except AdnError as e:
            refused.append(e.code)
    torch.cuda.synchronize()
    b.close()
    assert refused == [ADN_E_CAPACITY]


def test_empty_batches(be):
    """Nothing to read: row outputs are left alone, column sums are 0."""
    t = make(0, 96, F32, "channel")
    out = outputs(t, ["dx", "df", "dgate", "dpost_gain", "dpre_gain"])
    torch.cuda.synchronize()
    be.residual_norm_async(t["x"], t["f"], outputs=outputs(t, ["z", "y"]), gate=t["gate"])
    be.residual_norm_backward_async(t["z"], t["f"], dz=t["dz"], dy=t["dy"], gate=t["gate"], outputs=out)
    be.synchronize()
    assert all(float(out[k].abs().sum()) == 0 for k in ("dgate", "dpost_gain", "dpre_gain"))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_offsets_beyond_32_bits(be, dtype):
    """Rows at a stride that takes the last ones past 2^32 elements."""
    torch.cuda.empty_cache()
    rows, d, stride = 9, 300, 1 << 29
    t = make(rows, d, dtype, "element")
    ref, tol = reference(t, dtype)
    store = torch.zeros(8 * stride + 4096, device="cuda", dtype=dtype)
    names, u = ["x", "f", "z", "dz", "dy", "gate"], dict(t)
    place = lambda k: store[k * 304:].as_strided((rows, d), (stride, 1))  # noqa: E731
    for k, n in enumerate(names):
        u[n] = place(k)
        u[n].copy_(t[n])
    out = {n: place(6 + k) for k, n in enumerate(["z", "y", "dx", "df", "dgate"])}
    torch.cuda.synchronize()
    kw = dict(gate=u["gate"], post_gain=t["post_gain"], pre_gain=t["pre_gain"], **t["kw"])
    be.residual_norm_async(u["x"], u["f"], outputs={k: out[k] for k in ("z", "y")}, **kw)
    be.residual_norm_backward_async(u["z"], u["f"], dz=u["dz"], dy=u["dy"], outputs={k: out[k] for k in ("dx", "df", "dgate")}, **kw)
    be.synchronize()
    check(out, ref, tol)
    del store, u, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,d,dtype", [(40000, 2048, BF16), (50000, 512, F32)])
def test_streaming_sizes(be, rows, d, dtype):
    """More bytes than the caches hold (other loads): the first, middle and last rows, and the column sums."""
    t = make(rows, d, dtype, "channel", True)
    out = run(be, t, *names_of(t))
    ref, tol = reference(t, dtype)
    check(out, ref, tol)


# ---- refusals -------------------------------------------------------------------------------------
def args(**kw):
    x, v = torch.zeros((4, 8), device="cuda"), torch.zeros(8, device="cuda")
    p, q = x.data_ptr(), v.data_ptr()
    a = dict(rows=4, d=8, dtype=0, gate_kind=0, post_norm=1, keep=1.0, scale=1.0, eps=1e-6, x=p, x_stride=8, f=p, f_stride=8, z=p, z_stride=8,
             y=p, y_stride=8, dz=p, dz_stride=8, dy=p, dy_stride=8, dx=p, dx_stride=8, df=p, df_stride=8, dgate_stride=8, gate_stride=8)
    a.update({k: (q + 2 if val == "odd" else q if val == "vector" else val) for k, val in kw.items()})
    return _lib.AdnResidualNormArgs(**a), (x, v)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=(1 << 24) + 1), dict(d=0), dict(d=8193), dict(dtype=2), dict(gate_kind=4), dict(gate_sigmoid=2),
                                dict(post_norm=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(reserved=1), dict(gate="vector"), dict(gate_sigmoid=1),
                                dict(gate_kind=1), dict(gate_kind=2), dict(gate_kind=3), dict(post_norm=0, post_gain="vector"), dict(f=None),
                                dict(f_stride=7), dict(f_stride=(1 << 32) + 1), dict(post_gain="odd"), dict(pre_gain="odd"), dict(gate_kind=1, gate="odd")])
@pytest.mark.parametrize("entry", ["adn_residual_norm_async", "adn_residual_norm_backward_async"])
def test_refused_by_both(be, kw, entry):
    import ctypes as C
    a, keep = args(**kw)
    assert getattr(_lib.lib(), entry)(be._ctx, C.byref(a)) == ADN_E_INVALID
    assert _lib.lib().adn_last_error().decode()
    del keep


@pytest.mark.parametrize("entry,kw", [
    ("adn_residual_norm_async", dict(x=None)), ("adn_residual_norm_async", dict(z=None, y=None)), ("adn_residual_norm_async", dict(y=None, pre_gain="vector")),
    ("adn_residual_norm_async", dict(z_stride=16)), ("adn_residual_norm_backward_async", dict(dz=None, dy=None)),
    ("adn_residual_norm_backward_async", dict(z=None)), ("adn_residual_norm_backward_async", dict(dx=None, df=None)),
    ("adn_residual_norm_backward_async", dict(dgate="vector")), ("adn_residual_norm_backward_async", dict(dy=None, dpre_gain="vector")),
    ("adn_residual_norm_backward_async", dict(post_norm=0, dpost_gain="vector")), ("adn_residual_norm_backward_async", dict(dx_stride=16)),
    ("adn_residual_norm_backward_async", dict(dpost_gain="odd"))])
def test_refused_by_one(be, entry, kw):
    import ctypes as C
    a, keep = args(**kw)
    assert getattr(_lib.lib(), entry)(be._ctx, C.byref(a)) == ADN_E_INVALID
    del keep
