"""AdamW over a list of tensors and the norm of its gradients against the definition in 64 bits (needs an MI355X).

Tolerances, u = 2^-24, states of 32 bits.  m' = b1 m + c1 g: the constants rounded to fp32 (u each), g times the coefficient
(its rounding and the product's: 2 u), two products and a sum: 6 u (|b1 m| + |c1 g|).  v' in the same way, g twice: 10 u v'.
The way A = m' / bc1 / (sqrt(v' / bc2) + eps): half of v's 10 u, the corrections (expm1 2 u, its argument rounded u, the reciprocal or
root 2 u: 5 u each), root and reciprocal to 1 ulp (2 u each), three products and a sum: 30 u relative, and m's error over the
denominator.  p' = p - lr (A + wd p): lr and lr_scale's product 2 u, wd u, the sums u each: lr (36 u |A| + dA + 6 u |wd p|) + 2 u (|p| + |p'|).
States of 8 bits: codes and scales exactly (their arithmetic is in 64 bits); m' and v' rounded once to fp32 in the way to p'.
A copy is p' rounded once: half a step, 2^-8 relative, behind p's tolerance."""
import numpy as np
import pytest
import torch

from aideen_amd import _lib, synth
from aideen_amd._lib import ADN_E_INVALID, AdnError
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
G64, M1, M2 = np.uint64(0x9E3779B97F4A7C15), np.uint64(0xBF58476D1CE4E5B9), np.uint64(0x94D049BB133111EB)


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


# ---- the definition on the host ----------------------------------------------------------------
def mix64(x):
    x = (x ^ (x >> np.uint64(30))) * M1
    x = (x ^ (x >> np.uint64(27))) * M2
    return x ^ (x >> np.uint64(31))


def random_bits(seed, step, block, n):
    """The 16 bits of m and of v of the n values of a block, counted from the list's first."""
    with np.errstate(over="ignore"):
        key = mix64(np.uint64(seed) + np.uint64(step) * G64)
        a = np.uint32(mix64(key + np.uint64(block + 1) * G64) & np.uint64(0xFFFFFFFF))
        r = a + np.arange(n, dtype=np.uint32) * np.uint32(0x9E3779B9)
        r = (r ^ (r >> np.uint32(16))) * np.uint32(0x7FEB352D)
        r = (r ^ (r >> np.uint32(15))) * np.uint32(0x846CA68B)
        r = r ^ (r >> np.uint32(16))
    return (r & np.uint32(0xFFFF)).astype(np.float64), (r >> np.uint32(16)).astype(np.float64)


def to_codes(x, bits, floor):
    """(values of the codes, scale) of a block of doubles."""
    top = np.abs(x).max()
    E = max(int(np.frexp(top)[1]) - 1, -110) if top > 0 else -110
    scale = 2.0 ** (E - 7)
    a = np.abs(x) / scale
    step = 2.0 ** (np.maximum(np.frexp(np.maximum(a, 2.0 ** -30))[1] - 1, -6) - 3.0)
    q = np.floor(a / step + bits / 65536) * step
    if floor:
        q = np.where((x > 0) & (q == 0), 2.0 ** -9, q)
    return np.where(x < 0, -q, q), scale


def reference(state, cfg):
    """(what each tensor of the list holds after the step, the tolerances of p): lists of dicts in 64 bits."""
    b1, b2, eps, lr, seed, t, coef = (cfg[k] for k in ("b1", "b2", "eps", "lr", "seed", "t", "coef"))
    out, block = [], 0
    for s in state:
        p, g = s["p"], s["g"] * coef
        m, v = b1 * s["m"] + (1 - b1) * g, b2 * s["v"] + (1 - b2) * g * g
        den = np.sqrt(v / (1 - b2 ** t)) + eps
        away = m / (1 - b1 ** t) / den
        rate, wd = lr * s["lr_scale"], s["wd"]
        new = p - rate * (away + wd * p)
        dm = 6 * U * (np.abs(b1 * s["m"]) + np.abs((1 - b1) * g))
        tol = rate * (36 * U * np.abs(away) + dm / (1 - b1 ** t) / den + 6 * U * np.abs(wd * p)) + 2 * U * (np.abs(p) + np.abs(new))
        r = dict(p=new, tol_p=tol + 1e-45, m=m, v=v, tol_m=dm + 1e-45, tol_v=10 * U * v + 1e-45)
        if cfg["bits"] == 8:
            blocks = -(-p.size // 256)
            r["m8"], r["v8"], r["ms"], r["vs"] = np.zeros(p.size), np.zeros(p.size), np.zeros(blocks), np.zeros(blocks)
            for i in range(blocks):
                a, b = i * 256, min(p.size, i * 256 + 256)
                lo, hi = random_bits(seed, t - 1, block + i, b - a)
                r["m8"][a:b], r["ms"][i] = to_codes(m[a:b], lo, False)
                r["v8"][a:b], r["vs"][i] = to_codes(v[a:b], hi, True)
            block += blocks
        out.append(r)
    return out


class List:
    """A list of tensors on the GPU, each behind `offset` values of a larger buffer, with guards around it."""

    def __init__(self, sizes, bits=32, grad=lambda i: F32, copy=lambda i: False, offset=0, seed=0, spread=2.0):
        g = torch.Generator().manual_seed(seed * 7 + len(sizes))
        self.sizes, self.bits, self.stores = sizes, bits, []
        mk = self._mk
        rnd = lambda n: torch.randn(n, generator=g, dtype=torch.float64)  # noqa: E731
        self.p = [mk(rnd(n) * 0.05, F32, offset) for n in sizes]
        mag = [torch.pow(10.0, -3 + spread * (torch.rand(n, generator=g, dtype=torch.float64) - 0.5)) for n in sizes]
        self.g = [mk(rnd(n) * a, grad(i), offset) for i, (n, a) in enumerate(zip(sizes, mag))]
        m = [rnd(n) * a * 0.3 for n, a in zip(sizes, mag)]
        v = [torch.rand(n, generator=g, dtype=torch.float64) * a * a for n, a in zip(sizes, mag)]
        self.copy = [mk(torch.zeros(n), BF16, offset) if copy(i) else None for i, n in enumerate(sizes)]
        self.step = torch.tensor([16 + seed], device="cuda", dtype=torch.int32)
        self.ms = self.vs = None
        if bits == 8:
            self.ms = [torch.pow(2.0, torch.randint(-14, -8, (-(-n // 256),), generator=g)).float().cuda() for n in sizes]
            self.vs = [torch.pow(2.0, torch.randint(-28, -20, (-(-n // 256),), generator=g)).float().cuda() for n in sizes]
            self.m = [mk((rnd(n) * 60).clamp(-256, 256).float(), F8, offset) for n in sizes]
            self.v = [mk((rnd(n).abs() * 60).clamp(2.0 ** -9, 256).float(), F8, offset) for n in sizes]
        else:
            self.m, self.v = [mk(x, F32, offset) for x in m], [mk(x, F32, offset) for x in v]
        self.lr_scale, self.wd = [1.0 + 0.25 * (i % 3) for i in range(len(sizes))], [0.1 * (i % 2) for i in range(len(sizes))]

    def _mk(self, x, dtype, offset):
        n, size = x.numel(), torch.empty(0, dtype=dtype).element_size()
        raw = torch.full(((offset + n + 5) * size,), 0x35, device="cuda", dtype=torch.uint8)
        t = raw.view(dtype)[offset:offset + n]
        t.copy_(x.to(F32).to(dtype))
        self.stores.append((raw, offset * size, n * size))
        return t

    def guards(self):
        return all(bool((raw[:a] == 0x35).all()) and bool((raw[a + n:] == 0x35).all()) for raw, a, n in self.stores)

    def host(self):
        def dec(t, s, n):
            x = t.float().double().cpu().numpy()
            return x if s is None else x * np.repeat(s.double().cpu().numpy(), 256)[:n]
        return [dict(p=self.p[i].double().cpu().numpy(), g=self.g[i].double().cpu().numpy(),
                     m=dec(self.m[i], self.ms and self.ms[i], n), v=dec(self.v[i], self.vs and self.vs[i], n),
                     lr_scale=self.lr_scale[i], wd=self.wd[i]) for i, n in enumerate(self.sizes)]

    def optimizer(self, be, seed=5, betas=(0.9, 0.999), eps=1e-8):
        kw = dict(m_scale=self.ms, v_scale=self.vs) if self.bits == 8 else {}
        return be.adamw(self.p, self.g, m=self.m, v=self.v, step=self.step, copies=self.copy, betas=betas, eps=eps, seed=seed,
                        weight_decay=self.wd, lr_scale=self.lr_scale, **kw)

    def check(self, before, cfg):
        ref = reference(before, cfg)
        for i, (r, n) in enumerate(zip(ref, self.sizes)):
            if not n:
                continue
            p = self.p[i].double().cpu().numpy()
            err = np.abs(p - r["p"])
            assert (err <= r["tol_p"]).all(), f"p of tensor {i}: {np.max(err / r['tol_p'])} tolerances"
            if self.copy[i] is not None:
                assert torch.equal(self.copy[i], self.p[i].to(BF16))
            if self.bits == 8:
                for name, codes, scale in (("m", self.m[i], self.ms[i]), ("v", self.v[i], self.vs[i])):
                    assert np.array_equal(scale.double().cpu().numpy(), r[name + "s"]), f"{name}_scale of tensor {i}"
                    got = codes.float().double().cpu().numpy()
                    assert np.array_equal(got, r[name + "8"]), f"{name} of tensor {i}: {(got != r[name + '8']).sum()} codes differ"
            else:
                for name in "mv":
                    got = getattr(self, name)[i].double().cpu().numpy()
                    assert (np.abs(got - r[name]) <= r["tol_" + name]).all(), f"{name} of tensor {i}"
        assert self.guards()


def cfg_of(lst, lr=1e-3, coef=1.0, seed=5, betas=(0.9, 0.999), eps=1e-8):
    return dict(bits=lst.bits, b1=betas[0], b2=betas[1], eps=eps, lr=lr, coef=coef, seed=seed, t=int(lst.step[0]) + 1)


def one_step(be, lst, lr=1e-3, seed=5, betas=(0.9, 0.999), eps=1e-8, **kw):
    opt = lst.optimizer(be, seed, betas, eps)
    cfg, before = cfg_of(lst, lr, 1.0, seed, betas, eps), lst.host()
    torch.cuda.synchronize()
    opt.step_async(lr=lr, **kw)
    be.synchronize()
    assert int(lst.step[0]) == cfg["t"]
    return cfg, before, opt


SIZES = [[1], [0, 3, 0], [255, 256, 257], [64, 1023, 1, 1024, 1025, 2], [4097, 5], [70001], [33] * 70, [20000, 3, 50000, 777]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_against_definition(be, sizes, bits):
    log(f"adamw {bits} {sizes[:4]}")
    for offset in (0, 1):
        lst = List(sizes, bits, grad=lambda i: BF16 if i % 3 == 1 else F32, copy=lambda i: i % 2 == 0, offset=offset, seed=len(sizes))
        cfg, before, _ = one_step(be, lst)
        lst.check(before, cfg)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_streaming_list(be, bits):
    """More values than the caches hold, so other loads and larger chunks; a tensor's end inside one."""
    n = (20 << 20) + 77
    lst = List([3, n], bits, grad=lambda i: BF16)
    keep = [t.clone() for t in (lst.p[1], lst.g[1], lst.m[1], lst.v[1])] + ([lst.ms[1].clone(), lst.vs[1].clone()] if bits == 8 else [])
    cfg, _, _ = one_step(be, lst)
    for a in (0, 256 * 4000, n // 256 * 256 - 512):  # parts of it, from a block's start
        b = min(n, a + 1024)
        s = [slice(a, b), slice(a // 256, -(-b // 256))]
        before = [dict(p=keep[0][s[0]].double().cpu().numpy(), g=keep[1][s[0]].double().cpu().numpy(), lr_scale=1.25, wd=0.1)]
        for k, t, sc in (("m", keep[2], 4), ("v", keep[3], 5)):
            x = t[s[0]].float().double().cpu().numpy()
            before[0][k] = x * np.repeat(keep[sc][s[1]].double().cpu().numpy(), 256)[:b - a] if bits == 8 else x
        ref = reference(before, dict(cfg, bits=32))[0]
        assert (np.abs(lst.p[1][s[0]].double().cpu().numpy() - ref["p"]) <= ref["tol_p"]).all()
        if bits == 8:
            for i in range(s[1].start, s[1].stop):
                c, d = i * 256 - a, min(b, i * 256 + 256) - a
                lo, hi = random_bits(cfg["seed"], cfg["t"] - 1, 1 + i, d - c)  # the first tensor is one block
                for codes, scale, x, bit, floor in ((lst.m, lst.ms, ref["m"], lo, False), (lst.v, lst.vs, ref["v"], hi, True)):
                    want, sc = to_codes(x[c:d], bit, floor)
                    assert float(scale[1][i]) == sc
                    assert np.array_equal(codes[1][a + c:a + d].float().double().cpu().numpy(), want)
        else:
            assert (np.abs(lst.m[1][s[0]].double().cpu().numpy() - ref["m"]) <= ref["tol_m"]).all()
            assert (np.abs(lst.v[1][s[0]].double().cpu().numpy() - ref["v"]) <= ref["tol_v"]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas,eps", [((0.0, 0.0), 1e-8), ((0.95, 0.9999), 1e-15), ((0.5, 0.5), 1.0), ((0.9, 0.999), 1e-30)])
def test_constants(be, bits, betas, eps):
    lst = List([700, 40], bits, spread=10.0)
    cfg, before, _ = one_step(be, lst, betas=betas, eps=eps)
    lst.check(before, cfg)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("steps", [0, 1, 999, 2 ** 31 - 2])
def test_counter(be, bits, steps):
    lst = List([300], bits)
    lst.step.fill_(steps)
    cfg, before, _ = one_step(be, lst)
    lst.check(before, cfg)


@pytest.mark.parametrize("bits", [32, 8])
def test_new_state_and_several_steps(be, bits):
    """From zeros, the state that the optimizer makes; then four steps, each from the one before."""
    lst = List([600, 31, 0], bits)
    opt = be.adamw(lst.p, lst.g, state_bits=bits, weight_decay=lst.wd, lr_scale=lst.lr_scale, seed=9)
    lst.m, lst.v, lst.ms, lst.vs, lst.step, lst.copy = opt.m, opt.v, opt.m_scale if bits == 8 else None, opt.v_scale if bits == 8 else None, opt.step, [None] * 3
    assert int(opt.step[0]) == 0 and all(float(t.float().abs().sum()) == 0 for t in opt.m + opt.v)
    for k in range(4):
        cfg, before = cfg_of(lst, 2e-3, 1.0, 9), lst.host()
        opt.step_async(lr=2e-3)
        be.synchronize()
        lst.check(before, cfg)
        for t in lst.g:
            t.mul_(-0.7)
        torch.cuda.synchronize()
    assert int(opt.step[0]) == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_stay(be, bits):
    """No gradient and no state: nothing moves without decay, codes stay 0."""
    lst = List([300, 5], bits)
    for t in lst.g + lst.m + lst.v:
        t.view(torch.uint8).zero_()
    lst.wd = [0.0, 0.0]
    keep = [t.clone() for t in lst.p]
    one_step(be, lst)
    assert all(torch.equal(a, b) for a, b in zip(keep, lst.p))
    assert all(float(t.float().abs().sum()) == 0 for t in lst.m + lst.v)
    if bits == 8:
        assert all(float(t) == 2.0 ** -117 for s in lst.ms + lst.vs for t in s)


def test_small_v_keeps_a_code(be):
    """Beside a value 2^40 times as large, one that is not zero has the smallest code and not none."""
    lst = List([256], 8)
    lst.g[0].fill_(1e-6)
    lst.g[0][7] = 1e3
    lst.g[0][9] = 0.0
    for t in lst.m + lst.v:
        t.view(torch.uint8).zero_()
    cfg, before, _ = one_step(be, lst)
    lst.check(before, cfg)
    v = lst.v[0].float()
    assert float(v[0]) == 2.0 ** -9 and float(v[9]) == 0.0 and 128 <= float(v[7]) <= 256


def test_rounding_follows_the_average(be):
    """v from 65536 alike values, each moved by a hundredth of a code's step or less a step: the mean of what 40 steps leave is the exact
    one within five deviations.  A step's error is a code's step times a coin, at most half a code step deviation, 1/16 of v: 40 of
    them less than 0.4 v, over 256 (the root of the count) 0.0016 v; rounding to nearest would not have moved."""
    n = 65536
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(F8) for _ in range(2))
    v.copy_(torch.full((n,), 128.0))
    s = [torch.full((n // 256,), 2.0 ** -30, device="cuda") for _ in range(2)]
    opt = be.adamw([p], [g], m=[m], v=[v], m_scale=[s[0]], v_scale=[s[1]], step=torch.zeros(1, device="cuda", dtype=torch.int32), seed=3)
    want = 128 * 2.0 ** -30
    torch.cuda.synchronize()
    for _ in range(40):
        opt.step_async(lr=0.0)
        want = 0.999 * want + 0.001 * float(g[0]) ** 2
    be.synchronize()
    got = float((v.float().double().view(-1, 256) * s[1].double()[:, None]).mean())
    assert abs(got - want) < 5 * 0.0016 * want
    assert want > 1.2 * 128 * 2.0 ** -30


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_gradient_that_is_not_a_number(be, bits, bad):
    """Without a norm it reaches its own value (and, in 8 bits, its block's states); other blocks do as ever."""
    lst, clean = List([1000, 10], bits), List([1000, 10], bits)
    lst.g[0][300] = bad
    one_step(be, clean)
    one_step(be, lst)
    same = torch.ones(1000, dtype=torch.bool, device="cuda")
    same[300] = False
    assert torch.equal(lst.p[0][same], clean.p[0][same]) and torch.equal(lst.p[1], clean.p[1])
    assert bool(torch.isnan(lst.p[0][300]))
    if bits == 8:
        assert bool(torch.isnan(lst.ms[0][1])) and bool(torch.isnan(lst.vs[0][1]))
        others = [0, 2, 3]
        assert torch.equal(lst.ms[0][others], clean.ms[0][others]) and torch.equal(lst.vs[0][others], clean.vs[0][others])
        same[256:512] = False
    for a, b in ((lst.m, clean.m), (lst.v, clean.v)):
        assert torch.equal(a[0][same].float(), b[0][same].float())


def test_moments_at_the_end_of_fp32(be):
    """m of 2^127 and more could be rounded to 2^128: its block is not a number; half of that is."""
    for g, bad in ((3.0e38, True), (1.6e38, False)):
        lst = List([256], 8)
        lst.g[0].fill_(0)
        lst.g[0][3] = g
        one_step(be, lst, betas=(0.0, 0.999))
        assert bool(torch.isnan(lst.ms[0][0])) == bad and bool(torch.isnan(lst.vs[0][0]))
        if not bad:
            assert bool(torch.isfinite(lst.m[0].float() * lst.ms[0]).all())


def test_v_beyond_fp32(be):
    lst = List([256], 8)
    lst.g[0][3] = 1e21
    one_step(be, lst)
    assert bool(torch.isnan(lst.vs[0][0])) and bool(torch.isfinite(lst.ms[0][0])) and bool(torch.isfinite(lst.p[0]).all())


# ---- the norm and what a step does with it --------------------------------------------------------
@pytest.mark.parametrize("sizes", [[], [0], [1], [3, 0, 4], [64, 65, 1024, 1023], [100000], [17] * 5000, [3000000, 1, 2500001]],
                         ids=lambda s: f"{len(s)}x{s[0] if s else 0}")
def test_grad_norm(be, sizes):
    """The sum in 64 bits is within 1e-10 of any other order's; one rounding to fp32: half a step and that."""
    log(f"norm {len(sizes)} {sizes[:3]}")
    for offset in (0, 3):
        store = torch.randn(sum(sizes) + offset * (len(sizes) + 1) + 8, device="cuda") * 1e-2
        grads, at = [], offset
        for i, n in enumerate(sizes):
            t = store[at:at + n]
            grads.append(t.to(BF16) if i % 2 and not offset else t)
            at += n + offset
        norm, want = torch.full((1,), 7.0, device="cuda"), 0.0
        if sizes:
            want = float(torch.stack([t.double().square().sum() for t in grads]).sum().sqrt())
        torch.cuda.synchronize()
        opt = be.adamw(None, grads)
        for _ in range(2):
            opt.grad_norm_async(norm)
            be.synchronize()
            assert abs(float(norm) - want) <= (U + 1e-10) * want


@pytest.mark.parametrize("big", [1e19, 3e38, 1e-30])
def test_norm_of_extreme_values(be, big):
    g = torch.full((3,), big, device="cuda")
    norm = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    be.adamw(None, [g]).grad_norm_async(norm)
    be.synchronize()
    want = float((g.double().square().sum().sqrt()).float())
    assert abs(float(norm) - want) <= 2 * U * want or (want == float("inf") and float(norm) == want)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm,scale", [(0.5, 1.0), (1e9, 1.0), (0.01, 0.125), (0.0, 0.125)])
def test_clipped(be, bits, max_norm, scale):
    lst = List([5000, 257], bits)
    opt, norm = lst.optimizer(be), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    opt.grad_norm_async(norm)
    be.synchronize()
    coef = scale * (min(1.0, max_norm / (float(norm) * scale + 1e-6)) if max_norm else 1.0)
    cfg, before = cfg_of(lst, coef=coef), lst.host()
    opt.step_async(lr=1e-3, grad_norm=norm, max_norm=max_norm, grad_scale=scale)
    be.synchronize()
    lst.check(before, cfg)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_skipped(be, bits, bad):
    """A norm that is not finite: nothing is written, the counter stays; the next step is an ordinary one."""
    lst = List([300, 2000], bits, copy=lambda i: True)
    lst.g[1][1234] = bad
    opt, norm = lst.optimizer(be), torch.zeros(1, device="cuda")
    keep = [raw.clone() for raw, _, _ in lst.stores] + [lst.step.clone()] + [t.clone() for t in (lst.ms or []) + (lst.vs or [])]
    torch.cuda.synchronize()
    opt.grad_norm_async(norm)
    opt.step_async(lr=1e-3, grad_norm=norm, max_norm=1.0)
    be.synchronize()
    assert not np.isfinite(float(norm))
    now = [raw for raw, _, _ in lst.stores] + [lst.step] + (lst.ms or []) + (lst.vs or [])
    assert all(torch.equal(a, b) for a, b in zip(keep, now))
    lst.g[1][1234] = 0.5
    torch.cuda.synchronize()
    opt.grad_norm_async(norm)
    be.synchronize()
    coef = min(1.0, 1.0 / (float(norm) + 1e-6))
    cfg, before = cfg_of(lst, coef=coef), lst.host()
    opt.step_async(lr=1e-3, grad_norm=norm, max_norm=1.0)
    be.synchronize()
    lst.check(before, cfg)


# ---- how a program uses it --------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [32, 8])
def test_equal_calls_give_equal_bits_and_states_can_be_restored(be, bits):
    a, b = List([9000, 77], bits), List([9000, 77], bits, offset=3)
    oa, ob = a.optimizer(be), b.optimizer(be)
    torch.cuda.synchronize()
    for _ in range(3):
        oa.step_async(lr=1e-3)
    ob.step_async(lr=1e-3)
    ob.close()
    ob = b.optimizer(be)  # the states alone carry a run on
    ob.step_async(lr=1e-3)
    ob.step_async(lr=1e-3)
    be.synchronize()
    for x, y in zip(a.p + a.m + a.v + [a.step], b.p + b.m + b.v + [b.step]):
        assert torch.equal(x.contiguous().view(-1).view(torch.uint8), y.contiguous().clone().view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured(be, bits):
    """Norm and step in one graph, the rate and the counter on the device: each replay against an eager twin's step."""
    a, b = List([5000, 300], bits), List([5000, 300], bits)
    oa, ob = a.optimizer(be), b.optimizer(be)
    na, nb, lr = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda"), torch.full((1,), 1e-3, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(s.cuda_stream)
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            oa.grad_norm_async(na)
            oa.step_async(lr=lr, grad_norm=na, max_norm=0.5)
        for k in range(4):
            with torch.cuda.stream(s):
                lr.fill_(1e-3 / (k + 1))
                for x, y in zip(a.g, b.g):
                    x.mul_(-1.1), y.mul_(-1.1)
                g.replay()
            torch.cuda.synchronize()
            ob.grad_norm_async(nb)
            ob.step_async(lr=lr, grad_norm=nb, max_norm=0.5)
            be.synchronize()
            assert torch.equal(na, nb) and int(a.step) == int(b.step) == 17 + k
            for x, y in zip(a.p + a.m + a.v, b.p + b.m + b.v):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        del g
    finally:
        torch.cuda.synchronize()
        be.set_stream(None)


def test_two_optimizers_of_a_context_and_a_list_without_values(be):
    a, b = List([2000], 32), List([2000], 8)
    oa, ob = a.optimizer(be), b.optimizer(be)
    empty = be.adamw([torch.zeros(0, device="cuda")], [torch.zeros(0, device="cuda")])
    none = be.adamw([], [])
    ca, cb, ha, hb = cfg_of(a), cfg_of(b), a.host(), b.host()
    torch.cuda.synchronize()
    oa.step_async(lr=1e-3), ob.step_async(lr=1e-3), empty.step_async(lr=1e-3), none.step_async(lr=1e-3)
    be.synchronize()
    a.check(ha, ca), b.check(hb, cb)
    assert int(empty.step[0]) == 1 and int(none.step[0]) == 1


def test_offsets_beyond_32_bits(be):
    """A tensor of 2^32 + 300 values in 8-bit states: the ends and the places where byte offsets pass 2^31, 2^32 and 2^34."""
    torch.cuda.empty_cache()
    n = 2 ** 32 + 300
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=BF16)
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8).view(F8) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 256), device="cuda") for _ in range(2))
    spots = [0, 2 ** 29, 2 ** 30, 2 ** 31, 2 ** 32 - 256, 2 ** 32]
    for k in spots:
        g[k:k + 256] = torch.randn(256, device="cuda").to(BF16)
    step, norm = torch.zeros(1, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda")
    opt = be.adamw([p], [g], m=[m], v=[v], m_scale=[ms], v_scale=[vs], step=step, seed=5, weight_decay=0.0)
    torch.cuda.synchronize()
    opt.grad_norm_async(norm)
    opt.step_async(lr=1e-2)
    be.synchronize()
    want = sum(float(g[k:k + 256].double().square().sum()) for k in spots) ** 0.5
    assert abs(float(norm) - want) <= 2 * U * want
    for k in spots:
        x = g[k:k + 256].double().cpu().numpy()
        lo, hi = random_bits(5, 0, k // 256, 256)
        for t, s, y, bits, floor in ((m, ms, (1 - 0.9) * x, lo, False), (v, vs, (1 - 0.999) * x * x, hi, True)):
            q, scale = to_codes(y, bits, floor)
            assert float(s[k // 256]) == scale and np.array_equal(t[k:k + 256].float().double().cpu().numpy(), q)
        # every value steps by the rate times its sign, but for eps
        assert np.abs(p[k:k + 256].double().cpu().numpy() + 1e-2 * x / (np.abs(x) + 1e-8)).max() <= 1e-2 * 40 * U
    assert int(torch.count_nonzero(p[2 ** 30 + 256:2 ** 31])) == 0 and int(torch.count_nonzero(p[-44:])) == 0
    del p, g, m, v, ms, vs, opt
    torch.cuda.empty_cache()


# ---- refusals ---------------------------------------------------------------------------------------
def test_overlaps_are_refused(be):
    x = torch.zeros(1000, device="cuda")
    p, g = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
    z = lambda: torch.zeros(100, device="cuda")  # noqa: E731
    st = lambda: torch.zeros(1, device="cuda", dtype=torch.int32)  # noqa: E731
    bad = [
        dict(params=[p, p], grads=[g, z()], m=[z(), z()], v=[z(), z()]),
        dict(params=[p], grads=[p], m=[z()], v=[z()]),
        dict(params=[x[:100]], grads=[g], m=[x[99:199]], v=[z()]),
        dict(params=[p, z()], grads=[g, z()], m=[x[:100], x[50:150]], v=[z(), z()]),
        dict(params=[p, z()], grads=[x[:100], z()], m=[z(), z()], v=[z(), x[50:150]]),
    ]
    for kw in bad:
        with pytest.raises(AdnError) as ei:
            be.adamw(step=st(), **kw)
        assert ei.value.code == ADN_E_INVALID and "overlap" in str(ei.value)
    # the same gradient twice is read twice, neighbours touch
    be.adamw([x[:100], x[100:200]], [g, g], m=[x[200:300], x[300:400]], v=[x[400:500], x[500:600]], step=st())


@pytest.mark.parametrize("kw", [dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(0.9, float("nan"))), dict(eps=0.0), dict(eps=1e-31),
                                dict(eps=float("nan")), dict(weight_decay=float("inf")), dict(lr_scale=[float("nan")]), dict(state_bits=16),
                                dict(seed=-1), dict(lr_scale=[1.0, 2.0])])
def test_refused_lists(be, kw):
    with pytest.raises(AdnError) as ei:
        be.adamw([torch.zeros(9, device="cuda")], [torch.zeros(9, device="cuda")], **kw)
    assert ei.value.code == ADN_E_INVALID


def test_refused_steps(be):
    opt, alone = be.adamw([torch.zeros(9, device="cuda")], [torch.zeros(9, device="cuda")]), be.adamw(None, [torch.zeros(9, device="cuda")])
    norm = torch.zeros(1, device="cuda")
    for kw in (dict(), dict(lr="fast"), dict(lr=float("nan")), dict(lr=1.0, max_norm=1.0), dict(lr=1.0, max_norm=-1.0, grad_norm=norm), dict(lr=1.0, grad_scale=0.0),
               dict(lr=1.0, grad_scale=float("inf")), dict(lr=1.0, max_norm=float("nan"), grad_norm=norm), dict(lr=torch.zeros(2, device="cuda")),
               dict(lr=1.0, grad_norm=torch.zeros(1))):
        with pytest.raises(AdnError) as ei:
            opt.step_async(**kw)
        assert ei.value.code == ADN_E_INVALID
    with pytest.raises(AdnError):
        alone.step_async(lr=1.0)
    with pytest.raises(AdnError):
        opt.grad_norm_async(torch.zeros(2, device="cuda"))
    opt.step_async(lr=np.float32(1e-3))  # any number
    be.synchronize()
    opt.close()
    for f in (lambda: opt.step_async(lr=1.0), lambda: opt.grad_norm_async(norm)):
        with pytest.raises(AdnError):
            f()


@pytest.mark.parametrize("bits", [32, 8, 0])
@pytest.mark.parametrize("what", ["null grad", "null param", "null m", "odd grad", "odd param", "odd copy", "grad_dtype", "reserved", "negative n", "scale", "step",
                                  "config", "bits", "count", "list"])
def test_refused_by_the_library(be, bits, what):
    import ctypes as C
    t = {k: torch.zeros(600, device="cuda") for k in ("p", "g", "m", "v", "ms", "vs", "c")}
    step = torch.zeros(1, device="cuda", dtype=torch.int32)
    a = {k: v.data_ptr() for k, v in t.items()}
    r = (_lib.AdnAdamwTensor * 1)()
    r[0] = ((None, a["g"], None, None, None, None, None, 512, 1.0, 0.0, 0, 0) if bits == 0 else
            (a["p"], a["g"], a["c"], a["m"], a["v"], a["ms"] if bits == 8 else None, a["vs"] if bits == 8 else None, 512, 1.0, 0.0, 0, 0))
    cfg = _lib.AdnAdamwConfig(0.9, 0.999, 1e-8, 0, step.data_ptr() if bits else None, bits, 0)
    n, recs, opt = 1, r, C.c_void_p()
    L = _lib.lib()
    assert L.adn_adamw_create(be._ctx, C.byref(cfg), n, recs, C.byref(opt)) == 0
    L.adn_adamw_destroy(opt)
    if what == "null grad":
        r[0].grad = None
    elif what == "null param":  # or one that does not belong there
        r[0].param = None if bits else a["p"]
    elif what == "null m":
        r[0].m = None if bits else a["m"]
    elif what == "odd grad":
        r[0].grad = a["g"] + 2
    elif what == "odd param":
        r[0].param = a["p"] + 1
    elif what == "odd copy":
        r[0].copy = a["c"] + 1
    elif what == "grad_dtype":
        r[0].grad_dtype = 2
    elif what == "reserved":
        r[0].reserved = 1
    elif what == "negative n":
        r[0].n = -1
    elif what == "scale":
        r[0].m_scale = None if bits == 8 else a["ms"]
    elif what == "step":
        cfg.step = step.data_ptr() + 1 if bits else None
        cfg.state_bits = bits or 32
    elif what == "config":
        cfg.reserved = 1
    elif what == "bits":
        cfg.state_bits = 16
    elif what == "count":
        n = -1
    elif what == "list":
        recs = None
    opt = C.c_void_p(5)
    assert L.adn_adamw_create(be._ctx, C.byref(cfg), n, recs, C.byref(opt)) == ADN_E_INVALID
    assert L.adn_last_error().decode() and not opt.value


def test_a_context_that_goes_first():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    opt = b.adamw([torch.zeros(9, device="cuda")], [torch.zeros(9, device="cuda")])
    b.close()
    with pytest.raises(AdnError) as ei:
        opt.step_async(lr=1.0)
    assert ei.value.code == ADN_E_INVALID
    opt.close()


def test_not_created_under_capture(be):
    s = torch.cuda.Stream()
    p, g, m, v = (torch.zeros(9, device="cuda") for _ in range(4))
    step = torch.zeros(1, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    be.set_stream(s.cuda_stream)
    try:
        graph, refused = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(graph, stream=s):
            try:
                be.adamw([p], [g], m=[m], v=[v], step=step)
            except AdnError as e:
                refused.append(e.code)
        assert refused == [-5]
    finally:
        torch.cuda.synchronize()
        be.set_stream(None)
