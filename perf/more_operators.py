"""The operators that take a training step from its gradients to new weights, and the norms around a residual block, through
the framework's public entry points and in plain torch: the AdamW step over many tensors with states in 32 or in 8 bits
(``aideen_amd.backend.GpuDeqBackend.adamw``, ``AdamW.step_async``), the norm of all gradients that a clipped step goes by
(``AdamW.grad_norm_async``), and the norm after a block with its gate and residual scale and the next block's norm
(``residual_norm_async``, ``residual_norm_backward_async``).

Parameters are the repository's own models (every weight of the d = 512, 8-slot, 50257-entry model, of a character model with 65
symbols, the two tables of the wide d = 2048 model) and generic lists of ragged tensors.  A list lives in one arena, as
programs that keep flat parameters have it, each tensor a view of it.  States are those of a run some steps old.
Rows are the throughput batch (32 x 256 tokens), long documents, decoding batches and generic ragged ones.
"""
import math

import torch

own = False  # run(): the framework's kernels (True) or plain torch operations

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 256  # values of an 8-bit state that share a scale
BETA1, BETA2, EPS, LR, DECAY, MAX_NORM = 0.9, 0.999, 1e-8, 2e-3, 0.1, 1.0
NORM_EPS = 1e-6  # the block's norm
MASK32 = 0xFFFFFFFF

# fields that a case may leave out
DEFAULTS = dict(bits=32, grad="f32", copy=False, clip=False, type="f32", gate="none", sigmoid=False, post=True, pre=True, back=False,
                keep=1.0, scale=1.0, dz=True)


def _c(name, **kw):
    return dict(name=name, **kw)


def listed():
    return [
        # Online updates of a character model: 21 tensors, 1.9 M parameters, clipped; launches and latency count.
        _c("adamw_char", op="adamw", model="char", clip=True),
        # A training step of the whole 512-wide model in fp32: 65 M parameters.
        _c("adamw_512", op="adamw", model="512"),
        # The wide model's tables (206 M parameters): bf16 gradients, fp32 weights with the bf16 copies that the products read.
        _c("adamw_tables_bf16", op="adamw", model="tables", grad="bf16", copy=True),
        # Hundreds of small ragged tensors (adapters, biases, norms) with states in 8 bits.
        _c("adamw8_ragged", op="adamw", model="ragged", bits=8, tensors=701, total=3100003),
        # The 512-wide model with states in 8 bits, clipped by the norm of all its gradients.
        _c("adamw8_512", op="adamw", model="512", bits=8, clip=True),
        # The wide tables in 8 bits: what a large vocabulary takes of memory is what such states are for.
        _c("adamw8_tables_bf16", op="adamw", model="tables", bits=8, grad="bf16", copy=True),
        # The norm alone, as a program that logs it or adds it up over ranks calls it: the character model, and the wide tables.
        _c("grad_norm_char", op="norm", model="char"),
        _c("grad_norm_tables_bf16", op="norm", model="tables", grad="bf16"),
        # A block's end in a decoding batch of 24 rows: a learned scale a channel, then the next norm.
        _c("residual_24", op="residual", rows=24, d=512, gate="channel"),
        # The solver's damped update (0.3 h + 0.7 norm(f)) with the head's norm behind it, at the throughput batch.
        _c("residual_8192", op="residual", rows=8192, d=512, keep=0.3, scale=0.7),
        # The backward pass of a block whose channels have learned scales, at the throughput batch.
        _c("residual_back_8192", op="residual", rows=8192, d=512, gate="channel", back=True),
        # The same for long documents (4 x 8192 tokens, less a few), wide bf16 rows and a gate computed from the input.
        _c("residual_back_32749", op="residual", rows=32749, d=2048, type="bf16", gate="element", sigmoid=True, back=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "norm", "residual", "residual"])
    if op != "residual":
        total = _log_int(rng, 2000, 60000000)
        c = dict(op=op, model="ragged", total=total, tensors=_log_int(rng, 1, min(2000, total // 16)), grad=rng.choice(["f32", "bf16"]))
        if op == "adamw":
            c.update(bits=rng.choice([32, 8]), copy=rng.random() < 0.4, clip=rng.random() < 0.5)
        return c
    rows = _log_int(rng, 1, 32768)
    d = rng.choice([64, 128, 192, 256, 320, 512, 512, 768, 1024, 2048, _log_int(rng, 33, 2048), _log_int(rng, 33, 2048)])
    gate = rng.choice(["none", "channel", "row", "element"])
    return dict(op=op, rows=rows, d=d, type=rng.choice(["f32", "bf16"]), gate=gate, sigmoid=gate != "none" and rng.random() < 0.5,
                post=rng.random() < 0.8, pre=rng.random() < 0.8, back=rng.random() < 0.6, keep=rng.choice([1.0, 1.0, 0.3]),
                scale=rng.choice([1.0, 0.7, 0.1]), dz=True)


def _full(case):
    return {**DEFAULTS, **case}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _sizes(c):
    """The tensors of a list: how many values each has."""
    if c["model"] == "tables":
        return [50257 * 2048] * 2
    if c["model"] == "ragged":
        g = torch.Generator().manual_seed(c["total"] * 31 + c["tensors"])
        share = torch.exp(1.5 * torch.randn(c["tensors"], generator=g, dtype=torch.float64))
        return [1 + int(v) for v in torch.floor(share / share.sum() * (c["total"] - c["tensors"]))]
    d, H, V, r, N = (512, 8, 50257, 32, 16) if c["model"] == "512" else (192, 8, 65, 32, 16)
    return ([H * d * d] * 6 + [V * d] * 2 + [H * d] * 3 + [d] * 2 + [V] + [H * d] * 3 + [H * d * r] * 2 + [H * N * d] * 2)


def _pad(c):
    """Tensors begin at multiples of this in the arena; what is between them is zero throughout."""
    return BLOCK if c["bits"] == 8 else 64


def _pow2(e):
    """Powers of two in 64 bits: as 32-bit ones, which a power function's last bits do not reach."""
    return torch.exp2(e.double()).float().double()


def prepare(case, seed):
    c = _full(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    s = dict(c=c, seed=int(seed) * 7919 + 5)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def uniform(shape, lo, hi):
        return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo

    if c["op"] == "residual":
        rows, d, ty = c["rows"], c["d"], TYPES[c["type"]]
        s["f"] = (normal(rows, d) * uniform((rows, 1), 0.2, 3.0)).to(ty)
        s["post_gain"] = uniform((d,), 0.75, 1.25) if c["post"] else None
        s["pre_gain"] = uniform((d,), 0.75, 1.25) if c["pre"] else None
        shape = {"none": None, "channel": (d,), "row": (rows, 1), "element": (rows, d)}[c["gate"]]
        gate = None if shape is None else normal(*shape) if c["sigmoid"] else uniform(shape, 0.05, 1.0)
        s["gate"] = gate.to(ty) if c["gate"] == "element" else gate
        if c["back"]:
            s["z"] = (normal(rows, d) * uniform((rows, 1), 0.5, 2.0)).to(ty)
            s["dz"] = (normal(rows, d) / rows).to(ty)
            s["dy"] = (normal(rows, d) / rows).to(ty) if c["pre"] else None
            s["out"] = dict(dx=torch.empty((rows, d), device="cuda", dtype=ty), df=torch.empty((rows, d), device="cuda", dtype=ty))
            if gate is not None:
                s["out"]["dgate"] = torch.empty_like(s["gate"])
            for k in ("post_gain", "pre_gain"):
                if s[k] is not None:
                    s["out"]["d" + k] = torch.empty(d, device="cuda")
        else:
            s["x"] = (normal(rows, d) * uniform((rows, 1), 0.5, 2.0)).to(ty)
            s["out"] = dict(z=torch.empty((rows, d), device="cuda", dtype=ty))
            if c["pre"]:
                s["out"]["y"] = torch.empty((rows, d), device="cuda", dtype=ty)
        return s

    n, pad = _sizes(c), _pad(c)
    padded = [-(-v // pad) * pad for v in n]
    starts = [0]
    for v in padded:
        starts.append(starts[-1] + v)
    total = starts[-1]
    there = torch.zeros(total, device="cuda", dtype=torch.bool)
    for a, v in zip(starts, n):
        there[a:a + v] = True

    def arena(v, dtype=torch.float32):
        return torch.where(there, v, 0.0).to(dtype)

    def views(t):
        return [t[a:a + v] for a, v in zip(starts, n)]
    # gradients of rows of different sizes, as rare and frequent entries have them
    size = torch.repeat_interleave(torch.pow(10.0, uniform((-(-total // 64),), -5.0, -2.0)), 64, output_size=-(-total // 64) * 64)[:total]
    s["g"] = arena(normal(total) * size, TYPES[c["grad"]])
    s.update(grads=views(s["g"]), norm=torch.zeros(1, device="cuda"))
    if c["op"] == "norm":
        return s
    s["p"] = arena(normal(total) * 0.04)
    m, v = arena(normal(total) * size * 0.4), arena(uniform((total,), 0.3, 2.0) * size * size)
    s["step"] = torch.full((1,), 37 + int(seed) % 100, device="cuda", dtype=torch.int32)
    s["decay"] = [DECAY if k > 60000 or c["model"] == "ragged" and k % 2 else 0.0 for k in n]
    s["decays"], s["padded"] = torch.tensor(s["decay"], device="cuda"), torch.tensor(padded, device="cuda")
    if c["bits"] == 8:
        for k, t in (("m", m), ("v", v)):
            top = t.view(-1, BLOCK).abs().amax(1).double()
            scale = _pow2(torch.frexp(torch.clamp(top, min=2.0 ** -110)).exponent - 8)
            code = (t.view(-1, BLOCK).double() / scale[:, None]).float().to(torch.float8_e4m3fn)
            if k == "v":  # no value that is there has a code of zero
                code = torch.where((t.view(-1, BLOCK) > 0) & (code.float() == 0), 2.0 ** -9, code.float()).to(torch.float8_e4m3fn)
            s[k], s[k + "_scale"] = code.view(-1), scale.float()
        blocks = [a // BLOCK for a in starts]
        s["scales"] = {k: [s[k][a:b] for a, b in zip(blocks, blocks[1:])] for k in ("m_scale", "v_scale")}
    else:
        s["m"], s["v"] = m, v
    s["copy"] = s["p"].to(torch.bfloat16) if c["copy"] else None
    s["views"] = {k: views(s[k]) for k in ("p", "m", "v", "copy") if s[k] is not None}
    return s


# ---------------------------------------------------------------------------------------------
# plain torch operations in 32 bits (64 for the norm and for states that are rounded to 8 bits), rounded once at the end
# ---------------------------------------------------------------------------------------------
def _plain_norm(s):
    return torch.sqrt(s["g"].double().square().sum()).float().view(1)


def _mix64(x):
    """SplitMix64's finaliser on int64 tensors."""
    x = (x ^ ((x >> 30) & 0x3FFFFFFFF)) * -0x40A7B892E31B1A47
    x = (x ^ ((x >> 27) & 0x1FFFFFFFFF)) * -0x6B2FB644ECCEEE15
    return x ^ ((x >> 31) & 0x1FFFFFFFF)


def _random16(s, blocks):
    """Two arrays of 16 random bits a value, by seed, step, block and place in the block."""
    key = _mix64(s["seed"] + s["step"].long() * -0x61C8864680B583EB)
    a = _mix64(key + (torch.arange(blocks, device="cuda") + 1) * -0x61C8864680B583EB) & MASK32
    r = (a[:, None] + torch.arange(BLOCK, device="cuda") * 0x9E3779B9) & MASK32
    r = ((r ^ (r >> 16)) * 0x7FEB352D) & MASK32
    r = ((r ^ (r >> 15)) * 0x846CA68B) & MASK32
    r = r ^ (r >> 16)
    return r & 0xFFFF, r >> 16


def _plain_codes(x, random, floor):
    """(codes' values, scales) of blocks of 64-bit values: e4m3 with 3 bits behind the point from 2^-6 up, rounded down after
    a random share of a step has been added; floor: what is not zero keeps the smallest code."""
    top = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -110)
    scale = _pow2(torch.frexp(top).exponent - 8)
    a = x.abs() / scale
    step = _pow2(torch.frexp(a).exponent.clamp(min=-5) - 4)
    q = torch.floor(a / step + random.double() / 65536) * step
    if floor:
        q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
    return torch.where(x < 0, -q, q).to(torch.float8_e4m3fn), scale[:, 0].float()


def _plain_adamw(s):
    c, out = s["c"], {}
    coef = torch.ones((), device="cuda", dtype=torch.float64)
    if c["clip"]:
        out["norm"] = s["norm"].copy_(_plain_norm(s))
        coef = torch.clamp(MAX_NORM / (s["norm"][0].double() + 1e-6), max=1.0)
    t = (s["step"][0] + 1).double()
    bc1, bc2 = 1 - BETA1 ** t, 1 - BETA2 ** t
    if c["bits"] == 8:
        g = s["g"].double().view(-1, BLOCK) * coef
        m = BETA1 * (s["m"].double().view(-1, BLOCK) * s["m_scale"].double()[:, None]) + (1 - BETA1) * g
        v = BETA2 * (s["v"].double().view(-1, BLOCK) * s["v_scale"].double()[:, None]) + (1 - BETA2) * g * g
        lo, hi = _random16(s, m.shape[0])
        m8, ms = _plain_codes(m, lo, False)
        v8, vs = _plain_codes(v, hi, True)
        s["m"].copy_(m8.view(-1)), s["v"].copy_(v8.view(-1))
        out.update(m_scale=s["m_scale"].copy_(ms), v_scale=s["v_scale"].copy_(vs))
        m, v = m.float().view(-1), v.float().view(-1)
    else:
        g = s["g"].float() * coef.float()
        m = s["m"].mul_(BETA1).add_((1 - BETA1) * g)
        v = s["v"].mul_(BETA2).add_((1 - BETA2) * g * g)
    step = m / bc1.float() / (torch.sqrt(v / bc2.float()) + EPS)
    decay = torch.repeat_interleave(s["decays"], s["padded"], output_size=s["p"].numel())
    s["p"].sub_(LR * (step + decay * s["p"]))
    s["step"].add_(1)
    if c["copy"]:
        out["copy"] = s["copy"].copy_(s["p"])
    out.update(p=s["p"], m=s["m"], v=s["v"], step=s["step"])
    return out


def _plain_gate(s):
    g = 1.0 if s["gate"] is None else s["gate"].float()
    return torch.sigmoid(g) if s["c"]["sigmoid"] else g


def _plain_residual(s):
    c, ty = s["c"], TYPES[s["c"]["type"]]
    f, gate = s["f"].float(), _plain_gate(s)
    rf = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + NORM_EPS) if c["post"] else 1.0
    gp = s["post_gain"] if c["post"] else 1.0
    n = f * rf * gp
    if not c["back"]:
        z = c["keep"] * s["x"].float() + c["scale"] * gate * n
        out = dict(z=z.to(ty))
        if c["pre"]:
            out["y"] = (z * (1.0 / torch.sqrt((z * z).mean(1, keepdim=True) + NORM_EPS)) * s["pre_gain"]).to(ty)
        return out
    z, up, out = s["z"].float(), s["dz"].float(), {}
    if c["pre"]:
        dy = s["dy"].float()
        rz = 1.0 / torch.sqrt((z * z).mean(1, keepdim=True) + NORM_EPS)
        a = dy * s["pre_gain"]
        up = up + rz * (a - z * (rz * rz) * (a * z).mean(1, keepdim=True))
        out["dpre_gain"] = (dy * z * rz).sum(0)
    out["dx"] = (c["keep"] * up).to(ty)
    dn = c["scale"] * up * gate
    if s["gate"] is not None:
        dgate = c["scale"] * up * n
        if c["sigmoid"]:
            dgate = dgate * gate * (1.0 - gate)
        out["dgate"] = dgate.sum(0) if c["gate"] == "channel" else dgate.sum(1, keepdim=True) if c["gate"] == "row" else dgate.to(ty)
    if c["post"]:
        out["dpost_gain"] = (dn * f * rf).sum(0)
        b = dn * gp
        dn = rf * (b - f * (rf * rf) * (b * f).mean(1, keepdim=True))
    out["df"] = dn.to(ty)
    return out


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
_KEPT = []


def _backend():
    """The one context that a program keeps.  A context has a stream of its own unless it is handed another, and torch's
    default stream cannot be handed over: torch's work moves to a stream that both use, behind what the default one holds,
    so that every tensor is made, used and read in one order."""
    if not _KEPT:
        from aideen_amd import synth
        from aideen_amd.backend import GpuDeqBackend
        be, stream = GpuDeqBackend(synth.ModelConfig(d=512, H=8, V=50257, flags=0), 1, 1), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        be.set_stream(stream.cuda_stream)
        _KEPT.append(be)
    return _KEPT[0]


def _optimizer(s):
    """The optimizer that a program keeps beside its parameters, made at the first step."""
    if "optimizer" not in s:
        c, be = s["c"], _backend()
        if c["op"] == "norm":
            s["optimizer"] = be.adamw(None, s["grads"])
        else:
            v = s["views"]
            s["optimizer"] = be.adamw(v["p"], s["grads"], m=v["m"], v=v["v"], step=s["step"], copies=v.get("copy"), betas=(BETA1, BETA2),
                                      eps=EPS, weight_decay=s["decay"], seed=s["seed"], **s.get("scales", {}))
    return s["optimizer"]


def _own_adamw(s):
    c, opt, out = s["c"], _optimizer(s), {}
    if c["op"] == "norm":
        opt.grad_norm_async(s["norm"])
        return s["norm"]
    if c["clip"]:
        opt.grad_norm_async(s["norm"])
        opt.step_async(lr=LR, grad_norm=s["norm"], max_norm=MAX_NORM)
        out["norm"] = s["norm"]
    else:
        opt.step_async(lr=LR)
    for k in ("p", "m", "v", "step", "m_scale", "v_scale", "copy"):
        if s.get(k) is not None:
            out[k] = s[k]
    return out


def _own_residual(s):
    c, be = s["c"], _backend()
    kw = dict(gate=s["gate"], gate_sigmoid=c["sigmoid"], post_norm=c["post"], post_gain=s["post_gain"], pre_gain=s["pre_gain"],
              keep=c["keep"], scale=c["scale"], eps=NORM_EPS, outputs=s["out"])
    if c["back"]:
        be.residual_norm_backward_async(s["z"], s["f"], dz=s["dz"], dy=s["dy"], **kw)
    else:
        be.residual_norm_async(s["x"], s["f"], **kw)
    return s["out"]


def run(s):
    op = s["c"]["op"]
    if own:
        return _own_residual(s) if op == "residual" else _own_adamw(s)
    return _plain_residual(s) if op == "residual" else _plain_norm(s) if op == "norm" else _plain_adamw(s)


def work(case):
    """Inputs read once, outputs written once."""
    c = _full(case)
    if c["op"] == "residual":
        n, e, full = c["rows"] * c["d"], 4 if c["type"] == "f32" else 2, c["gate"] == "element"
        if not c["back"]:
            return {"bytes": e * n * (3 + c["pre"] + full), "flops": n * (4 + 3 * c["post"] + 4 * c["pre"])}
        return {"bytes": e * n * (5 + 2 * c["pre"] - (not c["post"] and c["gate"] == "none" and not c["pre"]) + 2 * full),
                "flops": n * (6 + 8 * c["post"] + 10 * c["pre"])}
    n, grad = sum(_sizes(c)), 4 if c["grad"] == "f32" else 2
    if c["op"] == "norm":
        return {"bytes": grad * n, "flops": 2 * n}
    state = 4 if c["bits"] == 8 else 16
    return {"bytes": n * (8 + grad + state + 2 * c["copy"]) + (16 * n // BLOCK if c["bits"] == 8 else 0), "flops": n * 16}


# ---------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_residual(s):
    """Forward: the definition.  Backward: that of <dz, z> + <dy, y> by automatic differentiation, from the given z."""
    c = s["c"]
    leaf = lambda k: None if s.get(k) is None else s[k].detach().double().requires_grad_(c["back"])  # noqa: E731
    f, gate, gp, gq = leaf("f"), leaf("gate"), leaf("post_gain"), leaf("pre_gain")

    def normed(t, gain):
        return t / (t.pow(2).sum(1, keepdim=True) / c["d"] + NORM_EPS).sqrt() * gain
    branch = (normed(f, gp) if c["post"] else f) * c["scale"]
    if gate is not None:
        branch = branch * (1 / (1 + torch.exp(-gate)) if c["sigmoid"] else gate)
    if not c["back"]:
        z = s["x"].double() * c["keep"] + branch
        return dict(z=z, y=normed(z, gq)) if c["pre"] else dict(z=z)
    z = leaf("z")
    up, out = s["dz"].double(), {}
    if c["pre"]:
        more, out["dpre_gain"] = torch.autograd.grad((normed(z, gq) * s["dy"].double()).sum(), [z, gq])
        up = up + more
    out["dx"] = up * c["keep"]
    wanted = dict(df=f, dgate=gate, dpost_gain=gp if c["post"] else None)
    wanted = {k: v for k, v in wanted.items() if v is not None}
    out.update(zip(wanted, torch.autograd.grad((branch * up).sum(), list(wanted.values()))))
    return out


def _exponent(x):
    """floor(log2 x) of normal numbers, from the bits."""
    return (x.view(torch.int64) >> 52) - 1023


def _power(e):
    return ((e + 1023) << 52).view(torch.float64)


def _exact_adamw(s):
    c, g, out = s["c"], s["g"].double(), {}
    if c["clip"] or c["op"] == "norm":
        out["norm"] = torch.linalg.vector_norm(g).view(1)
        if c["op"] == "norm":
            return out["norm"]
        # the step reads the norm as it is handed over, in 32 bits
        length = float(out["norm"].float())
        g = g * min(1.0, MAX_NORM / (length + 1e-6))
    t = int(s["step"][0]) + 1
    eight, old = c["bits"] == 8, {}
    for k in ("m", "v"):
        old[k] = s[k].double()
        if eight:
            old[k] = old[k] * torch.repeat_interleave(s[k + "_scale"].double(), BLOCK)
    m = old["m"] * BETA1 + (1 - BETA1) * g
    v = old["v"] * BETA2 + (1 - BETA2) * g * g
    away = m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    if eight:
        bits = _exact_random(s["seed"], t - 1, m.numel())
    for k, x in (("m", m), ("v", v)):
        if not eight:
            out[k] = x
            continue
        # the two neighbours on the grid of codes, the upper one with the probability of the distance from the lower
        blocks = x.view(-1, BLOCK)
        exponent = _exponent(blocks.abs().amax(1).clamp(min=2.0 ** -110))
        out[k + "_scale"] = _power(exponent - 7)
        a = (blocks.abs() / out[k + "_scale"][:, None]).view(-1)
        grid = _power(_exponent(a.clamp(min=2.0 ** -6)) - 3)
        lower = torch.floor(a / grid)
        up = (a / grid - lower) * 65536 + (bits[k].double()) >= 65536
        code = (lower + up) * grid
        if k == "v":
            code = torch.where((code == 0) & (x > 0), 2.0 ** -9, code)
        out[k] = code * torch.sign(x)
    pieces = [torch.full((int(n),), w, device="cuda", dtype=torch.float64) for n, w in zip(s["padded"], s["decay"])]
    p = s["p"].double()
    out.update(p=p - LR * (away + torch.cat(pieces) * p), step=s["step"] + 1)
    if c["copy"]:
        out["copy"] = out["p"]
    return out


def _exact_random(seed, step, n):
    """The bits by Python's integers as far as they are shared by a block, then 32 bits at a time."""
    gold, whole = 0x9E3779B97F4A7C15, (1 << 64) - 1

    def signed(v):
        return v - (1 << 64) if v >> 63 else v

    def finish(x):
        for shift, factor in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
            x = x ^ ((x >> shift) & ((1 << (64 - shift)) - 1))
            x = x * signed(factor) if isinstance(x, torch.Tensor) else x * factor & whole
        return x ^ ((x >> 31) & ((1 << 33) - 1))
    key = finish((seed + step * gold) & whole)
    i = torch.arange(n, device="cuda")
    block = finish(signed(key) + (i // BLOCK + 1) * signed(gold))
    r = (block + (i % BLOCK) * 0x9E3779B9) % (1 << 32)
    r = (r ^ (r // (1 << 16))) * 0x7FEB352D % (1 << 32)
    r = (r ^ (r // (1 << 15))) * 0x846CA68B % (1 << 32)
    r = r ^ (r // (1 << 16))
    return dict(m=r % 65536, v=r // 65536)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_residual(s) if s["c"]["op"] == "residual" else _exact_adamw(s)
