"""The training operators of the language-model head that are measured, through the framework's public entry points
(``aideen_amd.backend.GpuDeqBackend``) and in plain torch: softmax cross entropy over the vocabulary with its gradients
(``lm_loss_async``), the head's RMS norm forward and backward (``rms_norm_async``, ``rms_norm_backward_async``), the scaled
embedding lookup and its gradient (``embed_lookup_async``, ``embed_grad_async``).

Sizes are the repository's presets (d = 512 with a vocabulary of 50257, the wide rows of d = 2048, 8192 tokens a batch), the
reference's evaluation shape (d = 192, 65 symbols, 128 positions) and generic ragged ones.  Head rows are normalised rows
times a gain, weights are drawn at twice the Xavier-uniform range, so logits spread as a trained head's do; token ids and
targets are Zipf-distributed ranks.  Padded batches mark rows without a token or target by -1.
"""
import math

import torch

own = False  # run(): the framework's kernels (True) or plain torch operations

EPS = 1e-5  # the LM head's norm
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# fields that a case may leave out: pad is the share of rows without a token or target
DEFAULTS = dict(type="f32", vocab=50257, bias=False, pad=0.0, grads=True)


def _c(name, **kw):
    return dict(name=name, **kw)


def listed():
    return [
        # An online update from a single token: one row of the head, every gradient.  The weights' bytes count.
        _c("loss_token", op="loss", rows=1, d=512, bias=True),
        # Evaluation of a character model, the reference's benchmark shape: launches and latency.
        _c("loss_char_128", op="loss", rows=128, d=192, vocab=65, bias=True),
        # Perplexity of one 256-token window: losses alone.
        _c("loss_eval_256", op="loss", rows=256, d=512, grads=False),
        # A training step on a small padded batch of ragged documents with wide rows, bf16 tensors.
        _c("loss_wide_531", op="loss", rows=531, d=1024, type="bf16", bias=True, pad=0.2),
        # The throughput batch (32 x 256 tokens) in fp32, the framework's own type.
        _c("loss_8192", op="loss", rows=8192, d=512),
        # The wide preset's head (d = 2048) in bf16: the largest product.
        _c("loss_deep_4096", op="loss", rows=4096, d=2048, type="bf16"),
        # The head's norm of a decoding batch of 24 rows.
        _c("norm_24", op="norm", rows=24, d=512, back=False),
        # The norm's backward pass of the throughput batch, with the gain's gradient.
        _c("norm_back_8192", op="norm", rows=8192, d=512, back=True),
        # The same for long documents (4 x 8192 tokens, less a few) with wide bf16 rows.
        _c("norm_back_32749", op="norm", rows=32749, d=2048, type="bf16", back=True),
        # Embedding rows of the throughput batch, scaled by sqrt(d) as heads with shared tables do.
        _c("embed_8192", op="embed", rows=8192, d=512, back=False, scaled=True),
        # The table's gradient from one 256-token window: the table's rows without a token are written too.
        _c("embed_back_256", op="embed", rows=256, d=512, back=True),
        # The table's gradient from long documents: the most frequent tokens have thousands of rows each.
        _c("embed_back_32768", op="embed", rows=32768, d=512, back=True, scaled=True, pad=0.05),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["loss", "loss", "norm", "embed"])
    d = rng.choice([64, 128, 192, 256, 320, 512, 512, 768, 1024, 2048])
    c = dict(op=op, d=d, type=rng.choice(["f32", "bf16"]))
    vocab = rng.choice([65, 512, 50257, _log_int(rng, 50, 60000), _log_int(rng, 50, 60000)])
    if op == "loss":
        # no dearer than the largest fp32 and bf16 cases
        most = (8192 * 512 if c["type"] == "f32" else 4096 * 2048) * 50257 // (d * vocab)
        c.update(rows=_log_int(rng, 1, min(16384, max(1, most))), vocab=vocab, bias=rng.random() < 0.5,
                 pad=rng.choice([0.0, 0.0, 0.1, 0.5]), grads=rng.random() < 0.75)
    elif op == "norm":
        c.update(rows=_log_int(rng, 1, 32768), back=rng.random() < 0.6)
        c["d"] = rng.choice([d, d, _log_int(rng, 33, 2048)])
    else:
        c.update(rows=_log_int(rng, 1, 32768), vocab=vocab, back=rng.random() < 0.6, scaled=rng.random() < 0.5,
                 pad=rng.choice([0.0, 0.0, 0.1]))
    return c


def _full(case):
    return {**DEFAULTS, **case}


def _scale(c):
    return math.sqrt(c["d"]) if c.get("scaled") else 1.0


def _tokens(c, g):
    """Zipf-distributed ranks; -1 where a padded batch has none."""
    p = 1.0 / torch.arange(1, c["vocab"] + 1, device="cuda", dtype=torch.float64) ** 1.1
    cdf = torch.cumsum(p / p.sum(), 0)
    u = torch.rand(c["rows"], device="cuda", generator=g, dtype=torch.float64)
    t = torch.searchsorted(cdf, u).clamp_(max=c["vocab"] - 1).to(torch.int32)
    if c["pad"]:
        gone = torch.rand(c["rows"], device="cuda", generator=g) < c["pad"]
        gone[0] = False
        t[gone] = -1
    return t


def prepare(case, seed):
    c = _full(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    n, d, ty = c["rows"], c["d"], TYPES[c["type"]]
    s = dict(c=c)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def uniform(shape, lo, hi):
        return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo

    def buffer(*shape, dtype=ty):
        return torch.empty(shape, device="cuda", dtype=dtype)

    if c["op"] == "loss":
        V, r = c["vocab"], 2 * math.sqrt(3.0 / d)
        x = normal(n, d)
        s["x"] = (x / x.square().mean(1, keepdim=True).sqrt() * uniform((d,), 0.75, 1.25)).to(ty)
        s["w"] = uniform((V, d), -r, r).to(ty)
        s["bias"] = uniform((V,), -0.05, 0.05) if c["bias"] else None
        s["targets"] = _tokens(c, g)
        counted = s["targets"] >= 0
        s["dloss"] = counted.float() / counted.sum()  # the mean over the rows that have a target
        s["out"] = dict(loss=buffer(n, dtype=torch.float32), lse=buffer(n, dtype=torch.float32))
        if c["grads"]:
            s["out"].update(dx=buffer(n, d), dw=buffer(V, d))
            if c["bias"]:
                s["out"]["db"] = buffer(V, dtype=torch.float32)
    elif c["op"] == "norm":
        s["x"] = (normal(n, d) * uniform((n, 1), 0.2, 3.0)).to(ty)
        s["gain"] = uniform((d,), 0.75, 1.25)
        if c["back"]:
            s["dy"] = (normal(n, d) / n).to(ty)
            s["out"] = dict(dx=buffer(n, d), dg=buffer(d, dtype=torch.float32))
        else:
            s["out"] = dict(y=buffer(n, d))
    else:
        V = c["vocab"]
        s["tokens"] = _tokens(c, g)
        if c["back"]:
            s["dout"] = (normal(n, d) / n).to(ty)
            s["out"] = dict(dtable=buffer(V, d))
        else:
            s["table"] = uniform((V, d), -0.2, 0.2).to(ty)
            s["out"] = dict(out=buffer(n, d))
    return s


# ---------------------------------------------------------------------------------------------
# plain torch operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------------------------
def _plain_loss(s):
    c, ty = s["c"], TYPES[s["c"]["type"]]
    x, w = s["x"].float(), s["w"].float()
    logits = x @ w.t()
    if c["bias"]:
        logits = logits + s["bias"]
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    counted = s["targets"] >= 0
    t = s["targets"].long().clamp(min=0)
    loss = torch.where(counted, lse - logits.gather(1, t[:, None])[:, 0], 0.0)
    out = dict(loss=loss, lse=torch.where(counted, lse, 0.0))
    if c["grads"]:
        p = p / total
        p[torch.arange(c["rows"], device=p.device), t] -= 1.0
        p = p * torch.where(counted, s["dloss"], 0.0)[:, None]
        out.update(dx=(p @ w).to(ty), dw=(p.t() @ x).to(ty))
        if c["bias"]:
            out["db"] = p.sum(0)
    return out


def _plain_norm(s):
    c, ty = s["c"], TYPES[s["c"]["type"]]
    x = s["x"].float()
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    if not c["back"]:
        return dict(y=(x * r * s["gain"]).to(ty))
    dy = s["dy"].float()
    a = dy * s["gain"]
    dx = r * (a - x * (r * r) * (a * x).mean(1, keepdim=True))
    return dict(dx=dx.to(ty), dg=(dy * x * r).sum(0))


def _plain_embed(s):
    c, ty = s["c"], TYPES[s["c"]["type"]]
    there = (s["tokens"] >= 0)[:, None]
    t = s["tokens"].long().clamp(min=0)
    if not c["back"]:
        return dict(out=torch.where(there, s["table"][t].float() * _scale(c), 0.0).to(ty))
    rows = torch.where(there, s["dout"].float() * _scale(c), 0.0)
    return dict(dtable=torch.zeros((c["vocab"], c["d"]), device=rows.device).index_add_(0, t, rows).to(ty))


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


def _own(s):
    c, be, o = s["c"], _backend(), s["out"]
    if c["op"] == "loss":
        be.lm_loss_async(s["x"], s["targets"], w=s["w"], bias=s["bias"], dloss=s["dloss"], outputs=o)
    elif c["op"] == "norm" and c["back"]:
        be.rms_norm_backward_async(s["x"], s["dy"], gain=s["gain"], eps=EPS, outputs=o)
    elif c["op"] == "norm":
        be.rms_norm_async(s["x"], o["y"], gain=s["gain"], eps=EPS)
    elif c["back"]:
        be.embed_grad_async(s["dout"], s["tokens"], o["dtable"], scale=_scale(c))
    else:
        be.embed_lookup_async(s["tokens"], o["out"], table=s["table"], scale=_scale(c))
    return o


def run(s):
    if own:
        return _own(s)
    op = s["c"]["op"]
    return _plain_loss(s) if op == "loss" else _plain_norm(s) if op == "norm" else _plain_embed(s)


def work(case):
    """Inputs read once, outputs written once; the products of the logits and, with gradients, of dx and dw."""
    c = _full(case)
    n, d, V, e = c["rows"], c["d"], c["vocab"], 4 if c["type"] == "f32" else 2
    if c["op"] == "loss":
        by = e * (n + V) * d + 4 * (4 * n + (V if c["bias"] else 0))
        if not c["grads"]:
            return {"bytes": by, "flops": 2 * n * V * d + 4 * n * V}
        return {"bytes": by + e * (n + V) * d + (4 * V if c["bias"] else 0), "flops": 6 * n * V * d + 6 * n * V}
    if c["op"] == "norm":
        return {"bytes": (3 if c["back"] else 2) * e * n * d + (8 if c["back"] else 4) * d, "flops": (11 if c["back"] else 4) * n * d}
    # a lookup reads the rows of the distinct tokens, at most one a position
    there = n * (1 - c["pad"])
    return {"bytes": 4 * n + e * d * (there + V if c["back"] else min(there, V) + n), "flops": n * d}


# ---------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_loss(s):
    """loss_i = log sum_v exp(z_iv) - z_i,t(i); d loss_i / d z_iv = softmax_iv - [v = t(i)]; a block of rows at a time."""
    c = s["c"]
    n, V, d = c["rows"], c["vocab"], c["d"]
    w = s["w"].double()
    out = dict(loss=torch.zeros(n, device="cuda", dtype=torch.float64), lse=torch.zeros(n, device="cuda", dtype=torch.float64))
    if c["grads"]:
        out["dx"] = torch.zeros((n, d), device="cuda", dtype=torch.float64)
        out["dw"] = torch.zeros((V, d), device="cuda", dtype=torch.float64)
        db = torch.zeros(V, device="cuda", dtype=torch.float64)
    wt = w.t().contiguous()
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        x, t, g = s["x"][a:b].double(), s["targets"][a:b].long(), s["dloss"][a:b].double()
        z = torch.mm(x, wt)
        if c["bias"]:
            z += s["bias"].double()
        lse = torch.logsumexp(z, 1)
        picked = torch.nonzero(t >= 0)[:, 0]
        out["lse"][a + picked] = lse[picked]
        out["loss"][a + picked] = lse[picked] - z[picked, t[picked]]
        if c["grads"]:
            dz = torch.exp(z - lse[:, None])
            dz[picked, t[picked]] -= 1.0
            dz *= torch.where(t >= 0, g, torch.zeros_like(g))[:, None]
            out["dx"][a:b] = torch.mm(dz, w)
            out["dw"] += torch.mm(dz.t().contiguous(), x)
            db += dz.sum(0)
    if c["grads"] and c["bias"]:
        out["db"] = db
    return out


def _exact_norm(s):
    """y_i = g_i x_i / R, R = sqrt(sum x^2 / d + eps): dR/dx_j = x_j / (d R)."""
    c = s["c"]
    x, g = s["x"].double(), s["gain"].double()
    R = (x.pow(2).sum(1) / c["d"] + EPS).sqrt()[:, None]
    if not c["back"]:
        return dict(y=g * x / R)
    dy = s["dy"].double()
    dR = -(dy * g * x).sum(1, keepdim=True) / R ** 2
    return dict(dx=dy * g / R + dR * x / (c["d"] * R), dg=(dy * (x / R)).sum(0))


def _exact_embed(s):
    """The lookup is the product of the tokens' indicator matrix with the table; its gradient the transposed product."""
    c = s["c"]
    keep = torch.nonzero(s["tokens"] >= 0)[:, 0]
    t = s["tokens"][keep].long()
    if not c["back"]:
        out = torch.zeros((c["rows"], c["d"]), device="cuda", dtype=torch.float64)
        out[keep] = s["table"].double()[t] * _scale(c)
        return dict(out=out)
    order = torch.argsort(t, stable=True)
    sums = torch.cumsum(s["dout"].double()[keep][order], 0)  # prefix sums of the rows in token order
    sums = torch.cat([torch.zeros((1, c["d"]), device="cuda", dtype=torch.float64), sums])
    ends = torch.searchsorted(t[order], torch.arange(c["vocab"] + 1, device="cuda"))
    return dict(dtable=(sums[ends[1:]] - sums[ends[:-1]]) * _scale(c))


def exact(case, seed):
    s = prepare(case, seed)
    op = s["c"]["op"]
    return _exact_loss(s) if op == "loss" else _exact_norm(s) if op == "norm" else _exact_embed(s)
