"""AdamW over a list of tensors, and the norm of the list's gradients, over the C ABI (``adn_adamw_*``).

The reference's trainers step their weights by AdamW (``gpu_lm_head.rs``, ``gpu_embedding.rs:496-670``);
here one launch serves the whole list, with moments in fp32 or in 8 bits.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import check, lib

_TORCH = {}
_NO_NUMBER = (TypeError, ValueError, RuntimeError, OverflowError)  # what float() and the structures' fields raise


def _torch():
    """torch, and the types that are met here, looked up once."""
    if not _TORCH:
        import torch
        _TORCH.update(torch=torch, tensor=torch.Tensor, f32=torch.float32, bf16=torch.bfloat16, i32=torch.int32, codes=(torch.float8_e4m3fn, torch.uint8))
    return _TORCH


def _invalid(msg: str) -> "_lib.AdnError":
    return _lib.AdnError(_lib.ADN_E_INVALID, msg)


class AdamW:
    """The optimizer of lists of tensors: ``params`` (float32), their ``grads`` (float32 or bfloat16, each as
    it is), each contiguous, of any sizes, on the context's GPU, two of a place in the lists of as many values.

    ``m`` and ``v`` are lists of float32 tensors, or (states of 8 bits) of float8_e4m3fn or uint8 ones, with
    ``m_scale`` and ``v_scale``, float32 [ceil(n / 256)] each; ``step`` is an int32 tensor of one value, the steps done.
    They are the caller's to save and restore.  None of them given: new ones, of ``state_bits``, kept as the
    attributes of those names.  ``copies``: bfloat16 tensors (or None in a place) that receive the new parameters.
    ``weight_decay`` and ``lr_scale`` are numbers, or lists with one a tensor.  ``params`` None: a list of
    gradients alone, for ``grad_norm_async``.

    A handle keeps its tensors; ``close`` (or its end) gives its device tables to the context's next lists, but for
    those that a captured call has left to its graph, and a graph's tensors are the caller's to keep.  Calls only enqueue on
    the context's stream; the caller orders it with the streams that fill and read the tensors, and keeps ``lr``, ``grad_norm`` and
    ``norm`` until then."""

    def __init__(self, backend, params, grads, *, m=None, v=None, m_scale=None, v_scale=None, step=None, copies=None,
                 state_bits: int = 32, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, lr_scale=1.0, seed: int = 0):
        self._opt = C.c_void_p()
        self._backend = backend
        self._device = backend.device
        T = _torch()
        grads = list(grads)
        k = len(grads)
        alone = params is None
        if alone and any(x is not None for x in (m, v, m_scale, v_scale, step, copies)):
            raise _invalid("a list of gradients alone has no states and no copies")
        params = [None] * k if alone else list(params)
        given = [x is not None for x in (m, v, step)]
        if not alone and any(given) and not all(given):
            raise _invalid("m, v and step go together")
        if len(params) != k:
            raise _invalid(f"as many grads as params expected ({len(params)}), got {k}")
        either, single = (T["f32"], T["bf16"]), (T["f32"],)
        for i, (p, g) in enumerate(zip(params, grads)):
            self._check(g, "grads", i, either, None)
            if not alone:
                self._check(p, "params", i, single, g.numel())
        if not alone and not any(given):
            if m_scale is not None or v_scale is not None:
                raise _invalid("scales without states")
            m, v, m_scale, v_scale, step = self._new_state(params, state_bits)
        eight = False
        if not alone:
            m, v = list(m), list(v)
            eight = k > 0 and len(m) > 0 and getattr(m[0], "dtype", None) in T["codes"] or m_scale is not None
            if eight != (m_scale is not None) or eight != (v_scale is not None):
                raise _invalid("m_scale and v_scale go with states of 8 bits")
            m_scale, v_scale = (list(m_scale), list(v_scale)) if eight else ([None] * k, [None] * k)
            copies = [None] * k if copies is None else list(copies)
            for name, x in (("m", m), ("v", v), ("m_scale", m_scale), ("v_scale", v_scale), ("copies", copies)):
                if len(x) != k:
                    raise _invalid(f"{name} must have {k} entries, got {len(x)}")
            self._check(step, "step", None, (T["i32"],), 1)
        decay, scale = self._numbers(weight_decay, "weight_decay", k), self._numbers(lr_scale, "lr_scale", k)
        kinds, f32, block = T["codes"] if eight else (T["f32"],), T["f32"], _lib.ADAMW_BLOCK
        recs = (_lib.AdnAdamwTensor * max(k, 1))()
        for i, g in enumerate(grads):
            n, dtype = g.numel(), _lib.ADN_T_F32 if g.dtype is f32 else _lib.ADN_T_BF16
            if alone:
                recs[i] = (None, g.data_ptr(), None, None, None, None, None, n, 1.0, 0.0, dtype, 0)
                continue
            mp, vp, cp = self._check(m[i], "m", i, kinds, n), self._check(v[i], "v", i, kinds, n), None
            ms = vs = None
            if eight:
                blocks = -(-n // block)
                ms, vs = self._check(m_scale[i], "m_scale", i, (f32,), blocks), self._check(v_scale[i], "v_scale", i, (f32,), blocks)
            if copies[i] is not None:
                cp = self._check(copies[i], "copies", i, (T["bf16"],), n)
            recs[i] = (params[i].data_ptr(), g.data_ptr(), cp, mp, vp, ms, vs, n, scale[i], decay[i], dtype, 0)
        try:
            seed = int(seed)
        except _NO_NUMBER:
            seed = -1
        if not 0 <= seed < 1 << 64:
            raise _invalid("seed must be a number in [0, 2^64)")
        try:
            beta1, beta2 = betas
            cfg = _lib.AdnAdamwConfig(beta1=beta1, beta2=beta2, eps=eps, seed=seed, state_bits=0 if alone else 8 if eight else 32)
        except _NO_NUMBER:
            raise _invalid("betas must be two numbers and eps one") from None
        cfg.step = None if alone else step.data_ptr()
        check(lib().adn_adamw_create(backend._ctx, C.byref(cfg), k, recs, C.byref(self._opt)))
        self.params, self.grads, self.copies = params, grads, copies
        self.m, self.v, self.m_scale, self.v_scale, self.step = m, v, m_scale, v_scale, step

    def _check(self, t, name, i, dtypes, n):
        """The pointer of a contiguous tensor of n values (None: any number) on the context's GPU."""
        if not isinstance(t, _TORCH["tensor"]):
            raise _invalid(f"{name if i is None else f'{name}[{i}]'} must be a tensor, got {type(t).__name__}")
        if t.dtype not in dtypes or not t.is_contiguous() or (n is not None and t.numel() != n) or t.get_device() != self._device:
            name = name if i is None else f"{name}[{i}]"
            if t.dtype in dtypes and t.is_contiguous() and (n is None or t.numel() == n):
                raise _invalid(f"{name} must be on the context's GPU (cuda:{self._device}), got {t.device}")
            kinds = " or ".join(str(d) for d in dtypes)
            raise _invalid(f"{name} must be a contiguous {kinds} tensor" + ("" if n is None else f" of {n} values"))
        return t.data_ptr()

    @staticmethod
    def _numbers(x, name, k):
        """[k] floats: a number (of Python, numpy or torch) for all tensors, or one a tensor."""
        try:
            if isinstance(x, (int, float)) or getattr(x, "ndim", 1) == 0:
                return [float(x)] * k
            x = [float(v) for v in x]
        except _NO_NUMBER:
            raise _invalid(f"{name} must be a number or {k} of them") from None
        if len(x) != k:
            raise _invalid(f"{name} must be a number or {k} of them, got {len(x)}")
        return x

    def _new_state(self, params, state_bits):
        if state_bits not in (32, 8):
            raise _invalid("state_bits must be 32 or 8")
        T = _torch()
        torch, dev = T["torch"], f"cuda:{self._device}"
        eight = state_bits == 8

        def zeros(size):
            return [torch.zeros(size(p), device=dev, dtype=T["f32"]) for p in params]

        def codes():
            return [torch.zeros(p.shape, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn) for p in params]
        blocks = lambda p: -(-p.numel() // _lib.ADAMW_BLOCK)  # noqa: E731
        m, v = (codes(), codes()) if eight else (zeros(lambda p: p.shape), zeros(lambda p: p.shape))
        ms, vs = (zeros(blocks), zeros(blocks)) if eight else (None, None)
        step = torch.zeros(1, device=dev, dtype=T["i32"])
        torch.cuda.current_stream(self._device).synchronize()  # the context's stream is another one
        return m, v, ms, vs, step

    def grad_norm_async(self, norm) -> None:
        """norm [1] float32 = the square root of the sum of the squares of all gradients, summed in 64 bits."""
        if not self._opt:
            raise _invalid("the optimizer is closed")
        check(lib().adn_adamw_grad_norm_async(self._opt, self._backend._vector(norm, "norm", 1)))

    def step_async(self, *, lr=None, grad_norm=None, max_norm: float = 0.0, grad_scale: float = 1.0) -> None:
        """One step.  lr: a number, or a float32 tensor of one value that the step reads when it runs (a captured
        step's rate).  grad_norm: ``grad_norm_async``'s result; the step is skipped as a whole where it is not
        finite, and with max_norm > 0 the gradients are scaled so that their norm is at most max_norm.
        grad_scale is a factor of every gradient (and so of the norm)."""
        if not self._opt:
            raise _invalid("the optimizer is closed")
        try:
            s = _lib.AdnAdamwStep(max_norm=max_norm, grad_scale=grad_scale)
        except _NO_NUMBER:
            raise _invalid("max_norm and grad_scale must be numbers") from None
        vector = self._backend._vector
        if hasattr(lr, "data_ptr"):
            s.lr_device = vector(lr.reshape(1) if lr.numel() == 1 else lr, "lr", 1)
        else:
            try:
                s.lr = float(lr)
            except _NO_NUMBER:
                raise _invalid("lr must be a number or a tensor of one value") from None
        s.grad_norm = vector(grad_norm, "grad_norm", 1)
        check(lib().adn_adamw_step_async(self._opt, C.byref(s)))

    def close(self) -> None:
        if self._opt:
            lib().adn_adamw_destroy(self._opt)
            self._opt = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
