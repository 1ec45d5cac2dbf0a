"""Argument checks of the residual norms and the optimizer that need no GPU."""
import ctypes as C
import re

import pytest
import torch

from aideen_amd import _lib, synth
from aideen_amd._lib import ADN_E_INVALID, AdnError
from aideen_amd.backend import GpuDeqBackend


def host_backend():
    """A backend without a context: enough for the checks that come before the library call."""
    be = GpuDeqBackend.__new__(GpuDeqBackend)
    be.model = synth.ModelConfig(d=64, H=2, V=300)
    be._ctx, be._device = None, 0
    return be


def test_null_arguments_are_errors():
    L = _lib.lib()
    opt = C.c_void_p(1)
    assert L.adn_residual_norm_async(None, None) == ADN_E_INVALID
    assert L.adn_residual_norm_backward_async(None, C.byref(_lib.AdnResidualNormArgs())) == ADN_E_INVALID
    assert L.adn_adamw_create(None, C.byref(_lib.AdnAdamwConfig()), 0, None, C.byref(opt)) == ADN_E_INVALID
    assert not opt.value  # the handle is null after an error
    assert L.adn_adamw_create(None, None, 0, None, None) == ADN_E_INVALID
    assert L.adn_adamw_grad_norm_async(None, None) == ADN_E_INVALID
    assert L.adn_adamw_step_async(None, None) == ADN_E_INVALID
    L.adn_adamw_destroy(None)
    assert L.adn_last_error().decode()


@pytest.mark.parametrize("name,mirror,size", [("adn_residual_norm_args", _lib.AdnResidualNormArgs, 40 + 24 * 8),
                                              ("adn_adamw_tensor", _lib.AdnAdamwTensor, 8 * 8 + 16),
                                              ("adn_adamw_config", _lib.AdnAdamwConfig, 5 * 8 + 8), ("adn_adamw_step", _lib.AdnAdamwStep, 3 * 8 + 8)])
def test_structs_match_the_header(name, mirror, size):
    text = open(_lib.HEADER).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in body.split(";") for n in re.findall(r"\*?(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [f[0] for f in mirror._fields_]
    assert C.sizeof(mirror) == size


@pytest.mark.parametrize("f", [
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m)),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(w=m)),
    lambda b, m, v: b.residual_norm_async(m, v, outputs=dict(z=m)),
    lambda b, m, v: b.residual_norm_async(m[:, :3], m, outputs=dict(z=m)),
    lambda b, m, v: b.residual_norm_async(m.half(), m.half(), outputs=dict(z=m.half())),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m), gate=v),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m), gate=m[:2]),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m), gate=m[:3, :1]),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m), gate=v.sum()),
    lambda b, m, v: b.residual_norm_async(m, m, outputs=dict(z=m), gate=m[None]),
    lambda b, m, v: b.residual_norm_backward_async(m, m, outputs=dict(dz=m)),
    lambda b, m, v: b.residual_norm_backward_async(m, m, dy=m, outputs=dict(dgate=m)),
    lambda b, m, v: b.residual_norm_backward_async(m, m, dy=m[:1], outputs=dict(dx=m)),
    lambda b, m, v: b.residual_norm_backward_async(m, v, dy=m, outputs=dict(dx=m)),
    lambda b, m, v: b.adamw([m], [m]),
    lambda b, m, v: b.adamw([m], []),
    lambda b, m, v: b.adamw([m], [v]),
    lambda b, m, v: b.adamw([m.bfloat16()], [m]),
    lambda b, m, v: b.adamw([m[:, :3]], [m[:, :3]]),
    lambda b, m, v: b.adamw([], [], m=[]),
    lambda b, m, v: b.adamw(None, [], step=v),
    lambda b, m, v: b.adamw([], [], m=[], v=[], step=v, m_scale=[]),
    lambda b, m, v: b.adamw([], [], m_scale=[], v_scale=[]),
    lambda b, m, v: b.adamw([], [], state_bits=4),
])
def test_refused_before_the_library_is_called(f):
    """Host tensors, unknown names, shapes and lists that do not fit."""
    m, v = torch.zeros((4, 8)), torch.zeros(4)
    with pytest.raises(AdnError) as ei:
        f(host_backend(), m, v)
    assert ei.value.code == ADN_E_INVALID
