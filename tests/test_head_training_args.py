"""Argument checks of the head's training operators that need no GPU."""
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


def test_null_context_is_an_error():
    L = _lib.lib()
    n = C.c_int32()
    assert L.adn_context_device(None, C.byref(n)) == ADN_E_INVALID
    assert L.adn_lm_loss_async(None, None) == ADN_E_INVALID
    assert L.adn_lm_loss_async(None, C.byref(_lib.AdnLmLossArgs())) == ADN_E_INVALID
    assert L.adn_rms_norm_async(None, 1, 1, 0, None, 1, None, 0.0, None, 1) == ADN_E_INVALID
    assert L.adn_rms_norm_backward_async(None, 1, 1, 0, None, 1, None, 0.0, None, 1, None, 1, None) == ADN_E_INVALID
    assert L.adn_embed_lookup_async(None, 1, 1, 1, 0, None, None, 1, 1.0, None, 1) == ADN_E_INVALID
    assert L.adn_embed_grad_async(None, 1, 1, 1, 0, None, None, 1, 1.0, None, 1) == ADN_E_INVALID
    assert L.adn_last_error().decode()


def test_args_struct_matches_the_header():
    text = open(_lib.HEADER).read()
    body = re.search(r"typedef struct adn_lm_loss_args \{(.*?)\} adn_lm_loss_args;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n for decl in body.split(";") for n in re.findall(r"\*?(\w+)\s*(?:,|$)", decl.strip())]
    assert names == [f[0] for f in _lib.AdnLmLossArgs._fields_]
    assert C.sizeof(_lib.AdnLmLossArgs) == 16 + 14 * 8
    assert re.search(r"#define ADN_T_F32 0u", text) and re.search(r"#define ADN_T_BF16 1u", text)


@pytest.mark.parametrize("f", [
    lambda b, m, v, t: b.lm_loss_async(m, t, w=m, outputs=dict(loss=v)),
    lambda b, m, v, t: b.lm_loss_async(m, t, w=m, outputs=dict(z=v)),
    lambda b, m, v, t: b.lm_loss_async(v, t, w=m, outputs=dict(loss=v)),
    lambda b, m, v, t: b.lm_loss_async(m, t, w=m[:, :3], outputs=dict(loss=v)),
    lambda b, m, v, t: b.lm_loss_async(m.half(), t, w=m.half(), outputs=dict(loss=v)),
    lambda b, m, v, t: b.rms_norm_async(m, m),
    lambda b, m, v, t: b.rms_norm_async(v, v),
    lambda b, m, v, t: b.rms_norm_backward_async(m, m, outputs=dict(dz=m)),
    lambda b, m, v, t: b.rms_norm_backward_async(m, m[:1], outputs=dict(dx=m)),
    lambda b, m, v, t: b.embed_lookup_async(t, m, table=m),
    lambda b, m, v, t: b.embed_lookup_async(t, v, table=m),
    lambda b, m, v, t: b.embed_grad_async(m, t, m),
    lambda b, m, v, t: b.embed_grad_async(m, t, m[:, :2]),
    lambda b, m, v, t: b.embed_grad_async(m, t, v),
])
def test_refused_before_the_library_is_called(f):
    """Host tensors, unknown names and shapes that do not fit."""
    m, v, t = torch.zeros((4, 8)), torch.zeros(4), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AdnError) as ei:
        f(host_backend(), m, v, t)
    assert ei.value.code == ADN_E_INVALID
