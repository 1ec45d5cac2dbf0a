"""What stands in a tensor's place in the optimizer's lists and is none, as a parameter's gradient that no pass has made (needs an MI355X)."""
import numpy as np
import pytest
import torch

from aideen_amd import synth
from aideen_amd._lib import ADN_E_INVALID, AdnError
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    yield b
    b.close()


@pytest.mark.parametrize("other", [None, 0.0, [0.0] * 9, np.zeros(9, dtype=np.float32)], ids=["none", "number", "list", "array"])
@pytest.mark.parametrize("what", ["params", "grads", "m", "v", "m_scale", "v_scale", "step", "copies", "alone"])
@pytest.mark.parametrize("bits", [32, 8])
def test_refused(be, bits, what, other):
    z = lambda dtype=torch.float32, n=9: torch.zeros(n, device="cuda", dtype=dtype)  # noqa: E731
    kind = torch.float32 if bits == 32 else torch.uint8
    kw = dict(params=[z(), z()], grads=[z(), z()], m=[z(kind), z(kind)], v=[z(kind), z(kind)], step=z(torch.int32, 1), copies=[z(torch.bfloat16), None])
    if bits == 8:
        kw.update(m_scale=[z(n=1), z(n=1)], v_scale=[z(n=1), z(n=1)])
    torch.cuda.synchronize()
    if what == "alone":
        bad = lambda: be.adamw(None, [z(), other])  # noqa: E731
    elif what == "step" or (bits == 32 and what.endswith("scale")):
        bad = lambda: be.adamw(**{**kw, what: other if other is not None else [other]})  # noqa: E731
    else:
        for i in (0, 1):
            kw[what][i] = other
            if what == "copies" and other is None:
                be.adamw(**kw).close()  # no copy wanted there
                return
            with pytest.raises(AdnError) as ei:
                be.adamw(**kw)
            assert ei.value.code == ADN_E_INVALID and what in str(ei.value)
            kw[what][i] = kw[what][1 - i]
        return
    with pytest.raises(AdnError) as ei:
        bad()
    assert ei.value.code == ADN_E_INVALID
