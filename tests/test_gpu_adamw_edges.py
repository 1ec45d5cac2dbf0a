"""AdamW at the ends of its documented range: coefficients and second moments below the normal numbers of fp32 (needs an MI355X).
Definition and tolerances are those of the optimizer's own tests."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd._lib import ADN_E_INVALID, AdnError
from aideen_amd.backend import GpuDeqBackend
from test_gpu_adamw import List, cfg_of, log, one_step

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 2, 8)
    yield b
    b.close()


def fresh(lst):
    for t in lst.m + lst.v:
        t.view(torch.uint8).zero_()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm,grad_scale", [(1e-9, 1.0), (1e-7, 1e-10), (0.0, 1e-40)])
def test_a_coefficient_below_the_normal_numbers(be, bits, max_norm, grad_scale):
    """Large gradients times a coefficient of fewer than 24 bits in fp32: the moments keep the definition's 6 and 10 u."""
    log(f"coefficient {bits} {max_norm} {grad_scale}")
    lst = List([600, 0, 5, 1025], bits, grad=lambda i: BF16 if i == 2 else F32)
    fresh(lst)
    for t in lst.g:
        t.mul_(1e33)
    opt, norm = lst.optimizer(be, eps=1e-15), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    opt.grad_norm_async(norm)
    be.synchronize()
    scale = float(torch.tensor(grad_scale))  # as the call holds it
    limit = float(torch.tensor(max_norm))
    coef = scale * (min(1.0, limit / (float(norm) * scale + 1e-6)) if max_norm else 1.0)
    assert coef < 2.0 ** -126
    cfg, before = cfg_of(lst, coef=coef, eps=1e-15), lst.host()
    opt.step_async(lr=1e-3, grad_norm=norm, max_norm=max_norm, grad_scale=grad_scale)
    be.synchronize()
    lst.check(before, cfg)


@pytest.mark.parametrize("bits", [32, 8])
def test_second_moments_below_the_normal_numbers(be, bits):
    """v' in [2^-127.5, 2^-126], which a bias correction of 2^-30 makes 2^-15 of eps under the root: 512 u of the way, where 36 u are allowed.
    v' itself is rounded to 2^-150, 1.4 u of its root, which is 2^-15 of the denominator."""
    lst = List([700, 3], bits)
    fresh(lst)
    g = torch.Generator(device="cuda").manual_seed(2)
    for t, p in zip(lst.g, lst.p):
        t.copy_(2.0 ** -48 * (0.6 + 0.4 * torch.rand(t.shape, device="cuda", generator=g)))
        t[1::2].neg_()
        p.zero_()
    lst.step.zero_()
    cfg, before, _ = one_step(be, lst, betas=(0.9, 1 - 2.0 ** -30), eps=2.0 ** -33)
    lst.check(before, cfg)
