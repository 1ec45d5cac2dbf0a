"""AdamW at the ends of its documented range: coefficients and second moments below the normal numbers of fp32, arguments within
the list's own tensors (needs an MI355X).
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


@pytest.mark.parametrize("bits", [32, 8])
def test_words_of_a_step_within_its_tensors_are_refused(be, bits):
    """The rate and the norm are read by all workgroups of a step: not from what some of them have written.  The norm is not
    written over a gradient or a state either; beside them is fine."""
    flat, norm = torch.zeros(1000, device="cuda"), torch.zeros(1, device="cuda")
    lst = List([300, 40], bits, copy=lambda i: True)
    lst.p[1] = flat[500:540]
    lst.g[1] = flat[600:640]
    opt = lst.optimizer(be)
    word = lambda t: t.view(-1).view(torch.uint8)[:4].view(F32)  # noqa: E731
    written = [lst.p[0][:1], lst.p[0][299:], flat[500:501], flat[539:540], word(lst.m[0]), word(lst.v[1]), opt.step.view(F32)]
    written += [lst.copy[0][2:4].view(F32)] + ([lst.ms[0][1:], lst.vs[1][:1]] if bits == 8 else [])
    for w in written:
        for kw in (dict(lr=w), dict(lr=1.0, grad_norm=w)):
            with pytest.raises(AdnError) as ei:
                opt.step_async(**kw)
            assert ei.value.code == ADN_E_INVALID and "overlap" in str(ei.value)
    for w in written + [lst.g[0][5:6], flat[600:601], flat[639:640]]:
        with pytest.raises(AdnError) as ei:
            opt.grad_norm_async(w)
        assert ei.value.code == ADN_E_INVALID and "overlap" in str(ei.value)
    torch.cuda.synchronize()
    before, cfg = lst.host(), cfg_of(lst)
    flat[499:500].fill_(1e-3)
    torch.cuda.synchronize()
    opt.grad_norm_async(flat[540:541])
    opt.grad_norm_async(norm)
    opt.step_async(lr=flat[499:500], grad_norm=flat[540:541])
    be.synchronize()
    assert torch.equal(flat[540:541], norm)
    cfg["lr"] = float(flat[499])
    lst.check(before, cfg)


def test_a_rate_beyond_fp32_is_refused(be):
    lst = List([40], 32)
    opt = lst.optimizer(be)
    for lr in (3.5e38, -1e39, 1e300):
        with pytest.raises(AdnError) as ei:
            opt.step_async(lr=lr)
        assert ei.value.code == ADN_E_INVALID
    for t in lst.g + lst.m:
        t.zero_()
    before = lst.p[0].clone()
    torch.cuda.synchronize()
    lst.wd = [0.0]
    lst.optimizer(be).step_async(lr=3.4e38)
    be.synchronize()
    assert torch.equal(lst.p[0], before)


@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_a_rate_on_the_device_of_any_shape(be, shape):
    """A tensor of one value is one whatever its dimensions."""
    lst, rate = List([300], 32), torch.full(shape, 2e-3, device="cuda")
    opt, cfg, before = lst.optimizer(be), cfg_of(lst, float(rate)), lst.host()
    torch.cuda.synchronize()
    opt.step_async(lr=rate)
    be.synchronize()
    lst.check(before, cfg)
    for bad in (torch.zeros(shape, device="cuda", dtype=torch.float64), torch.zeros(shape), torch.zeros((0,), device="cuda"), torch.zeros((2, 1), device="cuda")):
        with pytest.raises(AdnError) as ei:
            opt.step_async(lr=bad)
        assert ei.value.code == ADN_E_INVALID
