"""States of 8 bits beside those of 32 over some hundred steps (needs an MI355X).

All values of a list have the gradient c at every step, so that in 32 bits each step is lr (but for eps).  In 8 bits m and v are
rounded by independent bits whose expectation is the value: E[m] = its exact value, E[v] too, and the expected step is lr E[x^(-1/2)], x = v / E[v].
At least 1 (Jensen).  A rounding of b2 v + (1 - b2) c^2, v being a code of step v / 8 at most, has a variance of at most its distance to the code times the
step: (1 - b2) c^2 v / 8, and v is at most (1 - b2) t c^2: the variances of T steps sum to at most ((1 - b2) T c^2)^2 / 16, so that var x <= 1/16 for T well below
1 / (1 - b2) (0.26 at T = 300, where v is 0.26 c^2).  x^(-1/2) <= 1 - (x - 1) / 2 + 1.12 (x - 1)^2 for x >= 1/4, three deviations below 1, beyond which there is one
value in some hundred at a step of a few lr: E <= 1 + 1.12 / 16 + 0.02 = 1.09.  Over 65536 values the mean of independent runs, each with a deviation of less than 1/3 of its own
length (m's and v's), is within 5 * 0.0014 = 0.007."""
import pytest
import torch

from aideen_amd import synth
from aideen_amd.backend import GpuDeqBackend

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def be():
    b = GpuDeqBackend(synth.ModelConfig(d=64, H=2, V=300, N=1, flags=0), 1, 1)
    yield b
    b.close()


@pytest.mark.parametrize("c", [1e-3, -2.0, 1e-12])
def test_a_run_goes_as_far_as_in_32_bits(be, c):
    n, steps, lr = 65536, 300, 1e-3
    far = {}
    for bits in (32, 8):
        p, g = torch.zeros(n, device="cuda"), torch.full((n,), c, device="cuda")
        opt = be.adamw([p], [g], state_bits=bits, eps=1e-20, weight_decay=0.0, seed=11)
        torch.cuda.synchronize()
        for _ in range(steps):
            opt.step_async(lr=lr)
        be.synchronize()
        far[bits] = float(p.double().mean()) * (-1 if c > 0 else 1)
        if bits == 32:
            # v carries at most u a step (b2's rounding and the sum's), half of it under the root, m ten steps' at a time: with a step's own
            # 36 u at most 220 u of lr a step, and as many roundings of p of half a step of fp32 at 0.3
            assert abs(far[32] - steps * lr) <= steps * (220 * 2.0 ** -24 * lr + 2.0 ** -26)
        else:
            for scale, codes, want in ((opt.m_scale, opt.m, c), (opt.v_scale, opt.v, c * c * (1 - 0.999 ** steps))):
                got = float((codes[0].float().double().view(-1, 256) * scale[0].double()[:, None]).mean())
                assert abs(got - want) <= 0.007 * abs(want)
        opt.close()
    assert 0.993 <= far[8] / far[32] <= 1.097


def test_gradients_far_below_their_blocks_largest_step_less(be):
    """The smallest code of v is 2^-16 to 2^-17 of the block's largest v.  A gradient of 2^-6 of the largest keeps codes of 3 bits, 1/8 at most
    from v, and so the step of 32 bits within 1/16 and that of the value itself.  One of 2^-12 has the smallest code after the first step: with beta1 = 0, of which m is the
    gradient, the second is 2^-12 / sqrt(2^-16 to 2^-17 times (1 - b2) / (1 - b2^2) = 1/2), 1/8 to 1/11.4 of the rate."""
    n, lr = 256, 1e-3
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 2.0 ** -12, device="cuda")
    g[0] = 1.0
    g[1:9] = 2.0 ** -6
    opt = be.adamw([p], [g], state_bits=8, betas=(0.0, 0.999), eps=1e-20, weight_decay=0.0, seed=11)
    torch.cuda.synchronize()
    opt.step_async(lr=lr)
    be.synchronize()
    first = p.double().clone()
    assert float((first / -lr - 1).abs().max()) <= 40 * 2.0 ** -24  # the first is taken from the moments as they are formed
    opt.step_async(lr=lr)
    be.synchronize()
    step = (p.double() - first) / -lr
    assert bool((step[0:1] - 1).abs().max() <= 0.07)
    assert bool(((step[1:9] > 0.9) & (step[1:9] < 1.1)).all())
    assert bool(((step[9:] > 1 / 11.5) & (step[9:] < 1 / 7.5)).all())
