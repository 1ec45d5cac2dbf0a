"""Numbers of other kinds in the optimizer's arguments; needs no GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from aideen_amd import optimizer
from aideen_amd._lib import ADN_E_INVALID, AdnError
from test_optimizer_args import host_backend


@pytest.mark.parametrize("x", [0.25, 1, np.float32(0.25), np.float64(0.25), np.int64(3), np.array(0.25), torch.tensor(0.25), torch.tensor(2)])
def test_one_number_is_for_all_tensors(x):
    got = optimizer.AdamW._numbers(x, "weight_decay", 3)
    assert got == [float(x)] * 3 and all(type(v) is float for v in got)


@pytest.mark.parametrize("x", [[0.25, 1, np.float32(3)], (0.25, 1.0, 3.0), np.array([0.25, 1.0, 3.0], dtype=np.float32), torch.tensor([0.25, 1.0, 3.0])])
def test_one_number_a_tensor(x):
    assert optimizer.AdamW._numbers(x, "lr_scale", 3) == [0.25, 1.0, 3.0]


@pytest.mark.parametrize("x", [None, "0.1", "abc", [0.1, None, 0.2], [[0.1]] * 3, object(), 1j, np.array([0.1]), torch.zeros(2), torch.zeros(3, 2), [0.1, 0.2], 10 ** 400])
def test_what_is_no_number_is_refused(x):
    with pytest.raises(AdnError) as ei:
        optimizer.AdamW._numbers(x, "weight_decay", 3)
    assert ei.value.code == ADN_E_INVALID and "weight_decay" in str(ei.value)


@pytest.mark.parametrize("kw", [dict(betas=0.9), dict(betas=(0.9,)), dict(betas=("a", 0.9)), dict(betas=None), dict(betas=(0.9, 0.99, 0.999)), dict(eps="small"),
                                dict(eps=None), dict(seed="x"), dict(seed=None), dict(seed=[1]), dict(eps=torch.ones(2)), dict(betas=(torch.ones(2), 0.9)), dict(seed=float("inf"))])
def test_constants_of_other_kinds_are_refused(kw):
    with pytest.raises(AdnError) as ei:
        host_backend().adamw(None, [], **kw)
    assert ei.value.code == ADN_E_INVALID and list(kw)[0] in str(ei.value)


def test_constants_of_numpy_are_taken():
    """Refused by the library behind the checks alone, as this backend has no context."""
    with pytest.raises(AdnError) as ei:
        host_backend().adamw(None, [], betas=np.array([0.9, 0.99]), eps=np.float32(1e-6), seed=np.uint64(2 ** 64 - 1))
    assert "null argument" in str(ei.value)


@pytest.mark.parametrize("kw", [dict(max_norm="x"), dict(max_norm=None), dict(grad_scale="x"), dict(grad_scale=[1.0]), dict(max_norm=torch.ones(2)), dict(grad_scale=10 ** 400)])
def test_numbers_of_a_step_are_refused(kw):
    opt = optimizer.AdamW.__new__(optimizer.AdamW)
    opt._opt, opt._backend = C.c_void_p(1), host_backend()
    try:
        with pytest.raises(AdnError) as ei:
            opt.step_async(lr=1.0, **kw)
        assert ei.value.code == ADN_E_INVALID and list(kw)[0] in str(ei.value)
    finally:
        opt._opt = C.c_void_p()  # there is no list behind it
