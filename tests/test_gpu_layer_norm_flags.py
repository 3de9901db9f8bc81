"""layer_norm_backward's `need` takes any truth values, whatever the layout of the rows."""

import numpy as np
import pytest
import torch

import apexw_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("need", [(1, 1, 1), (1, 0, 1), (0, 2, 0), tuple(np.array([True, True, False])), [True, 1, 0.0],
                                  ("x", "", None)])
def test_any_truth_value(need, strided):
    x = torch.randn(30, 80, device="cuda")
    x = x[:, 8:72] if strided else x[:, :64].contiguous()
    w, b, dy = torch.randn(64, device="cuda"), torch.randn(64, device="cuda"), torch.randn(30, 64, device="cuda")
    _, mean, rstd = apexw_amd.layer_norm_forward(x, w, b)
    whole = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b)
    some = apexw_amd.layer_norm_backward(dy, x, mean, rstd, w, b, need)
    for a, s, n in zip(whole, some, need):
        assert torch.equal(a, s) if n else s is None


class Undecided:
    def __bool__(self):
        raise ArithmeticError("neither")


@pytest.mark.parametrize("strided", [False, True])
def test_an_error_of_a_flag_is_raised(strided):
    x = torch.randn(30, 80, device="cuda")[:, 8:72]
    x = x if strided else x.contiguous()
    _, mean, rstd = apexw_amd.layer_norm_forward(x)
    with pytest.raises(ArithmeticError):
        apexw_amd.layer_norm_backward(x, x, mean, rstd, None, None, (Undecided(), True, True))
