"""CPU tests of arguments of the layer operators that are refused for what they hold: rows without features,
impossible values, missing inputs, half of a pair of outputs. Nothing goes to the library."""
import pytest
import torch

import xspmm_b200 as xs

f16, f32 = torch.float16, torch.float32


class HostExecutor:
    """Stands in for an executor whose tensors live on the host; a call past the checks fails the test."""
    device = torch.device("cpu")

    @property
    def handle(self):
        pytest.fail("the call went to the library")


EX = HostExecutor()


def t(*shape, dtype=f16):
    return torch.zeros(*shape, dtype=dtype)


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(EX, *args, **kw)


@pytest.mark.parametrize("rows", [0, 4])
def test_rows_without_features(rows):
    w, m = t(0, dtype=f32), t(rows, dtype=f32)
    refused("at least one column", xs.layer_norm, t(rows, 0), w, w, 1e-5, t(rows, 0))
    refused("at least one column", xs.layer_norm_backward, t(rows, 0), t(rows, 0), w, m, m)


@pytest.mark.parametrize("eps", [-1e-5, float("nan"), float("inf")])
def test_eps(eps):
    refused("eps must be", xs.layer_norm, t(4, 8), None, None, eps, t(4, 8))


def test_missing_inputs():
    m = t(4, dtype=f32)
    refused("mean is needed", xs.layer_norm_backward, t(4, 8), t(4, 8), None, None, m)
    refused("rstd is needed", xs.layer_norm_backward, t(4, 8), t(4, 8), None, m, None)
    x, w, y = t(4, 8), t(6, 8), t(4, 6)
    refused("gate is needed", xs.gated_ffn_backward, y, x, w, w, None, y)
    refused("up is needed", xs.gated_ffn_backward, y, x, w, w, y, None)


def test_half_of_the_weights_gradients():
    x, w, y = t(4, 8), t(6, 8), t(4, 6)
    refused("both or neither", xs.gated_ffn_backward, y, x, w, w, y, y, None, w)
    refused("both or neither", xs.gated_ffn_backward, y, x, w, w, y, y, None, None, w)
