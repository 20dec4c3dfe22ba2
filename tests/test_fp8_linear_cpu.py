"""What ``FP8BlockLinear`` refuses before anything is launched."""

import pytest
import torch

from practice_cuda_b200.fp8_linear import FP8BlockLinear
from practice_cuda_b200.registry import QuantResult


def test_quantized_input_of_another_kind_is_refused():
    """Scales or values that the kernels would read as what they are not, or from another device's memory."""
    lin = FP8BlockLinear(256, 128, bias=False)
    x = torch.zeros(4, 256)
    data, scale = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2)
    for bad in (
        QuantResult(data, scale.bfloat16(), "", "block", {}),
        QuantResult(data, scale.double(), "", "block", {}),
        QuantResult(data, scale.to("meta"), "", "block", {}),
        QuantResult(data.to("meta"), scale, "", "block", {}),
        QuantResult(data.to(torch.float8_e5m2), scale, "", "block", {}),
        QuantResult(data[:2], scale, "", "block", {}),
        QuantResult(data, scale[:, :1], "", "block", {}),
    ):
        with pytest.raises(ValueError, match="quantized input"):
            lin(x, bad)
    lin.scaling = "e8m0"
    with pytest.raises(ValueError, match="quantized input"):
        lin(x, QuantResult(data, scale, "", "block", {}))
