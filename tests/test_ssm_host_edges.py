"""CPU: calls of the state space mixer's and the norms' entry points that never reach a kernel."""
import warnings

import pytest
import torch

from hdla_impl_b200 import layer_ops, ssm


def calls_of_all():
    """Calls of the five entry points between other operations, on the CPU."""
    x, w, A, bc = torch.zeros(1, 4, 8), torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(1, 4, 2)
    return [(lambda x, w: ssm.short_convolution(x + 1, w, cu_seqlens=[0, 4])[0] * 2, x, w),
            (lambda x, w: ssm.short_convolution_step(x + 1, torch.zeros(1, 3, 8), w) * 2, x[:, 0], w),
            (lambda x, bc: ssm.selective_scan(x + 1, x, A, bc, bc)[0] * 2, x, bc),
            (lambda x, bc: ssm.selective_scan_step(x + 1, x, A, bc, bc, torch.zeros(1, 8, 2)) * 2, x[:, 0], bc[:, 0]),
            (lambda x, w: layer_ops.rms_norm_residual(x + 1, pre_weight=w)[1] * 2, x, w[:, 0])]


@pytest.mark.parametrize("k", range(5))
def test_torch_compile_leaves_the_calls_out_without_complaint(k):
    """A compiled function reaches the call as it is (here: its refusal of CPU tensors), with no warning that the compiler met
    something that it does not know."""
    f, a, b = calls_of_all()[k]
    torch._dynamo.reset()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            torch.compile(f, backend="eager")(a, b)
