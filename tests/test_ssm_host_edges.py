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


@pytest.mark.parametrize("cu", [[0, 2.5, 4], [0.0, 4.0], torch.tensor([0, 2.5, 4]), torch.tensor([[0, 4]]), torch.tensor(4), 4, ["0", "4"]])
def test_offsets_that_are_no_whole_numbers_are_refused(cu):
    """None is cut to a whole number in silence: those on the host are refused as those on the GPU are."""
    x, w, A, bc = torch.zeros(1, 4, 8), torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(1, 4, 2)
    for f in (lambda: ssm.short_convolution(x, w, cu_seqlens=cu), lambda: ssm.selective_scan(x, x, A, bc, bc, cu_seqlens=cu)):
        with pytest.raises(ValueError, match="vector of integers"):
            f()


@pytest.mark.parametrize("shape", [(8,), (4, 8), (1, 1, 4, 8)])
def test_inputs_of_other_dimensions_are_refused_with_offsets_too(shape):
    x, w, A, bc = torch.zeros(shape), torch.zeros(8, 4), torch.zeros(8, 2), torch.zeros(1, 4, 2)
    for f in (lambda: ssm.short_convolution(x, w, cu_seqlens=[0, 4]), lambda: ssm.selective_scan(x, x, A, bc, bc, cu_seqlens=[0, 4])):
        with pytest.raises(ValueError, match="3 dimensions"):
            f()


def test_offsets_of_any_whole_number_type_are_taken():
    """(As far as the refusal of CPU tensors.)"""
    import numpy as np
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    for cu in ([0, 4], (0, 2, 4), np.array([0, 4], dtype=np.int32), torch.tensor([0, 4], dtype=torch.int32), list(torch.tensor([0, 4])), range(0, 5)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            ssm.short_convolution(x, w, cu_seqlens=cu)
