"""Calls of the 4-bit operators that are refused on the host, and rules of their kernels that are checked on the sources."""
import pytest
import torch

from fastllm_py_b200.native import mxfp4
from fastllm_py_b200.native.ops import KernelError


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("kernel", [0, 1, 2])
def test_a_gated_product_has_a_unit(kernel):
    """Without one the up half would have no place in the result; a plain product goes without."""
    w = mxfp4.Matrix.empty(64, 96, "cpu")
    with pytest.raises(KernelError, match="activation"):
        mxfp4.linear_gated(bf(5, 96), w, bf(5, 32), activation=None, kernel=kernel)
    with pytest.raises(KernelError, match="activation"):
        mxfp4.linear_gated(bf(0, 96), w, bf(0, 32), None)
    with pytest.raises(KernelError, match="CUDA device only"):
        mxfp4.linear(bf(5, 96), w, bf(5, 64), activation=None, kernel=kernel)
