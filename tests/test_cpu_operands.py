"""Operands that a kernel would read or write out of range are refused before anything is launched (no GPU)."""

import pytest
import torch


@pytest.mark.parametrize("a,b", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                 (torch.float32, torch.float16)])
def test_gemm_refuses_operands_of_two_dtypes(a, b):
    """The kernel reads both operands as the first one's type: b of a smaller one would be read past its end."""
    from orthrus_training_b200 import ops

    with pytest.raises(ValueError, match="one dtype on one device"):
        ops.gemm(torch.zeros(4, 8, dtype=a), torch.zeros(6, 8, dtype=b))


def test_gemm_refuses_operands_of_two_devices():
    from orthrus_training_b200 import ops

    with pytest.raises(ValueError, match="one dtype on one device"):
        ops.gemm(torch.zeros(4, 8), torch.zeros(6, 8, device="meta"))
