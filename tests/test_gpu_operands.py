"""Operands of the LM-head products that are refused, and views that are taken (GPU)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_gemm_refusals():
    from orthrus_training_b200 import objective, ops

    h, W = torch.zeros(4, 16, device=DEV), torch.zeros(24, 16, device=DEV)
    for a, b in ((h, W.bfloat16()), (h.bfloat16(), W), (h, W.cpu())):
        with pytest.raises(ValueError, match="one dtype on one device"):
            ops.gemm(a, b)
        with pytest.raises(ValueError, match="one dtype on one device"):
            objective.teacher_top_logits(a, b, 2)
    for out in (torch.zeros(4, 23, device=DEV), torch.zeros(3, 24, device=DEV), torch.zeros(24, 4, device=DEV).t(),
                torch.zeros(4, 24, device=DEV, dtype=torch.bfloat16), torch.zeros(4, 24)):
        with pytest.raises(ValueError, match="writes a row-major"):
            ops.gemm(h, W, out=out)
