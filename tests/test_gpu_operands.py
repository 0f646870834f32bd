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


def test_distillation_refuses_an_empty_head():
    from orthrus_training_b200 import ops

    for dtype in (torch.float32, torch.bfloat16):
        h, v, i = torch.zeros(4, 8, device=DEV, dtype=dtype), torch.zeros(4, 2, device=DEV), torch.zeros(4, 2, device=DEV).long()
        with pytest.raises(ValueError):
            ops.lmhead_topk_kl(h, v, i, None, torch.zeros(0, 8, device=DEV, dtype=dtype))
        with pytest.raises(ValueError):
            ops.lmhead_topk_kl(h[:, :0], v, i, None, torch.zeros(6, 0, device=DEV, dtype=dtype))
