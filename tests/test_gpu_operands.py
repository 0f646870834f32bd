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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 33])
def test_teacher_top_logits_of_views(dtype, d):
    """Rows and an LM head that start off a 16-byte boundary, or are strided, give what their copies give."""
    from orthrus_training_b200 import objective

    g = torch.Generator().manual_seed(d)
    flat = torch.randn(70 * d + 3, generator=g).to(DEV, dtype)
    wide = torch.randn(200, d + 5, generator=g).to(DEV, dtype)
    head = torch.randn(200 * d + 1, generator=g).to(DEV, dtype)
    for h, W in ((flat[3:].view(70, d), wide[:, 2 : d + 2]), (wide[::3, 1 : d + 1], head[1:].view(200, d))):
        got = objective.teacher_top_logits(h, W, 9, chunk_rows=32)
        want = objective.teacher_top_logits(h.clone().contiguous(), W.clone().contiguous(), 9, chunk_rows=32)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
