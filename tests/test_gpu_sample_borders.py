"""How near to a border a drawn token can differ from the 64-bit definition (GPU).

A weight is rounded to a multiple of 2^-S of the largest, S = min(44, 62 - ceil(log2 V)), so the sum of V
of them is off by at most V 2^-(S+1); the exponentials, and the fp64 that brings a slice to the row's
maximum, add less than 2^-42. The rows here are the worst case: one peak above entries that weigh 0.45 of
a unit each, which all round to nothing where they stand in the peak's slice."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bits(V):
    return min(44, 62 - math.ceil(math.log2(V)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,batch", [(2 ** 20, 9), (151936, 8), (151936, 130), (50257, 8), (50257, 400), (1000, 64)])
def test_tail_of_lost_weights(V, batch, dtype):
    """The token's own interval of the 64-bit running sum holds the uniform, give or take the bound, in
    batches that cut the row into slices of 2048 and of 8192 entries."""
    from orthrus_training_b200 import ops

    S = _bits(V)
    bound = V * 2.0 ** -(S + 1) + 2.0 ** -42
    u = torch.tensor([0.0, 2.0 ** -40, 2.0 ** -30, 2.0 ** -28.5, 2.0 ** -26, 2.0 ** -24, 0.25, 0.5, 1 - 2.0 ** -24])
    u = u.repeat(batch // len(u) + 1)[:batch].float().to(DEV)
    for peak in (V - 1, V // 2 + 1, 0):
        for f in (dict(), dict(top_p=1 - 2.0 ** -24), dict(top_k=V - 1)):
            row = torch.full((V,), math.log(0.45) - S * math.log(2.0), device=DEV).to(dtype)
            row[peak] = 0.0
            token = ops.sample_logits(row.expand(batch, V), u, **f)
            w = row.double().exp()
            c = w.cumsum(0)
            lo, hi, total = (c - w)[token], c[token], c[-1]
            assert (lo / total - bound <= u.double()).all() and (u.double() <= hi / total + bound).all(), (peak, f)
