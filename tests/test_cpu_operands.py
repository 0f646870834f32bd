"""Operands that a kernel would read or write out of range are refused before anything is launched (no GPU)."""

import subprocess
import sys

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


def test_distillation_workspace_of_refused_sizes():
    """Sizes that the distillation refuses need no workspace; asking for it does not end the process (in one
    of its own, which a division by no tiles would end)."""
    from orthrus_training_b200 import _lib as L

    calls = []
    for bad in (dict(V=0), dict(d=0), dict(V=-7), dict(d=-1), dict(n=-1), dict(m=-1), dict(k=0), dict(k=1025),
                dict(n=2 ** 31), dict(V=2 ** 31), dict(dtype=7)):
        for dtype in (L.F32, L.BF16):
            a = dict(dict(n=4, m=4, V=10, d=8, k=2, chunk=4096, dtype=dtype), **bad)
            calls.append(tuple(a.values()))
    code = ("from orthrus_training_b200 import _lib as L\n"
            f"print([L.lib().orthrus_lmhead_topk_kl_workspace_bytes(*c) for c in {calls}])")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == str([0] * len(calls)), (run.returncode, run.stdout, run.stderr[-500:])


@pytest.mark.parametrize("size", ["n", "V", "d"])
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_distillation_refuses_sizes_past_its_loops(size, dtype):
    """Loops over rows, entries and columns step past their end in 32 bits: near 2^31 they would wrap around."""
    import ctypes

    from orthrus_training_b200 import _lib as L

    a = dict(dict(n=4, V=10, d=8), **{size: 2 ** 31 - 512})
    got = L.lib().orthrus_lmhead_topk_kl_fwd(64, a["n"], 64, 64, 2 ** 31 - 1, 2, 64, None, 64, a["V"], a["d"], ctypes.c_float(1.0),
                                             None, None, 0, 64, 64, 64, 64, None, None, 128, 64, 1 << 62, getattr(L, dtype),
                                             None)
    assert got == L.EINVAL


@pytest.mark.parametrize("at", [65, 66, 68, 72])
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_workspaces_off_their_boundary(dtype, at):
    import ctypes

    from orthrus_training_b200 import _lib as L

    lib, f, code = L.lib(), ctypes.c_float, getattr(L, dtype)
    assert lib.orthrus_topk_rows(64, 8, 2, 8, 2, f(1), 64, 64, 64, at, 1 << 50, code, None) == L.EINVAL
    assert lib.orthrus_sample_logits(64, 8, 2, 8, 64, None, f(1), None, 0, None, f(1), None, f(0), 64, at, 1 << 50, code,
                                     None) == L.EINVAL
    assert lib.orthrus_lmhead_topk_kl_fwd(64, 4, 64, 64, 4, 2, 64, None, 64, 10, 8, f(1), None, None, 0, 64, 64, 64, 64, None,
                                          None, 128, at, 1 << 50, code, None) == L.EINVAL
