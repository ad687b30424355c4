"""The first GEMM of a thread that has bound no device yet."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_a_backward_pass_that_begins_with_a_gemm():
    """Autograd's thread has bound no device yet where a GEMM is the first call of the process's first backward pass."""
    code = """
import sys
sys.path.insert(0, %r)
import torch
from primus_dlrm_b200.ops import dense
x = torch.randn(2, 8, 64, device="cuda").bfloat16().requires_grad_()
w, wn = torch.randn(64, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(0, 64, 64, device="cuda").bfloat16()
y = dense.mixed_linear(x, 8, w, wn)
dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
torch.cuda.synchronize()
print("DONE", bool(dx.isfinite().all() and dw.isfinite().all()))
""" % str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert "DONE True" in r.stdout, r.stdout + r.stderr[-800:]
