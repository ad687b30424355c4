"""The error word of the GEMMs."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from primus_dlrm_b200.ops import dense

pytestmark = pytest.mark.gpu


def test_a_device_without_an_index_is_the_current_one():
    dense.tc_gemm(*(torch.zeros(1, 64, 64, device="cuda").bfloat16() for _ in range(3)))
    word = dense._err(torch.device("cuda", torch.cuda.current_device()))
    try:
        word.fill_(2)
        assert dense.gemm_error_code("cuda") == dense.gemm_error_code("cuda:0") == 2
    finally:
        word.zero_()
    assert dense.gemm_error_code("cuda") == 0


def test_a_first_call_inside_a_capture():
    """The word of a process whose first GEMM is captured is 0 before the replay, and a replay does not clear what it holds;
    made under inference mode, it serves a training step. In a process of its own."""
    code = """
import sys
sys.path.insert(0, %r)
import torch
from primus_dlrm_b200.ops import dense
t = [torch.zeros(1, 64, 64, device="cuda").bfloat16() for _ in range(3)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.inference_mode(), torch.cuda.graph(graph):
    dense.tc_gemm(*t)
word = dense._err(t[0].device)
print("INFERENCE", word.is_inference())
print("BEFORE", int(word.item()))
with torch.inference_mode():
    word.fill_(2)
graph.replay()
print("AFTER", int(word.item()))
with torch.inference_mode():
    word.zero_()
x, w = (torch.ones(1, 64, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
y = dense.mixed_linear(x, 64, w[0], w[:0], save8=True)
y.sum().backward()
print("TRAINED", float(x.grad[0, 0, 0]))
""" % str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]
    assert all(m in r.stdout for m in ("INFERENCE False", "BEFORE 0", "AFTER 2", "TRAINED 64.0")), r.stdout


def test_the_attention_has_a_word_of_its_own():
    """Asked for without an index, apart from the GEMMs', made in any mode, raised once."""
    from primus_dlrm_b200.ops import attention
    with torch.inference_mode():
        word = attention._err_word("cuda")
    assert not word.is_inference() and word.data_ptr() != dense._err("cuda").data_ptr()
    try:
        word.fill_(2)
        assert attention.attention_error_code("cuda") == attention.attention_error_code("cuda:0") == 2
        assert dense.gemm_error_code("cuda") == 0
        dense.check_errors("cuda")
        with pytest.raises(RuntimeError, match="attention: a bounded wait"):
            attention.check_errors("cuda")
        attention.check_errors("cuda")
    finally:
        word.zero_()
