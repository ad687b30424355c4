"""The error word of the GEMMs."""

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
