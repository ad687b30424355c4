"""Edges of the rotary norm, the paged 8-bit cache and its attention on the GPU: values of very different sizes, rows
that nobody computes, refusals."""
import pytest
import torch
from test_kv_cache_gpu import DEV

pytestmark = pytest.mark.gpu


def test_an_empty_angle_table_is_refused():
    """Before anything is launched: the rows' angles would be read from a table that has none."""
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    x, none = torch.ones(1, 4, 2, 32, device=DEV), rope_table(0, 32, device=DEV)
    for positions in (None, torch.zeros(4, dtype=torch.int32, device=DEV)):
        with pytest.raises(IndexError, match="outside"):
            qk_norm_rope(x, x, None, None, none, positions)
        with pytest.raises(IndexError, match="outside"):
            qk_norm_rope(x[:, :0], x, None, None, none, positions)
    y, _ = qk_norm_rope(x[:, :0], None, None, None, none)              # no rows, no angles
    assert y.shape == (1, 0, 2, 32)


def test_weights_lie_on_the_device_of_the_rows():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    x, t = torch.ones(1, 4, 2, 32, device=DEV), rope_table(4, 32, device=DEV)
    for other in ["cpu"] + [f"cuda:{i}" for i in range(1, torch.cuda.device_count())]:
        w = torch.ones(32, device=other)
        for a, b in ((w, None), (None, w)):
            with pytest.raises(RuntimeError, match="on its device"):
                qk_norm_rope(x, x, a, b, t)
