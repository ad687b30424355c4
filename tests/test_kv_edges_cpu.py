"""Edges of the rotary norm, the paged 8-bit cache and its attention that need no GPU."""
import pytest
import torch

from primus_dlrm_b200.ops.kv_cache import PagedKVCache, paged_attention


def test_copy_pages_outside_the_pool():
    c = PagedKVCache(4, 1, 32, 16)
    c.k_scale.copy_(torch.arange(4.0)[:, None] + 1)
    for src, dst in (([-1], [0]), ([0], [-1]), ([4], [0]), ([0], [4])):
        with pytest.raises(IndexError):
            c.copy_pages(torch.tensor(src), torch.tensor(dst))
    assert c.k_scale.flatten().tolist() == [1, 2, 3, 4]
    c.copy_pages(torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32))
    assert c.k_scale.flatten().tolist() == [2, 1, 3, 4]


def test_attention_has_no_gradient():
    c, table, lens = PagedKVCache(2, 1, 32, 16), torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    q = torch.randn(1, 2, 1, 32, requires_grad=True)
    o, lse = paged_attention(q, c, table, lens, return_lse=True)
    for y in (o, lse, paged_attention(q, c, table, lens)):
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward(retain_graph=True)
    with torch.no_grad():
        assert not paged_attention(q, c, table, lens).requires_grad
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            paged_attention(torch.autograd.forward_ad.make_dual(q.detach(), torch.ones(1, 2, 1, 32)), c, table, lens)


def test_models_that_score_without_a_cache():
    """A model whose ``score_candidates`` knows no cache is called as it always was, and refuses one."""
    from primus_dlrm_b200.evaluation.metrics import score_candidates

    class Model(torch.nn.Module):
        def score_candidates(self, user, cand, task, batch_size=1024):
            return cand["x"] * batch_size

    cand = {"x": torch.arange(3.0)}
    assert score_candidates(Model(), {}, cand, "t", 2).tolist() == [0, 2, 4]
    with pytest.raises(TypeError):
        score_candidates(Model(), {}, cand, "t", 2, kv_cache="fp8")


@pytest.mark.parametrize("rotary", [True, False])
def test_scores_over_8_bit_pages_are_near_the_exact_ones(rotary):
    """Keys and values carry 2^-4 relative error each, of random sign, averaged over some 30 tokens and added to a
    residual stream twice: a quarter of the scores' size bounds what reaches them by a wide margin, and any fault of
    pages or positions exceeds it."""
    from test_models_cpu import _batch
    from test_onetrans_rotary import _model, _split
    model = _model(rotary=rotary)
    user, cand, _ = _split(_batch(B=7, L=30, windows=2, seed=5), 7)
    with torch.no_grad():
        exact = model.score_candidates(user, cand, "listen_plus")
        got = model.score_candidates(user, cand, "listen_plus", kv_cache="fp8")
    assert (got - exact).abs().max() <= 0.25 * exact.abs().max()


def test_errors_of_a_cache_made_in_inference_mode():
    with torch.inference_mode():
        c = PagedKVCache(2, 1, 32, 16)
        c.err.fill_(1)
    with pytest.raises(RuntimeError, match="out of range"):
        c.check_errors()
    c.check_errors()


def test_copy_pages_of_other_kinds():
    """Lists, scalars for many, and shapes of ids as an assignment by index takes them; masks are no ids."""
    for src, dst, want in (([0], [1, 2], [1, 1, 1, 4]), (0, [3], [1, 2, 3, 1]), ([[0, 1]], [[2, 3]], [1, 2, 1, 2]), ([], [], [1, 2, 3, 4])):
        c = PagedKVCache(4, 1, 32, 16)
        c.k_scale.copy_(torch.arange(4.0)[:, None] + 1)
        c.copy_pages(src, torch.tensor(dst))
        assert c.k_scale.flatten().tolist() == want
    with pytest.raises(TypeError):
        c.copy_pages(torch.tensor([True, False, False, False]), torch.tensor([1]))
    with pytest.raises(TypeError):
        c.copy_pages(torch.tensor([0.0]), torch.tensor([1]))
