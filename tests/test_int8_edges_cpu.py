"""Products of 8-bit integers and layers with activations in 8 bits on the CPU: calls at the edge."""
import pytest
import torch
from torch.autograd import forward_ad

from primus_dlrm_b200.ops import dense
from primus_dlrm_b200.ops.int8 import Int8Weight, int8_linear, quantize_rows
from primus_dlrm_b200.ops.saved8 import load8, save8


def test_tangents_are_refused():
    """Forward-mode derivatives are refused as on the GPU, not dropped and not taken of the scales alone."""
    w, x = Int8Weight.from_float(torch.randn(5, 20)), torch.randn(4, 20)
    bias, res = torch.randn(5), torch.randn(4, 5)
    layer = [torch.randn(s).requires_grad_() for s in ((2, 7, 64), (2, 7, 64), (64, 64), (64, 64), (3, 64, 64), (3, 64, 64))]
    plain, saved = int8_linear(x, w, bias, residual=res), save8(x)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.detach(), torch.ones_like(t))  # noqa: E731
        for bad in (lambda: int8_linear(dual(x), w), lambda: int8_linear(x, w, dual(bias)),
                    lambda: int8_linear(x, w, residual=dual(res)), lambda: quantize_rows(dual(x)),
                    lambda: Int8Weight.from_float(dual(x)), lambda: Int8Weight.from_tensors(w.codes, dual(w.scale)),
                    lambda: save8(dual(x)), lambda: dense.mixed_linear(dual(layer[0]), 4, layer[2], layer[4], save8=True),
                    lambda: dense.mixed_ffn(dual(layer[0]), layer[1], 4, *layer[2:], save8=True)):
            with pytest.raises(RuntimeError, match="forward"):
                bad()
        # inside a level, but without a tangent
        assert torch.equal(int8_linear(x, w, bias, residual=res), plain) and torch.equal(save8(x).codes, saved.codes)
        assert torch.equal(load8(saved), load8(save8(x)))
    with torch.inference_mode():
        assert torch.equal(int8_linear(x, w, bias, residual=res), plain)


def test_scoring_reports_a_product_that_gave_up(monkeypatch):
    """Scores of integer weights do not leave before the products' error word was read; those of others do not read it."""
    from primus_dlrm_b200.ops import int8
    from test_models_cpu import _batch
    from test_onetrans_rotary import _model, _split
    model = _model(rotary=True)
    user, cand, _ = _split(_batch(B=5, L=30, windows=2, seed=5), 5)
    w8, asked = model.int8_weights(), []
    want = model.score_candidates(user, cand, "listen_plus", weights=w8)
    monkeypatch.setattr(int8, "check_errors", lambda device: asked.append(device))
    assert torch.equal(model.score_candidates(user, cand, "listen_plus", weights=w8), want) and asked == [torch.device("cpu")]
    model.score_candidates(user, cand, "listen_plus")
    assert len(asked) == 1

    # the code that a kernel leaves, read from a stub: raised once, and cleared
    monkeypatch.undo()
    word = torch.tensor([2], dtype=torch.int32)
    monkeypatch.setattr(int8, "_err_word", lambda device: word)
    with pytest.raises(RuntimeError, match="wait"):
        int8.check_errors("cuda")
    int8.check_errors("cuda")
    word.fill_(4)
    int8.check_errors("cpu")
    with pytest.raises(RuntimeError, match="aligned"):
        int8.check_errors("cuda:0")


def _layer_parts(dtype, seed=0, D=64, F_=128):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, z = r(2, 9, D).to(dtype), r(2, 9, D).to(dtype)
    return [t.requires_grad_() for t in (x, z, r(F_, D) / D ** 0.5, r(D, F_) / F_ ** 0.5, r(3, F_, D) / D ** 0.5, r(3, D, F_) / F_ ** 0.5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_projection_under_autocast(dtype, act):
    """The output is that of the 16-bit layer, its type too; gradients come in the types of the inputs."""
    x, _, w, _, wn, _ = _layer_parts(dtype)
    w, wn = (t.detach().to(dtype if dtype == torch.float64 else torch.float32).requires_grad_() for t in (w, wn))
    with torch.autocast("cpu", dtype=torch.bfloat16):
        a, b = (dense.mixed_linear(x, 6, w, wn, act=act, save8=s) for s in (False, True))
    assert a.dtype == b.dtype and torch.equal(a, b)
    ga, gb = (torch.autograd.grad(y, (x, w, wn), torch.ones_like(y)) for y in (a, b))
    for u, v, t in zip(ga, gb, (x, w, wn)):
        assert v.dtype == t.dtype and (u.double() - v.double()).norm() <= 0.03 * u.double().norm()


@pytest.mark.parametrize("ztype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_ffn_under_autocast(dtype, ztype):
    x, z, w1, w2, wn1, wn2 = _layer_parts(dtype)
    z = z.detach().to(ztype).requires_grad_()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        a = z + dense.mixed_linear(dense.mixed_linear(x, 6, w1, wn1, act="gelu"), 6, w2, wn2)
        b = dense.mixed_ffn(x, z, 6, w1, w2, wn1, wn2, save8=True)
        with torch.no_grad():
            c = dense.mixed_ffn(x, z, 6, w1, w2, wn1, wn2, save8=True)
    assert a.dtype == b.dtype == c.dtype and torch.equal(a, b) and torch.equal(a, c)
    leaves = (x, z, w1, w2, wn1, wn2)
    for u, v, t in zip(*(torch.autograd.grad(y, leaves, torch.ones_like(y)) for y in (a, b)), leaves):
        assert v.dtype == t.dtype and (u.double() - v.double()).norm() <= 0.03 * u.double().norm()


@pytest.mark.parametrize("NS", [0, 3, 9])
def test_gradients_have_their_inputs_shapes(NS):
    """With no token of its own weight, some, and nothing else: an empty weight has an empty gradient."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).requires_grad_()  # noqa: E731
    x, z, w1, w2, wn1, wn2 = r(2, 9, 64), r(2, 9, 64), r(128, 64), r(64, 128), r(NS, 128, 64), r(NS, 64, 128)
    leaves = (x, z, w1, w2, wn1, wn2)
    y = dense.mixed_ffn(x, z, 9 - NS, w1, w2, wn1, wn2, save8=True)
    for t, d in zip(leaves, torch.autograd.grad(y.sum(), leaves)):
        assert d.shape == t.shape and d.dtype == t.dtype and d.isfinite().all()
    for act in (None, "gelu"):
        y = dense.mixed_linear(x, 9 - NS, w1, wn1, act=act, save8=True)
        for t, d in zip((x, w1, wn1), torch.autograd.grad(y.sum(), (x, w1, wn1))):
            assert d.shape == t.shape and d.dtype == t.dtype and d.isfinite().all()
