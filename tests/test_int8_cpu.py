"""8-bit activations and products of 8-bit integers in their eager form: the definitions in 64 bits, refusals, gradients
against differences."""
import math

import pytest
import torch

from primus_dlrm_b200.ops import dense
from primus_dlrm_b200.ops.int8 import Int8Weight, int8_linear, quantize_rows
from primus_dlrm_b200.ops.saved8 import load8, save8

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _spread(shape, dtype, seed=0):
    """Values over the type's whole range: normals times powers of two of each row."""
    g = _gen(seed)
    top = 14 if dtype == torch.float16 else 120
    e = torch.randint(-top, top, (*shape[:-1], 1), generator=g)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * torch.exp2(e.double())).clamp(
        -torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (33,), (5, 32), (3, 4, 70), (2, 0), (0, 64)])
def test_saved_values_are_within_half_a_step(shape, dtype):
    x = _spread(shape, dtype, seed=sum(shape))
    s = save8(x)
    y = load8(s)
    assert y.dtype == dtype and y.shape == x.shape and s.codes.shape == x.shape
    assert s.exponents.shape == (*shape[:-1], -(-shape[-1] // 32)) and s.nbytes == x.numel() + s.exponents.numel()
    if not x.numel():
        return
    pad = -shape[-1] % 32
    amax = torch.nn.functional.pad(x.double().abs(), (0, pad)).unflatten(-1, (-1, 32)).amax(-1)
    step = torch.exp2(s.exponents.double() - 127)
    assert (amax <= 127 * step).all() and ((amax > 63.5 * step) | (s.exponents == 1)).all()
    # half a step; a whole one where codes are held to 63, at the type's largest values
    step = step.repeat_interleave(32, -1)[..., :shape[-1]]
    off = (load8(s, torch.float32).double() - x.double()).abs()
    top = torch.finfo(dtype).max
    assert (off <= torch.where(x.double().abs() > 0.99 * top, 1.0, 0.5) * step).all()
    assert y.isfinite().all()
    if dtype != torch.float16:                               # 7 significant bits: exact
        assert torch.equal(y.float(), load8(s, torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_saved_edges(dtype):
    top = torch.finfo(dtype).max
    x = torch.zeros(9, 40, dtype=dtype)
    x[1, 3], x[2, 35], x[3, 0] = math.nan, math.inf, -math.inf
    x[4], x[5], x[6] = top, -top, torch.finfo(dtype).smallest_normal
    x[7, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], dtype=dtype)       # scale 1: ties go to even
    x[8, 0] = 127.5                                                      # past 127: scale 2
    s = save8(x)
    y = load8(s)
    assert s.exponents[0].tolist() == [1, 1] and y[0].eq(0).all()
    assert s.exponents[1].tolist() == [255, 1] and y[1, :32].isnan().all() and y[1, 32:].eq(0).all()
    assert s.exponents[2].tolist() == [1, 255] and s.exponents[3].tolist() == [255, 1]
    assert s.codes[1:4].abs().max() == 0
    assert y[4].isfinite().all() and (y[4].double() >= 63 / 64 * top).all() and torch.equal(y[4], -y[5])
    assert s.codes[7, :4].tolist() == [127, 0, 2, -2] and s.exponents[7, 0] == 127 and s.exponents[8, 0] == 128


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_to_codes(dtype):
    x = _spread((7, 5, 50), dtype, seed=3)
    x[0, 0] = 0
    x[0, 1, 7], x[0, 2, 8] = math.nan, math.inf
    codes, scale = quantize_rows(x)
    assert codes.dtype == torch.int8 and scale.shape == x.shape[:-1]
    assert scale[0, 1:3].isnan().all() and codes[0, :3].eq(0).all() and scale[0, 0] == 2.0 ** -126
    fine = scale.isfinite()
    off = (codes.double() * scale.double()[..., None] - x.double()).abs()
    # half a step and the 32-bit roundings of scale, reciprocal and product: 127 * 3 * 2^-24 of a step
    assert (off <= (0.5 + 127 * 3 * 2.0 ** -24) * scale.double()[..., None])[fine].all()
    assert (codes[fine].abs().amax(-1)[x[fine].abs().amax(-1) > 2.0 ** -118] == 127).all()


@pytest.mark.parametrize("act", [None, "gelu", "relu"])
@pytest.mark.parametrize("grouped", [False, True])
def test_product_is_the_integers(grouped, act):
    g = _gen(1)
    w = torch.randn(*((3,) if grouped else ()), 10, 37, generator=g)
    x = torch.randn(4, 3, 37, generator=g)
    res, bias = torch.randn(4, 3, 10, generator=g), torch.randn(10, generator=g)
    iw = Int8Weight.from_float(w)
    assert iw.codes.shape == w.shape and iw.scale.shape == w.shape[:-1] and (iw.in_features, iw.out_features) == (37, 10)
    assert ((iw.dequantize() - w).abs() <= 0.501 * iw.scale[..., None]).all()
    y = int8_linear(x, iw, bias, act=act, residual=res)
    a, s = quantize_rows(x)
    lin = torch.einsum("btk,tnk->btn" if grouped else "btk,nk->btn", a.double(), iw.codes.double())
    lin = lin * s.double()[..., None] * iw.scale.double() + bias.double()
    ref = {None: lambda v: v, "gelu": lambda v: v * torch.special.ndtr(v), "relu": torch.relu}[act](lin) + res.double()
    assert (y.double() - ref).abs().max() <= 8 * 2.0 ** -24 * (lin.abs().max() + res.abs().max())


def test_a_row_without_numbers_is_nan_and_alone():
    iw = Int8Weight.from_float(torch.randn(5, 20, generator=_gen()))
    x = torch.randn(4, 20, generator=_gen(1))
    y0 = int8_linear(x, iw)
    x[1, 3], x[2, 0] = math.inf, math.nan
    y = int8_linear(x, iw)
    assert y[1:3].isnan().all() and torch.equal(y[0], y0[0]) and torch.equal(y[3], y0[3])
    assert int8_linear(torch.zeros(0, 20), iw).shape == (0, 5)
    assert int8_linear(torch.zeros(20), iw).shape == (5,)


def test_refusals():
    w = torch.randn(5, 20)
    iw = Int8Weight.from_float(w)
    x = torch.randn(4, 20)
    for bad in (lambda: int8_linear(x, iw, act="tanh"), lambda: int8_linear(x[:, :19], iw),
                lambda: int8_linear(x.double(), iw), lambda: int8_linear(x, iw, torch.zeros(4)),
                lambda: int8_linear(x, iw, residual=torch.zeros(4, 6)),
                lambda: int8_linear(x, iw, residual=torch.zeros(4, 5).half()),
                lambda: Int8Weight.from_tensors(iw.codes.float(), iw.scale),
                lambda: Int8Weight.from_tensors(iw.codes, iw.scale[:4]),
                lambda: Int8Weight.from_tensors(iw.codes, iw.scale.double()),
                lambda: Int8Weight.from_tensors(iw.codes[:0], iw.scale[:0]),
                lambda: Int8Weight.from_float(torch.randn(1, 131073)),
                lambda: Int8Weight.from_float(w.double()), lambda: quantize_rows(x.long()),
                lambda: save8(x.double()), lambda: save8(torch.tensor(1.0)), lambda: load8(save8(x), torch.float64),
                lambda: int8_linear(x, Int8Weight.from_float(torch.randn(3, 5, 20)))):
        with pytest.raises(ValueError):
            bad()
    y = int8_linear(x.requires_grad_(), iw)
    with pytest.raises(RuntimeError, match="no gradient"):
        y.sum().backward()
    assert not save8(x).codes.requires_grad and not load8(save8(x)).requires_grad


def _ffn_parts(D=64, F=128, NS=3, seed=0, dtype=torch.float32):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return [r(2, 9, D), r(2, 9, D), r(F, D) / D ** 0.5, r(D, F) / F ** 0.5, r(NS, F, D) / D ** 0.5, r(NS, D, F) / F ** 0.5]


def _mixed64(x, ns, w, wn):
    return torch.cat([x[:, :ns] @ w.t(), torch.einsum("btk,tnk->btn", x[:, ns:], wn)], 1)


@pytest.mark.parametrize("NS", [0, 3])
def test_ffn_gradients_follow_the_formula_and_differences(NS):
    """Against the formula on the saved values (32-bit rounding), and against differences of the output along a direction,
    which the 8-bit values bend by at most max |gelu''| = 0.8 times half a step of each pre-activation, and by half a step
    of x in the weight gradient."""
    parts = [t.requires_grad_() for t in _ffn_parts(NS=NS)]
    x, z, w1, w2, wn1, wn2 = parts
    n_s = 9 - NS
    out = dense.mixed_ffn(x, z, n_s, w1, w2, wn1, wn2, save8=True)
    d = [t.detach().double() for t in parts]
    p = _mixed64(d[0], n_s, d[2], d[4])
    ref = d[1] + _mixed64(p * torch.special.ndtr(p), n_s, d[3], d[5])
    assert (out.double() - ref).abs().max() <= 1e-5
    dy = torch.randn(out.shape, generator=_gen(5))
    grads = torch.autograd.grad(out, parts, dy)
    xs, ps = (load8(save8(t)).double() for t in (x.detach(), p.float()))
    phi = torch.exp(-ps * ps / 2) / math.sqrt(2 * math.pi)
    dp = _mixed64(dy.double(), n_s, d[3].t(), d[5].transpose(1, 2)) * (torch.special.ndtr(ps) + ps * phi)
    h = ps * torch.special.ndtr(ps)
    S = slice(0, n_s)
    want = [_mixed64(dp, n_s, d[2].t(), d[4].transpose(1, 2)), dy.double(), torch.einsum("btn,btk->nk", dp[:, S], xs[:, S]),
            torch.einsum("btn,btk->nk", dy[:, S].double(), h[:, S]), torch.einsum("btn,btk->tnk", dp[:, n_s:], xs[:, n_s:]),
            torch.einsum("btn,btk->tnk", dy[:, n_s:].double(), h[:, n_s:])]
    for got, ref in zip(grads, want):
        assert got.shape == ref.shape and (got.double() - ref).abs().max() <= 1e-4 if ref.numel() else True

    def value(q):
        p = _mixed64(q[0], n_s, q[2], q[4])
        y = q[1] + _mixed64(p * torch.special.ndtr(p), n_s, q[3], q[5])
        return (y * dy.double()).sum()

    step = lambda t: torch.exp2(save8(t).exponents.double() - 127).repeat_interleave(32, -1)  # noqa: E731
    dh = _mixed64(dy.double(), n_s, d[3].t(), d[5].transpose(1, 2)).abs()
    for i in range(6):
        if not d[i].numel():
            continue
        v = torch.randn(d[i].shape, generator=_gen(10 + i), dtype=torch.float64)
        e = 1e-5
        up, dn = list(d), list(d)
        up[i], dn[i] = d[i] + e * v, d[i] - e * v
        diff = (value(up) - value(dn)) / (2 * e)
        q = list(d)
        q[i] = v
        zero = torch.zeros_like
        if i in (0, 2, 4):            # through the pre-activation: its own change, times gelu'' and half a step
            pv = _mixed64(v, n_s, d[2], d[4]) if i == 0 else _mixed64(
                d[0], n_s, v if i == 2 else zero(d[2]), v if i == 4 else zero(d[4]))
            bend = (dh * 0.8 * step(p.float()) / 2 * pv.abs()).sum()
            if i != 0:                # and x in place of its 8-bit values
                pe = _mixed64(step(d[0].float()) / 2, n_s, *(t.abs() for t in (
                    v if i == 2 else zero(d[2]), v if i == 4 else zero(d[4]))))
                bend = bend + (dh * 1.13 * pe).sum()
        elif i in (3, 5):             # h by half a step of p, slope at most 1.13
            he = _mixed64(1.13 * step(p.float()) / 2, n_s, *(t.abs() for t in (
                v if i == 3 else zero(d[3]), v if i == 5 else zero(d[5]))))
            bend = (dy.double().abs() * he).sum()
        else:
            bend = 0.0
        assert abs((grads[i].double() * v).sum() - diff) <= bend + 1e-3 * (1 + abs(diff))


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_projection_keeps_its_output_and_input_gradient(dtype, act):
    x, _, w, _, wn, _ = (t.requires_grad_() for t in _ffn_parts(dtype=dtype))
    a = dense.mixed_linear(x, 6, w, wn, act=act)
    b = dense.mixed_linear(x, 6, w, wn, act=act, save8=True)
    assert torch.equal(a, b)
    dy = torch.randn(a.shape, generator=_gen(2)).to(dtype)
    ga, gb = (torch.autograd.grad(t, (x, w, wn), dy) for t in (a, b))
    if act is None:
        eps = torch.finfo(dtype).eps
        assert (ga[0] - gb[0]).abs().max() <= 4 * eps * ga[0].abs().max()
        step = torch.exp2(save8(x).exponents.double() - 127).repeat_interleave(32, -1)
        bound = torch.einsum("btn,btk->nk", dy[:, :6].double().abs(), step[:, :6] / 2)
        assert ((ga[1].double() - gb[1].double()).abs() <= bound + 16 * eps * ga[1].abs().max()).all()
    for u, v in zip(ga, gb):
        assert u.dtype == v.dtype and u.shape == v.shape
        assert (u.double() - v.double()).norm() <= 0.03 * u.double().norm()


def test_nothing_is_kept_without_gradients():
    parts = _ffn_parts()
    y = dense.mixed_ffn(parts[0], parts[1], 6, *parts[2:], save8=True)
    assert y.grad_fn is None
    parts[0].requires_grad_()
    with torch.no_grad():
        assert torch.equal(dense.mixed_ffn(parts[0], parts[1], 6, *parts[2:], save8=True), y)
    out = dense.mixed_ffn(parts[0], parts[1], 6, *parts[2:], save8=True)
    (g,) = torch.autograd.grad(out.sum(), parts[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
