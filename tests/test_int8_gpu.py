"""8-bit activations and products of 8-bit integers on the GPU: codes bit for bit against the eager form, products and
gradients against 64 bits."""
import math

import pytest
import torch

from primus_dlrm_b200.ops import dense
from primus_dlrm_b200.ops.int8 import Int8Weight, _quantize_ref, int8_error_code, int8_linear, quantize_rows
from primus_dlrm_b200.ops.saved8 import _load_ref, _save_ref, load8, save8

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# GELU of the 16-bit types: Phi is a polynomial within 5.5e-6; of 32 bits: erff within 2 ulp of a value below 1, halved
PHI = {torch.bfloat16: 6e-6, torch.float16: 6e-6, torch.float32: 2.0 ** -23}


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def _spread(shape, dtype, seed=0, top=None):
    g = _gen(seed)
    top = (14 if dtype == torch.float16 else 120) if top is None else top
    e = torch.randint(-top, top + 1, (*shape[:-1], 1), generator=g, device=DEV)
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float64) * torch.exp2(e.double())
    return x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)


def _salt(x):
    """NaN, infinities, zeros and the largest values into some rows."""
    r = x.reshape(-1, x.shape[-1])
    for i, v in enumerate((math.nan, math.inf, -math.inf, torch.finfo(x.dtype).max, 0.0)):
        if r.shape[0] > i + 1:
            r[i + 1] = 0 if v == 0.0 else r[i + 1]
            r[i + 1, (7 * i) % r.shape[1]] = v
    return x


SHAPES = [(1, 1), (1, 8), (3, 31), (5, 32), (7, 33), (2, 3, 64), (9, 104), (257, 256), (4, 5, 1000), (33, 1001), (2, 4096),
          (3, 5003), (1500, 96), (1300, 2056)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_saved_bits(shape, dtype):
    x = _salt(_spread(shape, dtype, seed=sum(shape)))
    s = save8(x)
    codes, scale_bytes = _save_ref(x.reshape(-1, shape[-1]))
    assert torch.equal(s._codes, codes) and torch.equal(s._bytes, scale_bytes)
    for t in TYPES:
        got, ref = load8(s, t), _load_ref(codes, scale_bytes, t).view(shape)
        assert got.dtype == t and torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(ref.float()))
        assert torch.equal(got.isnan(), ref.isnan())
    assert load8(s).dtype == dtype


@pytest.mark.parametrize("dtype", TYPES)
def test_saved_views(dtype):
    big = _spread((6, 40, 200), dtype, seed=1)
    for x in (big[:, 3:, :96], big[:, :, 1:65], big.transpose(0, 1), big.transpose(1, 2), big[1:2, 0], big[:, ::3, ::2],
              big[0, 0].expand(5, 200), big[:0], big[..., :0]):
        s, c = save8(x), save8(x.contiguous())
        assert torch.equal(s.codes, c.codes) and torch.equal(s.exponents, c.exponents) and torch.equal(load8(s), load8(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_row_codes(shape, dtype):
    x = _salt(_spread(shape, dtype, seed=sum(shape) + 1))
    (codes, scale), (rc, rs) = quantize_rows(x), _quantize_ref(x)
    assert torch.equal(codes, rc) and torch.equal(torch.nan_to_num(scale), torch.nan_to_num(rs))
    assert torch.equal(scale.isnan(), rs.isnan())


def _product64(x, w, bias, act, res):
    """(result, size of its 32-bit roundings) in 64 bits, from the codes of the eager form."""
    a, s = _quantize_ref(x)
    lin = torch.einsum("...lk,lnk->...ln" if w.grouped else "...k,nk->...n", a.double(), w.codes.double())
    lin = lin * (s.double()[..., None] * w.scale.double())
    size = lin.abs()
    if bias is not None:
        lin = lin + bias.double()
        size = size + bias.double().abs()
    y = lin * torch.special.ndtr(lin) if act == "gelu" else lin.clamp(min=0) if act == "relu" else lin
    phi = lin.abs() if act == "gelu" else torch.zeros_like(lin)
    if res is not None:
        y, size = y + res.double(), size + res.double().abs()
    return y, size, phi


def _check(y, x, w, bias, act, res):
    ref, size, phi = _product64(x, w, bias, act, res)
    # conversion of the sum, product of scales, product, bias, GELU's product (slope up to 1.13), residual: 8 roundings
    tol = ROUND[y.dtype] * ref.abs() + 8 * 2.0 ** -24 * size + PHI[y.dtype] * phi + 1e-30
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25                               # subnormal steps of 2^-24
    assert y.shape == ref.shape and y.dtype == x.dtype
    nan = ref.isnan()
    assert torch.equal(nan, y.isnan())
    over = ref.abs() >= torch.finfo(y.dtype).max
    bad = ((y.double() - ref).abs() > tol) & ~nan & ~over
    assert not bad.any(), (bad.sum().item(), ((y.double() - ref).abs() / tol)[~nan & ~over].max().item())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N", [
    (1, 1, 1), (1, 16, 8), (1, 1024, 4096), (2, 15, 33), (3, 256, 768), (16, 4096, 1024), (17, 100, 64), (96, 333, 1001),
    (127, 128, 256), (128, 129, 257), (129, 127, 255), (200, 8200, 40), (300, 64, 2000), (1000, 384, 1152), (2500, 96, 520)])
def test_product(rows, K, N, dtype):
    g = _gen(rows + K + N)
    w = Int8Weight.from_float(torch.randn(N, K, generator=g, device=DEV))
    x = _salt(_spread((rows, K), dtype, seed=K, top=3)) if rows > 5 else _spread((rows, K), dtype, seed=K, top=3)
    res = torch.randn(rows, N, generator=g, device=DEV).to(dtype)
    bias = torch.randn(N, generator=g, device=DEV)
    if dtype == torch.float16:
        x = x.clamp(-60, 60)                                 # results stay inside the type
    for b, act, r in ((None, None, None), (bias, "gelu", None), (bias, "relu", res), (None, None, res)):
        _check(int8_linear(x, w, b, act=act, residual=r), x, w, b, act, r)
    assert int8_error_code(DEV) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,K,N", [(1, 3, 40, 24), (5, 1, 64, 64), (70, 16, 256, 130), (1024, 2, 100, 256), (300, 8, 512, 768)])
def test_product_of_a_weight_for_each_position(B, L, K, N, dtype):
    g = _gen(B)
    w = Int8Weight.from_float(torch.randn(L, N, K, generator=g, device=DEV))
    x = torch.randn(B, L, K, generator=g, device=DEV).to(dtype)
    res = torch.randn(B, L, N, generator=g, device=DEV).to(dtype)
    for act, r in ((None, res), ("gelu", None)):
        _check(int8_linear(x, w, None, act=act, residual=r), x, w, None, act, r)


def test_product_of_views():
    g = _gen(3)
    w = Int8Weight.from_float(torch.randn(72, 96, generator=g, device=DEV))
    big = torch.randn(7, 30, 300, generator=g, device=DEV).bfloat16()
    res = torch.randn(7, 30, 100, generator=g, device=DEV).bfloat16()
    bias = torch.randn(72, generator=g, device=DEV).bfloat16()
    for x, r in ((big[:, 2:, 5:101], res[:, 2:, 3:75]), (big[:, ::2, :192:2], res[:, ::2, :72]),
                 (big[:, 0, :96], res[:, 0, 28:]), (big.transpose(0, 1)[..., 8:104], res.transpose(0, 1)[..., :72]),
                 (big[3, 4, :96], res[3, 4, :72]), (big[:1, :1, :96].expand(3, 50, 96), res[:1, :1, :72].expand(3, 50, 72))):
        y = int8_linear(x, w, bias, residual=r)
        assert torch.equal(y, int8_linear(x.contiguous(), w, bias.float(), residual=r.contiguous()))
        _check(y, x, w, bias.float(), None, r)
    wl = Int8Weight.from_float(torch.randn(30, 72, 96, generator=g, device=DEV))
    x = big[:, :, 100:196]
    assert torch.equal(int8_linear(x, wl), int8_linear(x.contiguous(), wl))
    assert int8_linear(big[:0, :, :96], w).shape == (0, 30, 72) and int8_linear(big[:0, :, :96], wl).shape == (0, 30, 72)


def test_weights_as_given():
    g = _gen(4)
    codes = torch.randint(-128, 128, (50, 48), generator=g, device=DEV, dtype=torch.int8)     # -128 too
    scale = torch.rand(50, generator=g, device=DEV)
    x = torch.randn(9, 48, generator=g, device=DEV)
    _check(int8_linear(x, Int8Weight.from_tensors(codes, scale)), x, Int8Weight.from_tensors(codes, scale), None, None, None)
    w2 = Int8Weight.from_tensors(codes[:, 3:40], scale)
    _check(int8_linear(x[:, 3:40], w2), x[:, 3:40], w2, None, None, None)
    # the longest row: sums of 131072 products of 127 * 128
    K = 131072
    w = Int8Weight.from_tensors(torch.full((3, K), -128, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV))
    y = int8_linear(torch.ones(2, K, device=DEV), w)
    assert (y.double() + 128 * K).abs().max() <= 4 * 2.0 ** -24 * 128 * K


def test_product_refusals():
    w = Int8Weight.from_float(torch.randn(5, 20, device=DEV))
    x = torch.randn(4, 20, device=DEV)
    from torch.autograd import forward_ad
    for bad in (lambda: int8_linear(x[:, :19], w), lambda: int8_linear(x.double(), w),
                lambda: int8_linear(x, w, torch.zeros(4, device=DEV)), lambda: int8_linear(x, w, torch.zeros(5)),
                lambda: int8_linear(x, w, residual=torch.zeros(4, 6, device=DEV)),
                lambda: int8_linear(x, w, residual=torch.zeros(4, 5, device=DEV).half()),
                lambda: int8_linear(x, w, residual=torch.zeros(4, 5)),
                lambda: int8_linear(x, Int8Weight.from_float(torch.randn(3, 5, 20, device=DEV))),
                lambda: int8_linear(x, Int8Weight.from_float(torch.randn(5, 20)))):
        with pytest.raises(RuntimeError):
            bad()
    y = int8_linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        y.sum().backward()
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        int8_linear(forward_ad.make_dual(x, x), w)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        save8(forward_ad.make_dual(x, x))
    assert not save8(x.clone().requires_grad_())._codes.requires_grad


def test_product_on_another_stream_in_a_graph_and_twice():
    g = _gen(6)
    w = Int8Weight.from_float(torch.randn(130, 96, generator=g, device=DEV))
    x = torch.randn(40, 96, generator=g, device=DEV).bfloat16()
    ref = int8_linear(x, w, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [int8_linear(x, w, act="gelu") for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, ref) for t in got)
    buf = x.clone()
    graphs, outs = [], []
    for _ in range(2):                                       # two graphs of the same call
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(int8_linear(buf, w, act="gelu"))
        graphs.append(graph)
    x2 = torch.randn(40, 96, generator=g, device=DEV).bfloat16()
    buf.copy_(x2)
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, int8_linear(x2, w, act="gelu")) for t in outs)
    with torch.inference_mode():
        wi = Int8Weight.from_float(w.dequantize())
    assert torch.equal(int8_linear(x, wi, act="gelu"), int8_linear(x, Int8Weight.from_float(w.dequantize()), act="gelu"))


# ---------------------------------------------------------------- training layers
def _parts(B, T, D, F, NS, seed=0, wdtype=torch.float32):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x = (r(B, T, D) * torch.exp(0.5 * r(1, 1, D))).bfloat16()
    return [x, r(B, T, D).bfloat16(), (r(F, D) / D ** 0.5).to(wdtype), (r(D, F) / F ** 0.5).to(wdtype),
            (r(NS, F, D) / D ** 0.5).to(wdtype), (r(NS, D, F) / F ** 0.5).to(wdtype)]


def _mixed64(x, n_s, w, wn):
    return torch.cat([x[:, :n_s] @ w.t(), torch.einsum("btk,tnk->btn", x[:, n_s:], wn)], 1)


def _grads64(dy, x, n_s):
    return (torch.einsum("btn,btk->nk", dy[:, :n_s], x[:, :n_s]), torch.einsum("btn,btk->tnk", dy[:, n_s:], x[:, n_s:]))


def _within(got, ref, tol, what):
    assert got.shape == ref.shape, what
    bad = (got.double() - ref).abs() / (tol + 1e-30)
    assert not got.numel() or bad.max() <= 1, (what, bad.max().item())


def _kept(f):
    """(f(), the 8-bit tensors that it keeps for its backward pass, in order)."""
    kept = []

    def keep(t):
        if t.dtype in (torch.int8, torch.uint8):
            kept.append(t.detach())
        return t

    with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
        return f(), kept


SIZES = [(1, 1, 64, 64, 0), (2, 9, 64, 128, 3), (3, 130, 128, 320, 0), (5, 70, 256, 1024, 16), (1, 300, 192, 768, 8),
         (3, 500, 256, 512, 8), (2, 700, 512, 256, 40), (20, 515, 64, 320, 3), (9, 2300, 128, 192, 0)]


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,F,NS", SIZES)
def test_ffn(B, T, D, F, NS, wdtype):
    parts = [t.requires_grad_() for t in _parts(B, T, D, F, NS, wdtype=wdtype)]
    n_s = T - NS
    out, (xc, xe, pc, pe) = _kept(lambda: dense.mixed_ffn(parts[0], parts[1], n_s, *parts[2:], save8=True))
    assert torch.equal(out, dense.mixed_ffn(parts[0], parts[1], n_s, *parts[2:]))
    with torch.no_grad():
        assert torch.equal(out, dense.mixed_ffn(parts[0], parts[1], n_s, *parts[2:], save8=True))
    assert xc.dtype == pc.dtype == torch.int8 and torch.equal(xc, save8(parts[0])._codes)
    d = [t.detach().bfloat16().double() for t in parts]
    p = _mixed64(d[0], n_s, d[2], d[4]).view(B * T, F)
    # a saved pre-activation is the integer nearest to the 32-bit sum: D products, each within 2^-22 of the largest partial sum
    step = torch.exp2(pe.t().double() - 127).repeat_interleave(32, 1)
    slack = D * 2.0 ** -22 * _mixed64(d[0].abs(), n_s, d[2].abs(), d[4].abs()).view(B * T, F)
    ps, xs = _load_ref(pc, pe, torch.float32).double(), _load_ref(xc, xe, torch.float32).double().view(B, T, D)
    _within(ps, p, 0.5 * step + slack, "pre-activation")
    amax = p.abs().view(B * T, -1, 32).amax(-1)
    assert (amax <= 127 * step[:, ::32] + slack.view(B * T, -1, 32).amax(-1)).all()
    assert (amax >= 63.5 * step[:, ::32] - slack.view(B * T, -1, 32).amax(-1)).all()
    ps = ps.view(B, T, F)

    g = _gen(9)
    dy = torch.randn(B, T, D, generator=g, device=DEV).bfloat16()
    grads = torch.autograd.grad(out, parts, dy)
    dy64 = dy.double()
    dh = _mixed64(dy64, n_s, d[3].t(), d[5].transpose(1, 2))
    dh_size = _mixed64(dy64.abs(), n_s, d[3].abs().t(), d[5].abs().transpose(1, 2))
    slope = torch.special.ndtr(ps) + ps * torch.exp(-ps * ps / 2) / math.sqrt(2 * math.pi)
    dp, h = dh * slope, ps * torch.special.ndtr(ps)
    # rounded to bf16 on the way: dp and h; the polynomial Phi is 5.5e-6 off (slope and GELU / p alike), sums of 32 bits
    e_dp = 2.0 ** -8 * dp.abs() + 1e-5 * dh.abs() + D * 2.0 ** -22 * dh_size * 1.13
    e_h = 2.0 ** -8 * h.abs() + 6e-6 * ps.abs()
    want = [_mixed64(dp, n_s, d[2].t(), d[4].transpose(1, 2)), dy64, None, None, None, None]
    size = [_mixed64(e_dp + F * 2.0 ** -22 * dp.abs(), n_s, d[2].abs().t(), d[4].abs().transpose(1, 2)), torch.zeros_like(dy64)]
    want[2], want[4] = _grads64(dp, xs, n_s)
    want[3], want[5] = _grads64(dy64, h, n_s)
    n = B * T * 2.0 ** -22
    s2, s4 = _grads64(e_dp + n * dp.abs(), xs.abs(), n_s)
    s3, s5 = _grads64(dy64.abs(), e_h + n * h.abs(), n_s)
    # the shared weight's gradient is that of all rows less the NS rows' parts
    for s, parts_of in ((s2, s4), (s3, s5)):
        s += 2 * parts_of.sum(0) + 2.0 ** -22 * parts_of.shape[0] * s
    size += [s2, s3, s4, s5]
    for i, (got, ref, tol) in enumerate(zip(grads, want, size)):
        assert got.dtype == parts[i].dtype
        _within(got, ref, tol + 2 * ROUND[got.dtype] * (ref.abs() + tol), ("x", "z", "w1", "w2", "wn1", "wn2")[i])


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("B,T,D,F,NS", SIZES)
def test_projection(B, T, D, F, NS, act):
    x, _, w, _, wn, _ = (t.requires_grad_() for t in _parts(B, T, D, F, NS, seed=1))
    n_s = T - NS
    y, kept = _kept(lambda: dense.mixed_linear(x, n_s, w, wn, act=act, save8=True))
    assert torch.equal(y, dense.mixed_linear(x, n_s, w, wn, act=act)) and len(kept) == (4 if act else 2)
    dy = torch.randn(y.shape, generator=_gen(2), device=DEV).bfloat16()
    grads = torch.autograd.grad(y, (x, w, wn), dy)
    xs = load8(save8(x)).double()
    dp, e_dp = dy.double(), 0 * dy.double()
    if act == "gelu":
        ps = _load_ref(*kept[2:], torch.float32).double().view(B, T, F)
        slope = torch.special.ndtr(ps) + ps * torch.exp(-ps * ps / 2) / math.sqrt(2 * math.pi)
        dp = dp * slope
        e_dp = 2.0 ** -8 * dp.abs() + 1e-5 * dy.double().abs()
    wb, wnb = w.detach().bfloat16().double(), wn.detach().bfloat16().double()
    dx = _mixed64(dp, n_s, wb.t(), wnb.transpose(1, 2))
    sx = _mixed64(e_dp + F * 2.0 ** -22 * dp.abs(), n_s, wb.abs().t(), wnb.abs().transpose(1, 2))
    _within(grads[0], dx, sx + 2.0 ** -8 * (dx.abs() + sx), "x")
    (dw, dwn), n = _grads64(dp, xs, n_s), B * T * 2.0 ** -22
    sw, swn = _grads64(e_dp + n * dp.abs(), xs.abs(), n_s)
    sw = sw + 2 * swn.sum(0) + n * swn.abs().sum(0) + 2.0 ** -22 * _grads64(dp.abs(), xs.abs(), n_s)[1].sum(0)
    _within(grads[1], dw, sw + 2.0 ** -23 * dw.abs(), "w")
    _within(grads[2], dwn, swn + 2.0 ** -23 * dwn.abs(), "wn")


def test_layer_refusals():
    from torch.autograd import forward_ad
    x, z, w1, w2, wn1, wn2 = (t.requires_grad_() for t in _parts(2, 7, 64, 128, 3))
    n = lambda t: torch.zeros_like(t)[1:]  # noqa: E731
    for bad in (lambda: dense.mixed_linear(x, 4, w1, n(wn1), save8=True), lambda: dense.mixed_linear(x, 3, w1, wn1, save8=True),
                lambda: dense.mixed_linear(x, 8, w1, wn1[:0], save8=True),
                lambda: dense.mixed_ffn(x, z[:, :6], 4, w1, w2, wn1, wn2, save8=True),
                lambda: dense.mixed_ffn(x, z, 4, w1, w2, wn1, n(wn2), save8=True),
                lambda: dense.mixed_ffn(x, z, 4, w1, w2[:, :64], wn1, wn2[:, :, :64], save8=True),
                lambda: dense.mixed_ffn(x, z, 4, w1, w2.cpu(), wn1, wn2, save8=True)):
        with pytest.raises(RuntimeError):
            bad()
    y = dense.mixed_linear(x, 4, w1, wn1, save8=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        dense.mixed_linear(forward_ad.make_dual(x.detach(), x.detach()), 4, w1, wn1, save8=True)
    # gradients of some inputs only
    frozen = [t.detach() for t in (w1, w2, wn1, wn2)]
    out = dense.mixed_ffn(x, z, 4, *frozen, save8=True)
    full = dense.mixed_ffn(x, z, 4, w1, w2, wn1, wn2, save8=True)
    (dx,), (dx2, dw) = (torch.autograd.grad(o.sum(), i) for o, i in ((out, (x,)), (full, (x, w1))))
    assert torch.equal(dx, dx2) and dw.shape == w1.shape
    empty = dense.mixed_ffn(x[:0], z[:0], 4, w1, w2, wn1, wn2, save8=True)
    assert empty.shape == (0, 7, 64)


def test_layers_that_the_gemm_cannot_run():
    """Widths that are no multiple of 64, and fp32: through PyTorch, the same formulas."""
    for B, T, D, F, NS, dt in ((2, 7, 40, 72, 3, torch.bfloat16), (2, 7, 64, 128, 3, torch.float32)):
        x, z, w1, w2, wn1, wn2 = (t.to(dt).requires_grad_() for t in _parts(B, T, D, F, NS))
        a = dense.mixed_ffn(x, z, T - NS, w1, w2, wn1, wn2, save8=True)
        ref = dense._ffn_forward(x, z, w1, w2, wn1, wn2, T - NS)
        assert a.shape == z.shape and (a - ref).abs().max() <= 4 * torch.finfo(dt).eps * ref.abs().max()
        ga = torch.autograd.grad(a.sum(), (x, z, w1, w2, wn1, wn2))
        gr = torch.autograd.grad(ref.sum(), (x, z, w1, w2, wn1, wn2))
        for u, v in zip(ga, gr):
            assert u.dtype == v.dtype and (u.double() - v.double()).norm() <= 0.03 * v.double().norm()


def test_a_pre_activation_without_numbers():
    """Rows that overflow or hold NaN reach their own gradients only."""
    parts = _parts(1, 40, 64, 128, 0)
    parts[0][0, 3, 5] = math.nan
    parts[0][0, 20, 7] = 3e38                                # finite: its products overflow in 32 bits
    x, z, w1, w2, wn1, wn2 = (t.requires_grad_() for t in parts)
    out = dense.mixed_ffn(x, z, 40, w1, w2, wn1, wn2, save8=True)
    dx, dz = torch.autograd.grad(out, (x, z), torch.ones_like(out), retain_graph=True)
    assert dx[0, 3].isnan().all() and torch.equal(dz, torch.ones_like(dz))
    rest = [i for i in range(40) if i not in (3, 20)]
    assert dx[0, rest].isfinite().all()
    clean = [t.detach().clone() for t in parts]
    clean[0][0, 3], clean[0][0, 20] = 0, 0
    clean = [t.requires_grad_() for t in clean]
    out2 = dense.mixed_ffn(clean[0], clean[1], 40, *clean[2:], save8=True)
    (dx2,) = torch.autograd.grad(out2, clean[:1], torch.ones_like(out2))
    assert torch.equal(out[0, rest], out2[0, rest]) and torch.equal(dx[0, rest], dx2[0, rest])


def test_a_captured_training_step():
    g = _gen(8)
    parts = [t.requires_grad_() for t in _parts(4, 50, 128, 256, 4)]
    dy = torch.randn(4, 50, 128, generator=g, device=DEV).bfloat16()

    def step():
        h = dense.mixed_linear(parts[0], 46, parts[2][:128], parts[4][:, :128], save8=True)
        out = dense.mixed_ffn(h, parts[1], 46, *parts[2:], save8=True)
        return (out, *torch.autograd.grad(out, parts, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    graph.replay()
    ref = step()
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    for a, b in zip(got[2:], ref[2:]):                       # weight gradients add up in no fixed order
        assert (a.double() - b.double()).abs().max() <= 1e-5 * b.abs().max() + 1e-6


def test_every_row_has_its_own_weight():
    """n_s = 0: the shared weights get gradients of zeros, nothing else changes."""
    parts = [t.requires_grad_() for t in _parts(3, 5, 64, 128, 5, seed=3)]
    out = dense.mixed_ffn(parts[0], parts[1], 0, *parts[2:], save8=True)
    assert torch.equal(out, dense.mixed_ffn(parts[0], parts[1], 0, *parts[2:]))
    g = torch.autograd.grad(out, parts, torch.ones_like(out))
    assert g[2].eq(0).all() and g[3].eq(0).all() and g[4].ne(0).any() and g[5].ne(0).any()
    y = dense.mixed_linear(parts[0], 0, parts[2], parts[4], save8=True)
    dx, dw, dwn = torch.autograd.grad(y, (parts[0], parts[2], parts[4]), torch.ones_like(y))
    assert dw.eq(0).all() and dwn.ne(0).any() and dx.isfinite().all()


@pytest.mark.parametrize("B,T,NS", [(40, 1, 0), (40, 1, 1), (4, 9, 3), (1, 9, 3)])
def test_layers_of_views(B, T, NS):
    """Any stride over an axis of length 1, samples in two orders, an incoming gradient off 16 bytes: as of copies.

    One block of 64 rows covers each sum over rows, so no order of additions changes a weight's gradient."""
    def layers(x, z, dy):
        parts = [x.detach().requires_grad_(), z.detach().requires_grad_(),
                 *(t.requires_grad_() for t in _parts(B, T, 64, 128, NS, seed=8)[2:])]
        out = dense.mixed_ffn(parts[0], parts[1], T - NS, *parts[2:], save8=True)
        y = dense.mixed_linear(parts[0], T - NS, parts[2][:64], parts[4][:, :64], act="gelu", save8=True)
        return [out.detach(), y.detach(), *torch.autograd.grad((out, y), parts, (dy, dy))]

    x, z, dy = (t.clone() for t in (*_parts(B, T, 64, 128, NS, seed=8)[:2], _parts(B, T, 64, 128, NS, seed=9)[0]))
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, z)]
    if T == 1 and B > 1:
        turned = [t.as_strided(t.shape, (64, 64 * B, 1)) for t in (x, z)]
        assert all(t.is_contiguous() and t.stride(1) == 64 * B for t in turned)
    off = torch.cat([dy.new_zeros(1), dy.flatten()])[1:].view(dy.shape)
    assert off.data_ptr() % 16
    for a, b in zip(layers(*turned, off), layers(x, z, dy)):
        assert torch.equal(a, b)


def test_calls_at_once():
    """Two threads, each on its own stream, with rows for every form of the product."""
    import threading
    g = _gen(11)
    w = Int8Weight.from_float(torch.randn(300, 640, generator=g, device=DEV))
    xs = [torch.randn(m, 640, generator=g, device=DEV).bfloat16() for m in (1, 16, 90, 3000)]
    want = [int8_linear(x, w, act="gelu") for x in xs]
    saved = [load8(save8(x)) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for x, y, v in zip(xs, want, saved):
                    if not (torch.equal(int8_linear(x, w, act="gelu"), y) and torch.equal(load8(save8(x)), v)):
                        bad.append(x.shape)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_first_call_inside_a_capture():
    """Kernels that a process has not launched yet, captured at once, forward and backward; then a captured backward pass
    while an eager graph of the same leaves lives, which PyTorch's engine refuses (of its own operations alike) with an
    error that the process outlives. In a process of its own."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys
sys.path.insert(0, %r)
import torch
from primus_dlrm_b200.ops import dense
from primus_dlrm_b200.ops.int8 import Int8Weight, int8_linear
x = torch.randn(40, 4096, device="cuda").bfloat16()
w = Int8Weight.from_float(torch.randn(64, 4096, device="cuda"))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = int8_linear(x, w)
graph.replay()
torch.cuda.synchronize()
print("FORWARD", torch.equal(y, int8_linear(x, w)))

r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
p = [t.requires_grad_() for t in (r(2, 90, 64), r(2, 90, 64), r(128, 64), r(64, 128), r(3, 128, 64), r(3, 64, 128))]
dy = r(2, 90, 64)
step = lambda: torch.autograd.grad(dense.mixed_ffn(p[0], p[1], 87, *p[2:], save8=True), p, dy)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
near = lambda a, b: all(bool((u.double() - v.double()).abs().max() <= 2.0 ** -7 * v.abs().max()) for u, v in zip(a, b))
want = step()
print("BACKWARD", near(got, want))
alive = dense.mixed_ffn(p[0], p[1], 87, *p[2:], save8=True)
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        got = step()
    print("CAPTURED")
except RuntimeError as e:
    print("REFUSED", str(e)[:200])
print("AFTER", near(torch.autograd.grad(alive, p, dy), want))
print("END")
""" % str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert all(m in r.stdout for m in ("FORWARD True", "BACKWARD True", "AFTER True", "END")), r.stdout + r.stderr[-1500:]
