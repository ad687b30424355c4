"""Query/key norm with rotation against its formulas in 64 bits, forward and
backward, at the sizes, strides and types where it can go wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6
# one rounding of the result to the type (2^-8 relative for the 8 significant bits of bf16, 2^-11 for fp16's 11 and
# 2^-24 for fp32's 24) on top of 32-bit arithmetic: at most about 20 roundings of 2^-24 each in the chain norm, weight,
# rotation, mean. The latter are measured against the row's largest value, since the rotation and the mean mix a row,
# and in dx, a difference, against the largest value of its two terms.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
CHAIN = 24 * 2.0 ** -24


def _ref(x, w, ang, interleaved, dy=None):
    """y, dx, dw of one of the two inputs in 64 bits; ang [B or 1, T, rot]."""
    x = x.detach().double().requires_grad_(True)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    w = w.requires_grad_(True)
    h = ang.shape[-1] // 2
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    c, s = ang[:, :, None, :h].double(), ang[:, :, None, h:].double()
    i0 = torch.arange(0, 2 * h, 2) if interleaved else torch.arange(h)
    i1 = i0 + 1 if interleaved else i0 + h
    y2 = y.clone()
    y2[..., i0] = y[..., i0] * c - y[..., i1] * s
    y2[..., i1] = y[..., i0] * s + y[..., i1] * c
    if dy is None:
        return y2.detach(), None, None, None
    (g,) = torch.autograd.grad(y2, y, dy.double(), retain_graph=True)
    y2.backward(dy.double())
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS).detach()
    gw, xh = g * w.detach(), x.detach() * r
    terms = r * (gw.abs() + xh.abs() * (gw * xh).mean(-1, keepdim=True).abs())
    return y2.detach(), x.grad, w.grad, terms.amax(-1, keepdim=True)


def _close(got, ref, dtype, what, size=None):
    top = ref.abs().amax(-1, keepdim=True)
    tol = ROUND[dtype] * top + CHAIN * (top if size is None else size) + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -24                       # below 2^-14 fp16 steps are 2^-24
    assert got.dtype == dtype and got.shape == ref.shape
    worst = ((got.double() - ref).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, (what, worst)


def _inputs(B, T, Q, H, K, d, dtype, seed=0, strided=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(B, T, (H + 2 * K) * d, generator=g, device=DEV).to(dtype)
    q, k = qkv[:, T - Q:, :H * d].unflatten(-1, (H, d)), qkv[:, :, H * d:(H + K) * d].unflatten(-1, (K, d))
    if not strided:
        q, k = q.contiguous(), k.contiguous()
    wq, wk = (1 + 0.3 * torch.randn(d, generator=g, device=DEV) for _ in range(2))
    dq, dk = (torch.randn(t.shape, generator=g, device=DEV).to(dtype) for t in (q, k))
    return q, k, wq, wk, dq, dk


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,Q,H,K,d,rot", [
    (2, 7, 7, 4, 4, 32, 32), (1, 1, 1, 1, 1, 16, 16), (3, 33, 5, 6, 2, 64, 32), (2, 9, 9, 8, 1, 128, 128),
    (2, 5, 3, 3, 3, 48, 16), (1, 11, 11, 2, 2, 256, 256), (2, 6, 4, 2, 1, 34, 10), (1, 3, 2, 5, 5, 2, 2),
    (1, 4, 4, 1, 1, 254, 0), (5, 301, 299, 2, 2, 96, 96)])
def test_forward_and_backward(B, T, Q, H, K, d, rot, dtype, interleaved):
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    q, k, wq, wk, dq, dk = _inputs(B, T, Q, H, K, d, dtype, seed=T + d)
    table = rope_table(T + 50, rot, device=DEV)
    pos = torch.randint(0, T + 50, (B, T), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    leaf = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rope(*leaf, table, pos, eps=EPS, interleaved=interleaved)
    gq, gk, gwq, gwk = torch.autograd.grad((yq, yk), leaf, (dq, dk))
    plain = qk_norm_rope(q, k, wq, wk, table, pos.int(), eps=EPS, interleaved=interleaved)
    assert torch.equal(plain[0], yq) and torch.equal(plain[1], yk)
    for x, w, a, dy, y, gx, gw in ((q, wq, table[pos[:, T - Q:]], dq, yq, gq, gwq), (k, wk, table[pos], dk, yk, gk, gwk)):
        ry, rdx, rdw, terms = _ref(x, w, a, interleaved, dy)
        _close(y.detach(), ry, dtype, "y")
        _close(gx, rdx, dtype, "dx", terms)
        # a sum of n products of magnitude |dy| |xh| (some 4 each): n * 16 * 2^-24 bounds any order of 32-bit sums
        n = x.shape[0] * x.shape[1] * x.shape[2]
        assert (gw.double() - rdw).abs().max().item() <= (n + 30) * 40 * 2.0 ** -24
        assert gw.dtype == torch.float32


def test_default_positions_and_no_weights():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, qk_norm_rope_ref, rope_table
    q, k, *_ = _inputs(2, 10, 4, 2, 2, 32, torch.float32)
    table = rope_table(10, 32, device=DEV)
    got = qk_norm_rope(q, k, None, None, table)
    ref = qk_norm_rope_ref(q, k, None, None, table)
    for a, b in zip(got, ref):
        assert (a - b).abs().max().item() <= 2 * CHAIN * b.abs().max().item()
    only, none = qk_norm_rope(q, None, None, None, table, torch.arange(6, 10, device=DEV))
    assert none is None and torch.equal(only, got[0])


@pytest.mark.parametrize("how", ["misaligned", "transposed", "expanded", "inner"])
def test_strides(how):
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    g = torch.Generator(device=DEV).manual_seed(3)
    B, T, H, d = 3, 6, 4, 64
    if how == "misaligned":
        x = torch.randn(B * T * H * d + 1, generator=g, device=DEV).to(torch.bfloat16)[1:].view(B, T, H, d)
    elif how == "transposed":
        x = torch.randn(B, H, T, d, generator=g, device=DEV).to(torch.bfloat16).transpose(1, 2)
    elif how == "expanded":
        x = torch.randn(1, T, 1, d, generator=g, device=DEV).to(torch.bfloat16).expand(B, T, H, d)
    else:
        x = torch.randn(B, T, d, H, generator=g, device=DEV).to(torch.bfloat16).transpose(2, 3)
    table = rope_table(T, d, device=DEV)
    a = qk_norm_rope(x, x, None, None, table)
    b = qk_norm_rope(x.contiguous(), x.contiguous(), None, None, table)
    # sums in another order may round differently
    for u, v in zip(a, b):
        assert u.is_contiguous() and (u.float() - v.float()).abs().max().item() <= 2.0 ** -8 * v.float().abs().max().item()


def test_gradient_of_broadcast_and_unused_outputs():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    q, k, wq, wk, dq, dk = _inputs(2, 5, 5, 4, 1, 32, torch.float32)
    table = rope_table(5, 32, device=DEV)
    kk = k.detach().requires_grad_()
    _, yk = qk_norm_rope(q, kk.expand(-1, -1, 4, -1), wq, wk, table)        # one head for four: gradients add up
    yk.backward(dq)
    _, rdx, _, _ = _ref(k.expand(-1, -1, 4, -1), wk, table[None], False, dq)
    rdx = rdx.sum(2, keepdim=True)
    assert (kk.grad.double() - rdx).abs().max().item() <= 5 * CHAIN * rdx.abs().max().item() + 4 * CHAIN
    qq = q.detach().requires_grad_()
    yq, _ = qk_norm_rope(qq, k, wq, wk, table)
    yq.sum().backward()
    assert torch.isfinite(qq.grad).all()


def test_gradient_against_differences():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    q, k, wq, wk, dq, dk = _inputs(1, 3, 3, 2, 1, 32, torch.float32)
    table = rope_table(3, 32, device=DEV)
    leaf = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]

    def loss(a, b, c, e):
        y = qk_norm_rope(a, b, c, e, table)
        return (y[0].double() * dq.double()).sum() + (y[1].double() * dk.double()).sum()

    grads = torch.autograd.grad(loss(*leaf), leaf)
    g = torch.Generator(device=DEV).manual_seed(5)
    with torch.no_grad():
        for i, t in enumerate(leaf):
            v = torch.randn(t.shape, generator=g, device=DEV)
            h = 2.0 ** -6
            up = [x + h * v if j == i else x for j, x in enumerate(leaf)]
            dn = [x - h * v if j == i else x for j, x in enumerate(leaf)]
            slope = ((loss(*up) - loss(*dn)) / (2 * h)).item()
            want = (grads[i].double() * v.double()).sum().item()
            # central differences: h^2 / 6 times the third derivative (of the norm: some tens) plus 2^-24 / h a value
            size = grads[i].norm().item() * v.norm().item()
            assert abs(slope - want) <= 2e-2 * size, (i, slope, want)


def test_zero_rows_infinities_and_positions_outside():
    from primus_dlrm_b200.ops import rotary
    x = torch.randn(1, 4, 2, 32, device=DEV)
    x[0, 1] = 0
    x[0, 2, 0, 3] = float("inf")
    x[0, 2, 1, 3] = float("nan")
    table = rotary.rope_table(4, 32, device=DEV)
    y, _ = rotary.qk_norm_rope(x, None, None, None, table)
    assert (y[0, 1] == 0).all() and torch.isfinite(y[0, [0, 3]]).all()
    assert torch.isnan(y[0, 2, 1]).all()
    assert rotary.rotary_error_code(x.device) == 0
    rotary._err_word(x.device).zero_()
    leaf = x.detach()[:, [0, 3, 3]].requires_grad_()
    y, _ = rotary.qk_norm_rope(leaf, None, None, None, table, torch.tensor([0, 4, -1], device=DEV))
    assert rotary.rotary_error_code(x.device) == 1
    assert (y[0, 1:] == 0).all() and (y[0, 0] != 0).any()
    y.sum().backward()
    assert (leaf.grad[0, 1:] == 0).all()
    rotary._err_word(x.device).zero_()


def test_same_bits_each_time():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    q, k, wq, wk, dq, dk = _inputs(64, 100, 100, 8, 8, 32, torch.bfloat16)
    table = rope_table(100, 32, device=DEV)
    seen = []
    for _ in range(3):
        leaf = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        seen.append(torch.autograd.grad(qk_norm_rope(*leaf, table), leaf, (dq, dk)))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_other_stream():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    table = rope_table(50, 32, device=DEV)
    x = torch.randn(8, 50, 8, 32, device=DEV)
    want = qk_norm_rope(x, x, None, None, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = qk_norm_rope(x, x, None, None, table)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shape", [(0, 4, 2, 32), (2, 0, 2, 32), (2, 4, 0, 32)])
def test_empty(shape):
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    w = torch.ones(32, device=DEV, requires_grad=True)
    y, _ = qk_norm_rope(x, None, w, None, rope_table(4, 32, device=DEV))
    assert y.shape == shape
    y.sum().backward()
    assert (w.grad == 0).all()


def test_refusals():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    x = torch.zeros(1, 4, 2, 32, device=DEV)
    t = rope_table(4, 32, device=DEV)
    for bad in (
        lambda: qk_norm_rope(x[0], None, None, None, t),
        lambda: qk_norm_rope(x, x[:, :2], None, None, t),
        lambda: qk_norm_rope(x, x.bfloat16(), None, None, t),
        lambda: qk_norm_rope(x.double(), None, None, None, t),
        lambda: qk_norm_rope(x, None, torch.ones(16, device=DEV), None, t),
        lambda: qk_norm_rope(x, None, None, None, t.cpu()),
        lambda: qk_norm_rope(x, None, None, None, rope_table(4, 64, device=DEV)),
        lambda: qk_norm_rope(x, None, None, None, t, torch.arange(3, device=DEV)),
        lambda: qk_norm_rope(x, None, None, None, t, torch.arange(4, device=DEV).float()),
        lambda: qk_norm_rope(x[..., :31], None, None, None, rope_table(4, 30, device=DEV)),
        lambda: qk_norm_rope(torch.zeros(1, 1, 1, 258, device=DEV), None, None, None, t),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            bad()


def test_second_derivatives_are_refused():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    x = torch.randn(1, 4, 2, 32, device=DEV, requires_grad=True)
    y, _ = qk_norm_rope(x, None, None, None, rope_table(4, 32, device=DEV))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)
