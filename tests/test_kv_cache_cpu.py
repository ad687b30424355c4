"""Eager forms of the rotary norm, the paged 8-bit cache and its attention (CPU), and their refusals."""
import math

import pytest
import torch

from primus_dlrm_b200.ops.kv_cache import PagedKVCache, page_scale, paged_attention
from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def test_page_scale():
    """The smallest power of two that brings the magnitude to 448 or less."""
    for x in (448.0, 448.5, 1.75, 1.7500001, 1.0, 2.0 ** -91, 3e-45, 0.0, 3.4e38, 7.0, 7.5):
        s = page_scale(torch.tensor(x)).item()
        assert math.log2(s) == int(math.log2(s)) and s >= 2.0 ** -100
        t = torch.tensor(x).item()
        assert t / s <= 448 and (s == 2.0 ** -100 or t / (s / 2) > 448)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [8, 4, 0])
def test_rotation_is_relative(rot, interleaved):
    """Scores of rotated heads depend on positions through differences; heads leave with unit mean square."""
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, 6, 2, 8, generator=g, dtype=torch.float32) for _ in range(2))
    table = rope_table(200, rot)
    a = qk_norm_rope(q, k, None, None, table, torch.arange(6), interleaved=interleaved)
    b = qk_norm_rope(q, k, None, None, table, torch.arange(6) + 100, interleaved=interleaved)
    s = [torch.einsum("bihd,bjhd->bhij", x[0].double(), x[1].double()) for x in (a, b)]
    # angles of up to 106 radians' sines rounded to 2^-24 each, 8 products of size 2 or so
    assert (s[0] - s[1]).abs().max().item() < 1e-5
    assert (a[0].pow(2).mean(-1) - 1).abs().max().item() < 1e-5


def test_queries_are_the_last_tokens():
    q, k = torch.randn(2, 3, 2, 8), torch.randn(2, 7, 2, 8)
    table = rope_table(7, 8)
    yq, yk = qk_norm_rope(q, k, None, None, table)
    full, _ = qk_norm_rope(torch.cat([torch.zeros(2, 4, 2, 8), q], 1), k, None, None, table)
    assert torch.equal(yq, full[:, 4:])


def test_rotary_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    leaf = [torch.randn(1, 3, 2, 8, generator=g).requires_grad_(), torch.randn(1, 3, 1, 8, generator=g).requires_grad_(),
            torch.rand(8, generator=g).requires_grad_(), torch.rand(8, generator=g).requires_grad_()]
    table = rope_table(3, 8)

    def loss(*t):
        y = qk_norm_rope(*t, table)
        return (y[0].double() ** 3).sum() + (y[1].double() ** 3).sum()

    grads = torch.autograd.grad(loss(*leaf), leaf)
    with torch.no_grad():
        for i, t in enumerate(leaf):
            v, h = torch.randn(t.shape, generator=g), 2.0 ** -6
            up, dn = ([x + e * h * v if j == i else x for j, x in enumerate(leaf)] for e in (1, -1))
            slope, want = ((loss(*up) - loss(*dn)) / (2 * h)).item(), (grads[i] * v).sum().item()
            assert abs(slope - want) <= 2e-2 * grads[i].norm().item() * v.norm().item()


def test_rotary_refusals():
    x = torch.zeros(1, 4, 2, 8)
    t = rope_table(4, 8)
    with pytest.raises(ValueError):
        rope_table(4, 3)
    with pytest.raises(ValueError):
        qk_norm_rope(x[0], None, None, None, t)
    with pytest.raises(ValueError):
        qk_norm_rope(x, x[:, :2], None, None, t)
    with pytest.raises(IndexError):
        qk_norm_rope(x, None, None, None, t, torch.arange(1, 5))


@pytest.mark.parametrize("P", [16, 32, 64])
def test_append_read_round_trip(P):
    """Values survive to half an e4m3 step: 2^-4 relative, or half the subnormal step of the page's scale."""
    g = torch.Generator().manual_seed(P)
    c = PagedKVCache(8, 2, 32, P)
    table = _i32([[5, 1, 2, 7], [0, 3, 4, 6]])
    k, v = (torch.randn(2, 100 if P > 16 else 60, 2, 32, generator=g) for _ in range(2))
    n = k.shape[1]
    cut = 37
    c.append(k[:, :cut], v[:, :cut], table, _i32([0, 0]))
    c.append(k[:, cut:], v[:, cut:], table, _i32([cut, cut]))
    for got, x, s in zip(c.read(table, _i32([n, n]), n=n), (k, v), (c.k_scale, c.v_scale)):
        scale = s[table.long()].repeat_interleave(P, 1)[:, :n, :, None]
        # values of the first piece may have been rounded twice
        assert ((got.float() - x).abs() <= 2 ** -4 * x.abs() * 1.07 + 2 * 2 ** -10 * scale).all()
    assert (c.read(table, _i32([n, n]), _i32([n - 1, n]), 3)[0][0, 1:] == 0).all()


def test_attention_of_an_appended_history_matches_dense():
    """Step by step over the cache against dense causal attention of the values that the cache holds."""
    g = torch.Generator().manual_seed(3)
    T, H, G, d = 45, 2, 3, 32
    c = PagedKVCache(4, H, d, 16)
    table = _i32([[2, 0, 3]])
    k, v = (torch.randn(1, T, H, d, generator=g) for _ in range(2))
    q = torch.randn(1, T, H * G, d, generator=g).bfloat16()
    c.append(k, v, table, _i32([0]))
    kd, vd = (x[:, :T].float() for x in c.read(table, _i32([T])))
    w = torch.einsum("bihd,bjhd->bhij", q.float(), kd.repeat_interleave(G, 2)) * d ** -0.5
    w = w.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -math.inf)
    want = torch.einsum("bhij,bjhd->bihd", w.softmax(-1), vd.repeat_interleave(G, 2))
    o, lse = paged_attention(q, c, table, _i32([T]), return_lse=True)
    assert (o.float() - want).abs().max().item() <= 2 ** -8 * want.abs().max().item() + 1e-5
    assert (lse - w.logsumexp(-1).transpose(1, 2)).abs().max().item() < 1e-4
    for i in (0, 15, 16, 44):
        one = paged_attention(q[:, i:i + 1], c, table, _i32([i + 1]))
        assert (one.float() - want[:, i:i + 1]).abs().max().item() <= 2 ** -8 * want.abs().max().item() + 1e-5
    empty, lse = paged_attention(q[:, :2], c, table, _i32([0]), return_lse=True)
    assert (empty == 0).all() and (lse == -math.inf).all()


def test_copy_pages():
    c = PagedKVCache(4, 1, 32, 16)
    x = torch.randn(1, 10, 1, 32)
    c.append(x, x, _i32([[1]]), _i32([0]))
    c.copy_pages(torch.tensor([1, 1]), torch.tensor([0, 3]))
    a, b = c.read(_i32([[1]]), _i32([10])), c.read(_i32([[3]]), _i32([10]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cache_refusals():
    with pytest.raises(ValueError):
        PagedKVCache(4, 2, 48)
    with pytest.raises(ValueError):
        PagedKVCache(4, 2, 32, page_size=20)
    c = PagedKVCache(2, 1, 32, 16)
    x = torch.zeros(1, 4, 1, 32)
    for bad in (lambda: c.append(x, x, _i32([[0]]), _i32([14])), lambda: c.append(x, x, _i32([[0]]), _i32([-1])),
                lambda: c.append(x, x, _i32([[0]]), _i32([0]), k_weight=torch.ones(32)),
                lambda: c.append(x[0], x[0], _i32([[0]]), _i32([0])),
                lambda: PagedKVCache.from_tensors(c.k, c.v, c.k_scale[:1], c.v_scale),
                lambda: PagedKVCache.from_tensors(c.k.float(), c.v.float(), c.k_scale, c.v_scale)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        c.append(x, x, _i32([[2]]), _i32([0]))
    with pytest.raises(IndexError):
        paged_attention(x.bfloat16(), c, _i32([[-1]]), _i32([4]))
    with pytest.raises(IndexError):
        c.append(x, x, _i32([[0]]), _i32([0]), rope=rope_table(3, 32))
