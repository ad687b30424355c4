"""The paged 8-bit cache and its attention on the GPU against plain PyTorch:
append bit for bit against the eager form, attention against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _cache(n_pages, H, d, P, seed=0, spread=0.5):
    from primus_dlrm_b200.ops.kv_cache import PagedKVCache, page_scale
    g = torch.Generator(device=DEV).manual_seed(seed)
    parts = []
    for _ in range(2):
        x = torch.randn(n_pages, H, P, d, generator=g, device=DEV)
        x = x * torch.exp(spread * torch.randn(n_pages, H, 1, 1, generator=g, device=DEV))
        s = page_scale(x.abs().amax((2, 3)))
        parts.append(((x / s[..., None, None]).to(E4M3), s))
    return PagedKVCache.from_tensors(parts[0][0], parts[1][0], parts[0][1], parts[1][1])


def _clone(c, device):
    from primus_dlrm_b200.ops.kv_cache import PagedKVCache
    def f(t):
        return t.view(torch.uint8).clone().to(device).view(E4M3) if t.dtype == E4M3 else t.clone().to(device)
    return PagedKVCache.from_tensors(f(c.k), f(c.v), f(c.k_scale), f(c.v_scale))


def _table(lens, P, n_pages, seed=0, room=0):
    n = [-(-t // P) for t in lens]
    assert sum(n) <= n_pages
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).int()
    t, at = torch.full((len(n), max(n + [1]) + room), -1, dtype=torch.int32), 0
    for b, k in enumerate(n):
        t[b, :k] = ids[at:at + k]
        at += k
    return t.to(DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _same(a, b):
    """Caches hold the same bits (a NaN has one code)."""
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.view(torch.uint8).cpu(), y.view(torch.uint8).cpu())
    for x, y in ((a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        assert torch.equal(x.cpu(), y.cpu())


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("P,d,H", [(16, 32, 3), (32, 64, 2), (64, 128, 2), (64, 32, 1), (16, 128, 1)])
@pytest.mark.parametrize("held,new", [([0], [1]), ([0, 5, 63, 64], [1, 1, 1, 1]), ([3, 0, 17], [200, 64, 0]),
                                      ([15, 16, 31], [2, 1, 130])])
def test_append_matches_eager_bit_for_bit(P, d, H, dtype, held, new):
    """No norm and no rotation: every step is exact or one rounding, so the bits agree."""
    g = torch.Generator(device=DEV).manual_seed(7)
    after = [a + n for a, n in zip(held, new)]
    c = _cache(sum(-(-t // P) for t in after) + 2, H, d, P, seed=1, spread=2.0)
    table = _table(after, P, c.n_pages)
    N = sum(new)
    k, v = ((torch.randn(N, H, d, generator=g, device=DEV) * torch.exp(2 * torch.randn(N, 1, 1, generator=g, device=DEV)))
            .to(dtype) for _ in range(2))
    cu = _i32([0] + list(torch.tensor(new).cumsum(0)))
    ref = _clone(c, "cpu")
    c.append(k, v, table, _i32(held), cu, max(new))
    ref.append(k.cpu(), v.cpu(), table.cpu(), _i32(held).cpu(), cu.cpu())
    _same(c, ref)
    c.check_errors()
    # the uniform form and an unknown longest length do the same
    if len(set(new)) == 1:
        c2 = _clone(c, DEV)
        c2.append(k.view(len(new), new[0], H, d), v.view(len(new), new[0], H, d), table, _i32(held))
        _same(c2, c)
    c3 = _clone(c, DEV)
    c3.append(k, v, table, _i32(held), cu)
    _same(c3, c)
    # and reading gives the values back
    got = c.read(table, _i32(after))
    want = ref.read(table.cpu(), _i32(after).cpu())
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    first = _i32([max(0, a - 3) for a in held])
    got, want = c.read(table, _i32(after), first, 9), ref.read(table.cpu(), _i32(after).cpu(), first.cpu(), 9)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("P,d", [(16, 32), (64, 64), (32, 128)])
def test_append_with_norm_and_rotation(P, d, interleaved):
    """Values against 64 bits: one e4m3 rounding (2^-4 of the value above the subnormals, half the smallest step
    2^-10 of the scale below) on top of 32-bit arithmetic."""
    from primus_dlrm_b200.ops.rotary import rope_table
    g = torch.Generator(device=DEV).manual_seed(2)
    H, held, new = 2, [0, 21], [40, 40]
    after = [a + n for a, n in zip(held, new)]
    c = _cache(20, H, d, P)
    table = _table(after, P, 20)
    k, v = (torch.randn(2, 40, H, d, generator=g, device=DEV) for _ in range(2))
    w = 1 + 0.3 * torch.randn(d, generator=g, device=DEV)
    ang = rope_table(100, d, device=DEV)
    c.append(k, v, table, _i32(held), k_weight=w, norm_eps=1e-6, rope=ang, interleaved=interleaved)
    c.check_errors()
    got, _ = c.read(table, _i32(after), _i32(held), 40)
    for b in range(2):
        x = k[b].double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
        a = ang[held[b]:after[b]].double()
        h = d // 2
        i0 = torch.arange(0, d, 2) if interleaved else torch.arange(h)
        i1 = i0 + 1 if interleaved else i0 + h
        y = x.clone()
        y[..., i0] = x[..., i0] * a[:, None, :h] - x[..., i1] * a[:, None, h:]
        y[..., i1] = x[..., i0] * a[:, None, h:] + x[..., i1] * a[:, None, :h]
        big = 8.0 / 256                                   # scale of a page whose largest value is below 8 * 1.75
        assert y.abs().max() < 14
        assert ((got[b].double() - y).abs() <= 2.0 ** -4 * y.abs() * 1.0001 + 2.0 ** -10 * big + 1e-5).all()


def test_append_one_by_one_and_at_once():
    """Token by token a page's scale may only grow; the values stay within the roundings: each raise of the scale
    rounds what became subnormal again, by half a step 2^-10 of the new scale."""
    H, d, P, n = 2, 64, 32, 50
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = ((torch.randn(1, n, H, d, generator=g, device=DEV) * torch.linspace(0.01, 30, n, device=DEV)[None, :, None, None])
            for _ in range(2))
    one, all_ = _cache(4, H, d, P), _cache(4, H, d, P)
    table = _table([n], P, 4)
    all_.append(k, v, table, _i32([0]))
    for i in range(n):
        one.append(k[:, i:i + 1], v[:, i:i + 1], table, _i32([i]))
    assert torch.equal(one.k_scale[table[0].long()], all_.k_scale[table[0].long()])
    a, b = one.read(table, _i32([n]), n=n), all_.read(table, _i32([n]), n=n)
    for x, y, s in ((a[0], b[0], all_.k_scale), (a[1], b[1], all_.v_scale)):
        step = s[table[0].long()].repeat_interleave(P, 0)[:n] * 2.0 ** -9         # one step among the subnormals
        assert ((x[0] - y[0]).float().abs() <= step[..., None] * 1.0001).all()


def test_append_extremes():
    from primus_dlrm_b200.ops.kv_cache import page_scale
    H, d, P = 1, 32, 16
    c, table = _cache(3, H, d, P), _table([16], P, 3)
    k = torch.zeros(1, 16, H, d, device=DEV)
    k[0, 1, 0, 0], k[0, 2, 0, 0], k[0, 3, 0, :3] = float("inf"), float("nan"), torch.tensor([448.0, -1.0, 2.0 ** -9])
    v = torch.zeros_like(k)
    c.append(k, v, table, _i32([0]))
    page = int(table[0, 0])
    assert c.k_scale[page, 0].item() == 1.0 and c.v_scale[page, 0].item() == 2.0 ** -100
    got = c.read(table, _i32([16]))[0][0, :, 0].float()
    assert torch.isnan(got[1, 0]) and torch.isnan(got[2, 0]) and got[3, :3].tolist() == [448.0, -1.0, 2.0 ** -9]
    big = torch.full((1, 1, H, d), 3e38, device=DEV)
    c.append(big, big * 1e-38 * 1e-6, table, _i32([3]))
    assert c.k_scale[page, 0].item() == page_scale(big.amax()).item() == 2.0 ** 120
    got = c.read(table, _i32([4]))[0][0, :, 0].float()
    assert (got[0] == 0).all() and torch.isnan(got[1, 0]) and (got[3] > 2.9e38).all()
    c.check_errors()


@pytest.mark.parametrize("how", ["misaligned", "transposed", "expanded", "inner"])
def test_append_strides(how):
    g = torch.Generator(device=DEV).manual_seed(4)
    B, n, H, d, P = 2, 20, 2, 64, 16
    if how == "misaligned":
        x = torch.randn(B * n * H * d + 1, generator=g, device=DEV).bfloat16()[1:].view(B, n, H, d)
    elif how == "transposed":
        x = torch.randn(B, H, n, d, generator=g, device=DEV).bfloat16().transpose(1, 2)
    elif how == "expanded":
        x = torch.randn(B, n, 1, d, generator=g, device=DEV).bfloat16().expand(B, n, H, d)
    else:
        x = torch.randn(B, n, d, H, generator=g, device=DEV).bfloat16().transpose(2, 3)
    a, b = _cache(6, H, d, P), _cache(6, H, d, P)
    wide = torch.full((B, 8), -1, dtype=torch.int32, device=DEV)      # a page table that is part of a wider one
    table = _table([n + 3] * B, P, 6)
    wide[:, :table.shape[1]] = table
    a.append(x, x, wide[:, :table.shape[1]], _i32([3] * B))
    b.append(x.contiguous(), x.contiguous(), table, _i32([3] * B))
    _same(a, b)


def test_append_errors_skip():
    """A page id outside the pool, and positions behind the page table, are skipped and reported."""
    c = _cache(3, 1, 32, 16)
    x = torch.ones(2, 20, 1, 32, device=DEV)
    before = _clone(c, DEV)
    c.append(x, x, _i32([[7, -1], [99, 3]]), _i32([0, 0]))
    _same(c, before)
    with pytest.raises(RuntimeError, match="out of range"):
        c.check_errors()
    c.check_errors()
    c.append(x[:1], x[:1], _i32([[1]]), _i32([0]))                     # 16 of 20 tokens have a page
    assert c.k_scale[1, 0].item() == 2.0 ** -8
    with pytest.raises(RuntimeError):
        c.check_errors()
    c.append(x[:1], x[:1], _i32([[0]]), _i32([-4]))
    with pytest.raises(RuntimeError):
        c.check_errors()


# ---------------------------------------------------------------- attention
def _attn_check(q, c, table, lens, cu=None, max_q=None, **kw):
    from primus_dlrm_b200.ops.kv_cache import paged_attention, paged_attention_ref
    ref, lref = paged_attention_ref(q, c, table, lens, cu, kw.get("scale"), kw.get("causal", True), torch.float64)
    o, lse = paged_attention(q, c, table, lens, cu, max_q, return_lse=True, **kw)
    c.check_errors()
    o2 = paged_attention(q, c, table, lens, cu, max_q, **kw)
    assert torch.equal(o, o2) and o.dtype == q.dtype and o.shape == q.shape and lse.shape == q.shape[:-1]
    vmax = (c.v.float().nan_to_num().abs().amax((2, 3)) * c.v_scale).max().item()
    # one rounding to the output's type (8 or 11 significant bits); probabilities rounded to 11 bits (2^-11 of the
    # weighted mean of |v|, which is at most the largest |v|); exponents off by the 32-bit error of the scores: d + 8 roundings of 2^-24 of
    # sum |q k| <= |q| |k|, twice (score and maximum), and 2^-21 from the exponential
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    d = q.shape[-1]
    scale = kw.get("scale") or d ** -0.5
    kmax = (c.k.float().nan_to_num().norm(dim=-1).amax(-1) * c.k_scale).max().item()
    score = abs(scale) * q.float().norm(dim=-1).max().item() * kmax
    soft = 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * score + 2.0 ** -20
    tol = unit * ref.abs() * 1.01 + soft * vmax + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    inf = torch.isinf(o)                                         # only what the type cannot hold is infinite
    assert (ref.abs() + tol)[inf].gt(torch.finfo(q.dtype).max).all() and torch.equal(o[inf] > 0, ref[inf] > 0)
    bad = ((o.double() - ref).abs() - tol)[~inf]
    assert not torch.isnan(o).any() and bad.max().item() <= 0, bad.max().item()
    none = lref == -math.inf
    assert torch.equal(none, lse == -math.inf) and (o[none] == 0).all()
    # the sum: 32-bit scores as above, 2^-20 of the exponentials and roundings of the running sum
    err = (lse.double() - lref)[~none].abs()
    assert err.numel() == 0 or err.max().item() <= 2 * (d + 8) * 2.0 ** -24 * score + 2.0 ** -12, err.max().item()
    return o, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P,d,H,G", [(16, 32, 2, 1), (32, 64, 2, 4), (64, 128, 1, 5), (64, 32, 3, 8), (16, 128, 2, 16),
                                     (32, 32, 1, 20), (64, 64, 1, 1)])
@pytest.mark.parametrize("lens,n", [([1], 1), ([63, 64, 65, 1], 1), ([1000, 17], 1), ([33, 2, 129], 2), ([130, 300], 19),
                                    ([40, 257], 40)])
def test_attention(P, d, H, G, dtype, lens, n):
    g = torch.Generator(device=DEV).manual_seed(d + n)
    c = _cache(sum(-(-t // P) for t in lens) + 1, H, d, P, seed=n)
    table = _table(lens, P, c.n_pages, room=2)
    q = (1.5 * torch.randn(len(lens), n, H * G, d, generator=g, device=DEV)).to(dtype)
    _attn_check(q, c, table, _i32(lens))
    _attn_check(q, c, table, _i32(lens), causal=False, max_len=max(lens))


@pytest.mark.parametrize("P,d,H,G", [(16, 64, 2, 2), (64, 32, 1, 3), (64, 128, 2, 1)])
@pytest.mark.parametrize("lens,new", [([5, 70, 400], [5, 1, 123]), ([300, 0, 9, 64], [0, 0, 3, 64]), ([700], [700]),
                                      ([1, 2000, 3], [1, 1, 3])])
def test_attention_ragged(P, d, H, G, lens, new):
    g = torch.Generator(device=DEV).manual_seed(sum(lens))
    c = _cache(sum(-(-t // P) for t in lens) + 1, H, d, P)
    table = _table(lens, P, c.n_pages)
    q = torch.randn(sum(new), H * G, d, generator=g, device=DEV).bfloat16()
    cu = _i32([0] + list(torch.tensor(new).cumsum(0)))
    a, _ = _attn_check(q, c, table, _i32(lens), cu, max(new))
    _attn_check(q, c, table, _i32(lens), cu)
    _attn_check(q, c, table, _i32(lens), cu, causal=False, scale=0.05)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("P,d,H,G,most", [(64, 64, 4, 1, 300), (16, 64, 2, 3, 90), (32, 32, 4, 2, 130), (64, 32, 2, 1, 200),
                                          (16, 32, 8, 1, 65), (64, 128, 4, 1, 150), (32, 128, 2, 2, 70), (16, 128, 8, 1, 40),
                                          (32, 64, 8, 1, 40), (64, 32, 8, 1, 33), (64, 32, 4, 1, 300), (64, 128, 4, 1, 400)])
def test_many_rows(P, d, H, G, most, causal, dtype):
    """Enough rows and sequences for the forms that share copies among rows (and some just below), ragged, with rows
    without keys and empty sequences among them."""
    g = torch.Generator(device=DEV).manual_seed(d + most)
    B = 160 // H + 3
    new = [max(1, most - (i * 37) % most) for i in range(B)]
    lens = [max(0, n + (i * 53) % 211 - 40) for i, n in enumerate(new)]
    new[1], lens[1], lens[2], new[3] = 0, 40, 0, most
    c = _cache(sum(-(-t // P) for t in lens) + 1, H, d, P, seed=most)
    table = _table(lens, P, c.n_pages, room=1)
    q = (1.5 * torch.randn(sum(new), H * G, d, generator=g, device=DEV)).to(dtype)
    cu = _i32([0] + list(torch.tensor(new).cumsum(0)))
    o, _ = _attn_check(q, c, table, _i32(lens), cu, max(new), causal=causal)
    # the same, a sequence at a time (other forms): within both forms' tolerances
    for b in (0, 3, B - 1):
        a, e = int(cu[b]), int(cu[b + 1])
        _attn_check(q[None, a:e], c, table[b:b + 1], _i32(lens[b:b + 1]), causal=causal)


def test_many_rows_that_need_rescaling():
    """Scores that keep growing along the keys, so that running maxima are raised again and again; very different
    pages; and stale NaN codes behind every sequence's keys."""
    g = torch.Generator(device=DEV).manual_seed(2)
    for d, P in ((64, 64), (32, 16), (128, 32)):
        B, H, n, T = 40, 4, 100, 300
        c = _cache(B * -(-T // P), H, d, P, spread=2.0)
        table = _table([T] * B, P, c.n_pages)
        for j in range(table.shape[1]):
            c.k_scale[table[:, j].long()] *= 2.0 ** (j * P // 64)
        q = torch.randn(B, n, H, d, generator=g, device=DEV).bfloat16()
        lens = [T - 7 - i for i in range(B)]
        for x in (c.k, c.v):
            codes = x.view(torch.uint8)
            for b, t in enumerate(lens):
                codes[table[b, t // P].long(), :, t % P:] = 0x7F
                codes[table[b, t // P + 1:].long()] = 0x7F
        _attn_check(q, c, table, _i32(lens))


@pytest.mark.parametrize("n,lens", [(4, [2, 0, 4, 70]), (1, [0, 1, 0]), (70, [3, 65, 0])])
def test_rows_without_keys(n, lens):
    """More queries than tokens: the first rows see nothing and give zeros."""
    c = _cache(12, 2, 64, 16)
    table = _table(lens, 16, 12)
    q = torch.randn(len(lens), n, 4, 64, device=DEV).bfloat16()
    o, lse = _attn_check(q, c, table, _i32(lens))
    for b, t in enumerate(lens):
        assert (o[b, :max(0, n - t)] == 0).all() and (lse[b, :max(0, n - t)] == -math.inf).all()
        assert torch.isfinite(lse[b, max(0, n - t):]).all()


@pytest.mark.parametrize("n", [1, 5, 33])
@pytest.mark.parametrize("d,P", [(32, 64), (64, 16), (128, 32)])
def test_what_lies_behind_the_length_does_not_matter(n, d, P):
    """NaN codes behind a sequence's length, in its last page and in pages that nobody reads."""
    lens = [P + 1 + n, 3 * P - 1, n]
    c = _cache(16, 2, d, P)
    table = _table(lens, P, 16)
    q = torch.randn(3, n, 2, d, device=DEV).bfloat16()
    want, _ = _attn_check(q, c, table, _i32(lens))
    used = torch.zeros(16, P, dtype=torch.bool, device=DEV)
    for b, t in enumerate(lens):
        for j in range(t):
            used[table[b, j // P], j % P] = True
    for x in (c.k, c.v):
        x.view(torch.uint8)[(~used)[:, None, :, None].expand(x.shape)] = 0x7F
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    assert torch.equal(paged_attention(q, c, table, _i32(lens)), want)


def test_nan_in_a_visible_key_reaches_its_rows_only():
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(4, 1, 32, 16)
    table = _table([40], 16, 4)
    c.k.view(torch.uint8)[table[0, 2].long(), 0, 3] = 0x7F                # token 35
    q = torch.randn(1, 10, 1, 32, device=DEV).bfloat16()                  # positions 30 to 39
    o = paged_attention(q, c, table, _i32([40]))
    assert torch.isfinite(o[0, :5].float()).all() and torch.isnan(o[0, 5:].float()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 40])
def test_extreme_queries_and_scales(dtype, n):
    """Large and tiny queries and pages of very different scales: nothing over- or underflows on the way."""
    g = torch.Generator(device=DEV).manual_seed(6)
    c = _cache(12, 2, 64, 32, spread=3.0)
    c.k_scale[0::2] *= 2.0 ** -12
    c.v_scale[1::3] *= 2.0 ** 20
    lens = [100, 200]
    table = _table(lens, 32, 12)
    q = torch.randn(2, n, 2, 64, generator=g, device=DEV)
    top = 6e4 if dtype == torch.float16 else 1e30
    for f in (top, 1e-6, 0.0):
        x = (q / q.abs().max() * f).to(dtype)
        _attn_check(x, c, table, _i32(lens), scale=(64 ** -0.5 / f) if f else None)


@pytest.mark.parametrize("lens,n,G", [([20000], 1, 4), ([9000, 30, 4000], 3, 2), ([6000], 64, 1)])
def test_long(lens, n, G):
    g = torch.Generator(device=DEV).manual_seed(9)
    c = _cache(sum(-(-t // 64) for t in lens), 2, 64, 64)
    table = _table(lens, 64, c.n_pages)
    q = (2 * torch.randn(len(lens), n, 2 * G, 64, generator=g, device=DEV)).bfloat16()
    _attn_check(q, c, table, _i32(lens))


def test_offsets_past_32_bits():
    """Pages whose codes begin behind 2^32 bytes."""
    from primus_dlrm_b200.ops.kv_cache import PagedKVCache, paged_attention
    H, P, d = 16, 64, 128
    n_pages = (1 << 32) // (H * P * d) + 70
    big = PagedKVCache(n_pages, H, d, P, device=DEV)
    small = PagedKVCache(3, H, d, P, device=DEV)
    k, v = (torch.randn(1, 150, H, d, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(1, 20, H, d, device=DEV).bfloat16()
    tb, ts = _i32([[n_pages - 1, n_pages - 60, 0]]), _i32([[2, 1, 0]])
    for c, t in ((big, tb), (small, ts)):
        c.append(k, v, t, _i32([0]))
        c.check_errors()
    assert torch.equal(big.read(tb, _i32([150]))[1], small.read(ts, _i32([150]))[1])
    for x in (q, q[:, -1:]):
        assert torch.equal(paged_attention(x, big, tb, _i32([150])), paged_attention(x, small, ts, _i32([150])))


@pytest.mark.parametrize("how", ["misaligned", "transposed", "inner"])
@pytest.mark.parametrize("n", [1, 37])
def test_attention_query_strides(how, n):
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    B, H, d = 2, 4, 64
    if how == "misaligned":
        q = torch.randn(B * n * H * d + 1, device=DEV).bfloat16()[1:].view(B, n, H, d)
    elif how == "transposed":
        q = torch.randn(B, H, n, d, device=DEV).bfloat16().transpose(1, 2)
    else:
        q = torch.randn(B, n, d, H, device=DEV).bfloat16().transpose(2, 3)
    c = _cache(8, 2, d, 32)
    table = _table([50, 90], 32, 8)
    lens = _i32([50, 90])
    assert torch.equal(paged_attention(q, c, table, lens), paged_attention(q.contiguous(), c, table, lens))


def test_shared_pages():
    """Candidates that follow one history: each sequence equals its own copy."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(40, 2, 32, 16)
    C, n, S = 9, 5, 32
    table = torch.stack([_i32([30, 31, 2 * i]) for i in range(C)])
    q = torch.randn(C, n, 4, 32, device=DEV).bfloat16()
    lens = _i32([S + n] * C)
    o, _ = _attn_check(q, c, table, lens)
    for i in range(C):
        assert torch.equal(paged_attention(q[i:i + 1], c, table[i:i + 1], lens[i:i + 1])[0], o[i]) or \
            (paged_attention(q[i:i + 1], c, table[i:i + 1], lens[i:i + 1])[0].float() - o[i].float()).abs().max() < 2e-2


def test_longer_than_the_stated_most():
    """A sequence of more tokens than ``max_new`` / ``max_q`` is skipped and reported; the others are served."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(8, 1, 32, 16)
    x = torch.ones(33, 1, 32, device=DEV)
    before = _clone(c, DEV)
    c.append(x, x, _i32([[0, 1, 2], [3, 4, 5]]), _i32([0, 0]), _i32([0, 1, 33]), 16)
    assert c.k_scale[0, 0].item() == 2.0 ** -8
    assert torch.equal(c.k_scale[1:], before.k_scale[1:])
    with pytest.raises(RuntimeError, match="length"):
        c.check_errors()
    for n in (2, 140):                                                # few rows, many rows
        q = torch.randn(3 * n, 1, 32, device=DEV).bfloat16()
        table, lens, cu = _i32([[0, 1]] * 2), _i32([32, 32]), _i32([0, n, 3 * n])
        o = paged_attention(q, c, table, lens, cu, n)
        with pytest.raises(RuntimeError, match="length"):
            c.check_errors()
        # values lie in [0, 1]; either side is within 2^-9 (bf16) + 2^-10 (probabilities) of the exact sum
        alone = paged_attention(q[:n], c, table[:1], lens[:1], cu[:2], n)
        assert (o[:n].float() - alone.float()).abs().max() <= 2.0 ** -7
        c.check_errors()
    o, lse = paged_attention(q, c, table, lens, cu, 0, return_lse=True)
    assert (o == 0).all() and (lse == -torch.inf).all()


def test_attention_errors_mask():
    """A page id outside the pool counts as masked tokens; a length behind the page table is cut; both are reported."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(4, 1, 32, 16)
    for n in (1, 20):
        q = torch.randn(1, n, 1, 32, device=DEV).bfloat16()
        o = paged_attention(q, c, _i32([[0, 77]]), _i32([32]))
        assert torch.isfinite(o.float()).all()
        with pytest.raises(RuntimeError, match="out of range"):
            c.check_errors()
        o = paged_attention(q, c, _i32([[0]]), _i32([30]), causal=False)
        assert torch.equal(o, paged_attention(q, c, _i32([[0]]), _i32([16]), causal=False))
        with pytest.raises(RuntimeError, match="length"):
            c.check_errors()


def test_graph_and_stream():
    """Captured once, run on new lengths and queries."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(12, 2, 64, 32)
    table = _table([150, 150], 32, 12)
    q, lens = torch.randn(2, 1, 4, 64, device=DEV).bfloat16(), _i32([100, 30])
    k = torch.randn(2, 1, 2, 64, device=DEV).bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            c.append(k, k, table, lens)
            paged_attention(q, c, table, lens + 1)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(k, k, table, lens)
        o = paged_attention(q, c, table, lens + 1)
    for a, b in ((101, 31), (5, 149)):
        lens.copy_(_i32([a, b]))
        q.normal_()
        g.replay()
        got = o.clone()
        want = paged_attention(q, c, table, lens + 1)
        assert torch.equal(got, want)
    c.check_errors()


def test_refusals():
    from primus_dlrm_b200.ops.kv_cache import PagedKVCache, paged_attention
    c = _cache(4, 2, 32, 16)
    t, n = _i32([[0, 1]]), _i32([5])
    q = torch.zeros(1, 1, 4, 32, device=DEV, dtype=torch.bfloat16)
    k = torch.zeros(1, 1, 2, 32, device=DEV)
    from primus_dlrm_b200.ops.rotary import rope_table
    for bad in (
        lambda: paged_attention(q.float(), c, t, n),
        lambda: paged_attention(q[..., :16], c, t, n),
        lambda: paged_attention(q[:, :, :3], c, t, n),
        lambda: paged_attention(q[0], c, t, n),
        lambda: paged_attention(q.cpu(), c, t, n),
        lambda: paged_attention(q, c, t.long(), n),
        lambda: paged_attention(q, c, t, n.long()),
        lambda: paged_attention(q, c, t, _i32([5, 5])),
        lambda: paged_attention(q[0], c, t, n, _i32([0])),
        lambda: c.append(k, k[..., :16], t, n),
        lambda: c.append(k, k.bfloat16(), t, n),
        lambda: c.append(k.double(), k.double(), t, n),
        lambda: c.append(k[0], k[0], t, n),
        lambda: c.append(k, k, t, n.cpu()),
        lambda: c.append(k, k, t, n, k_weight=torch.ones(32, device=DEV)),
        lambda: c.append(k, k, t, n, rope=rope_table(9, 16, device=DEV)),
        lambda: c.read(t.long(), n),
        lambda: PagedKVCache(4, 2, 48, device=DEV),
        lambda: PagedKVCache(4, 2, 64, page_size=128, device=DEV),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    c.check_errors()
