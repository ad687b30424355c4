"""Edges of the rotary norm, the paged 8-bit cache and its attention on the GPU: values of very different sizes, rows
that nobody computes, refusals."""
import math

import pytest
import torch
from test_kv_cache_gpu import DEV, E4M3, _cache, _clone, _i32, _same, _table

pytestmark = pytest.mark.gpu

# forms of the attention: (d, page, heads, group, sequences, queries of each, keys) -> few rows of 8 and of 16 (shares of
# the keys, and a warp a segment), many rows on tcgen05, many rows at d = 128
FORMS = {
    "8 rows, d 32": (32, 16, 2, 1, 2, 7, 150), "8 rows, d 64": (64, 32, 2, 4, 2, 2, 900),
    "8 rows, d 128": (128, 16, 1, 2, 3, 4, 130), "8 rows, whole pages": (64, 64, 2, 1, 2, 6, 300),
    "16 rows, d 32": (32, 32, 2, 2, 2, 8, 140), "16 rows, d 64": (64, 16, 1, 1, 2, 12, 64),
    "16 rows, d 128": (128, 16, 2, 1, 1, 13, 200), "16 rows, long": (64, 16, 2, 1, 1, 40, 2500), "a warp a segment": (32, 16, 8, 1, 160, 16, 100),
    "tcgen05, d 32": (32, 16, 4, 1, 40, 128, 300), "tcgen05, d 64": (64, 32, 4, 1, 40, 100, 300),
    "many, d 128": (128, 32, 4, 1, 40, 100, 300), "many, d 128, pages of 16": (128, 16, 4, 2, 40, 50, 257),
}


def _plain(q, c, table, lens, causal=True, scale=None):
    """In 64 bits: o, sum_j p |v|, the largest p_j 448 vs_j of each row (keys that it sees only), and lse."""
    B, n, Hq, d = q.shape
    P, G, scale = c.page_size, Hq // c.n_kv_heads, d ** -0.5 if scale is None else scale
    o, a, top = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3))
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        T = int(lens[b])
        if T == 0:
            continue
        ids = table[b, :-(-T // P)].long()
        k, v = ((x.view(torch.uint8)[ids].view(E4M3).double() * s[ids].double()[..., None, None]).transpose(0, 1)
                .flatten(1, 2)[:, :T].repeat_interleave(G, 0) for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
        vs = c.v_scale[ids].double().T.repeat_interleave(P, 1)[:, :T].repeat_interleave(G, 0)
        w = q[b].double().transpose(0, 1) @ k.transpose(1, 2) * scale
        if causal:
            w = w.masked_fill(torch.arange(T, device=q.device) > (T - n + torch.arange(n, device=q.device))[:, None], -math.inf)
        z = torch.logsumexp(w, -1)
        p = torch.where(z[..., None] == -math.inf, 0.0, torch.exp(w - z[..., None]))
        o[b], a[b] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        top[b] = (p * 448 * vs[:, None]).amax(-1).transpose(0, 1)[..., None]
        lse[b] = z.transpose(0, 1)
    return o, a, top, lse


def _check_rows(q, c, table, lens, **kw):
    """Every row against its own size: a rounding to the output's type (8 or 11 significant bits); probabilities in 11
    bits, 2^-11 of sum p |v|, and what falls below them, 2^-30 of the largest product for each key; exponents off by the
    32-bit error of the scores, d + 8 roundings of 2^-24 of |q| |k| each, twice, and 2^-20 from the exponentials."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    ref, size, top, lref = _plain(q, c, table, lens, kw.get("causal", True), kw.get("scale"))
    o, lse = paged_attention(q, c, table, lens, return_lse=True, **kw)
    c.check_errors()
    d = q.shape[-1]
    unit = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    kmax = (c.k.float().nan_to_num().norm(dim=-1).amax(-1) * c.k_scale).max().item()
    score = abs(kw.get("scale") or d ** -0.5) * q.float().norm(dim=-1).max().item() * kmax
    soft = 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * score + 2.0 ** -20
    tol = unit * ref.abs() * 1.01 + soft * size + int(lens.max()) * 2.0 ** -30 * top + 2.0 ** -120
    assert torch.isfinite(o).all()
    worst = ((o.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, worst
    assert torch.equal(lref == -math.inf, lse == -math.inf)
    return o


def _queries(form, seed):
    d, P, H, G, B, n, T = FORMS[form]
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = _cache(B * -(-T // P), H, d, P, seed=seed)
    table = _table([T] * B, P, c.n_pages)
    return c, table, torch.randn(B, n, H * G, d, generator=g, device=DEV).bfloat16(), _i32([T - i % 9 for i in range(B)])


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


@pytest.mark.parametrize("P,d,H", [(16, 32, 1), (64, 128, 3), (32, 64, 16)])
@pytest.mark.parametrize("src,dst", [([0], [5]), ([3, 3, 1], [0, 2, 4]), ([0, 1, 2], [1, 2, 0]), ([4], [4]), ([], []),
                                     ([6], [0, 1, 2, 3])])
def test_copy_pages(P, d, H, src, dst):
    """As an assignment by index: every source is read first, one source serves many."""
    c = _cache(7, H, d, P, spread=2.0)
    want = _clone(c, "cpu")
    for t in (want.k.view(torch.uint8), want.v.view(torch.uint8), want.k_scale, want.v_scale):
        t[dst] = t[src]
    for kind in (torch.int64, torch.int32):
        got = _clone(c, DEV)
        got.copy_pages(torch.tensor(src, dtype=kind, device=DEV), torch.tensor(dst, dtype=kind, device=DEV))
        _same(got, want)
        got.check_errors()


def test_copy_pages_outside_the_pool_are_skipped_and_reported():
    """An id that a page table holds for no page (-1) must not become the last page."""
    c = _cache(4, 2, 64, 16)
    for src, dst in (([-1, 0], [1, 2]), ([1, 0], [4, 2]), ([0, 1 << 40], [2, 3]), ([0, 1], [2, -(1 << 40)])):
        before = _clone(c, "cpu")
        c.copy_pages(torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV))
        with pytest.raises(RuntimeError, match="out of range"):
            c.check_errors()
        before.copy_pages(torch.tensor([0]), torch.tensor([2]))
        _same(c, before)
        c.v_scale *= 2
    c.check_errors()


def test_a_page_table_beyond_32_bits_of_tokens_is_refused():
    """Before anything is launched: a length near 2^31 would overflow the kernels' counts of keys."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(2, 1, 32, 64)
    table = torch.zeros(1, (1 << 25) - 64, dtype=torch.int32, device=DEV)
    one, x = _i32([1]), torch.ones(1, 1, 1, 32, device=DEV, dtype=torch.bfloat16)
    for bad in (lambda: paged_attention(x, c, table, one), lambda: c.append(x, x, table, one),
                lambda: c.read(table, one, n=4)):
        with pytest.raises(RuntimeError, match="room"):
            bad()
    ok = table[:, :-1]
    c.append(x, x, ok, one)
    paged_attention(x, c, ok, one, max_len=64)
    c.read(ok, one, n=4)
    c.check_errors()


def _norm_ref(x, w, ang, dy):
    x, w = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True)) * w
    h = ang.shape[-1] // 2
    c, s = ang[:, None, :h].double(), ang[:, None, h:].double()
    y = torch.cat([y[..., :h] * c - y[..., h:] * s, y[..., :h] * s + y[..., h:] * c], -1)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy.double()))


@pytest.mark.parametrize("B,T,H", [(1, 1, 1), (1, 5, 3), (3, 37, 2), (70, 101, 5)])
@pytest.mark.parametrize("d", [32, 96, 128])
def test_rotary_without_eps(B, T, H, d):
    """eps = 0 with rows that are not zero, of any count: nothing of the rows that fill up a block reaches the sums. A
    position outside the table gives zeros, in the gradients too. 24 roundings of 2^-24 bound the chain of a row, whose
    gradient is a difference of terms of up to |dy| |w| sqrt(d) r each; sums of n products of some 16 each."""
    from primus_dlrm_b200.ops import rotary
    g = torch.Generator(device=DEV).manual_seed(T)
    x, dy = (torch.randn(B, T, H, d, generator=g, device=DEV) for _ in range(2))
    w = 1 + 0.3 * torch.randn(d, generator=g, device=DEV)
    table, pos = rotary.rope_table(T + 3, d, device=DEV), torch.arange(T, device=DEV)
    want = _norm_ref(x, w, table[pos], dy)
    leaf = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    y, _ = rotary.qk_norm_rope(leaf[0], None, leaf[1], None, table, pos, eps=0.0)
    got = (y.detach(), *torch.autograd.grad(y, leaf, dy))
    for a, b, size in zip(got, want, (16.0, 64.0, 16.0 * (B * T * H + 30))):
        assert torch.isfinite(a).all() and (a.double() - b).abs().max().item() <= 24 * 2.0 ** -24 * size
    out = pos.clone()
    out[T // 2] = T + 3
    y, _ = rotary.qk_norm_rope(leaf[0], None, leaf[1], None, table, out, eps=0.0)
    dx, dw = torch.autograd.grad(y, leaf, dy)
    keep = torch.arange(T, device=DEV) != T // 2
    assert (y[:, T // 2] == 0).all() and (dx[:, T // 2] == 0).all()
    assert torch.equal(y[:, keep], got[0][:, keep]) and torch.equal(dx[:, keep], got[1][:, keep])
    assert torch.isfinite(dw).all()
    assert rotary.rotary_error_code(DEV) == 1
    rotary._err_word(DEV).zero_()


@pytest.mark.parametrize("form", FORMS)
def test_value_scale_of_zero(form):
    """A page whose value scale is 0 holds zeros: it takes part in the softmax and adds nothing."""
    c, table, q, lens = _queries(form, 1)
    c.v_scale[table[:, 1].long()] = 0
    _check_rows(q, c, table, lens)
    c.v_scale.zero_()
    assert (_check_rows(q, c, table, lens, causal=False) == 0).all()


@pytest.mark.parametrize("form", FORMS)
def test_scores_of_large_magnitude(form):
    """Scores far below -1e30: the largest of them still takes the whole probability."""
    c, table, q, lens = _queries(form, 2)
    c.k.view(torch.uint8).fill_(0x38)                                # keys of 1.0 times their scale
    c.k_scale.fill_(2.0 ** 60)
    first = table[:, 0].long()
    c.k.view(torch.uint8)[first, :, 3] = 0x30                        # the fourth key of each sequence: 0.5
    q.fill_(-2.0 ** 60)
    q.view(torch.int16)[..., 0] ^= 1                                 # queries that are not all alike
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    o, lse = paged_attention(q, c, table, lens, return_lse=True, causal=False)
    G = q.shape[2] // c.n_kv_heads
    v = (c.v.view(torch.uint8)[first, :, 3].view(E4M3).float() * c.v_scale[first][..., None]).repeat_interleave(G, 1)
    assert torch.equal(o, v[:, None].expand(o.shape).to(o.dtype))    # an e4m3 code times 2^e is a bf16 number
    assert torch.isfinite(lse).all() and (lse < -1e30).all()
    c.check_errors()


@pytest.mark.parametrize("form", FORMS)
def test_values_near_the_largest(form):
    """Values whose sums over the keys would pass the largest 32-bit number."""
    c, table, q, lens = _queries(form, 3)
    c.v.view(torch.uint8)[:] &= 0x7F                                 # all of one sign, so that sums do not cancel
    c.v.copy_(c.v.float().clamp(min=240).to(E4M3))
    c.v_scale.fill_(2.0 ** 119)                                      # up to 448 * 2^119 = 2^127.8
    _check_rows(q, c, table, lens)
    c.v_scale.fill_(2.0 ** -100)                                     # and the smallest scale
    _check_rows(q, c, table, lens)


@pytest.mark.parametrize("step", [12, 26, 40, -26, 61])
@pytest.mark.parametrize("form", FORMS)
def test_pages_of_very_different_values(form, step):
    """Each page's values 2^step times those before: a row is as exact as the values that it sees allow, whatever the
    pages behind it hold."""
    c, table, q, lens = _queries(form, 4)
    for j in range(table.shape[1]):
        c.v_scale[table[:, j].long()] *= 2.0 ** (step * (j % 4) - (100 if step == 61 else 0))
    _check_rows(q, c, table, lens)
    _check_rows(q, c, table, lens, causal=False, scale=0.02)


@pytest.mark.parametrize("reach,step", [(40, 20), (60, 40), (70, 90), (50, 45)])
@pytest.mark.parametrize("form", FORMS)
def test_unlikely_keys_with_large_values(form, reach, step):
    """Keys of probability 2^-reach whose values are 2^step times the others', in the middle of a page's run: they count
    for what they are, be it nothing or nearly all."""
    c, table, q, lens = _queries(form, 5)
    d = q.shape[-1]
    c.k.view(torch.uint8)[:] = 0x38
    c.k_scale.fill_(1.0)
    page = table[:, 1].long()
    c.k.view(torch.uint8)[page] = 0xB8                               # -1
    c.v_scale[page] *= 2.0 ** step
    # q . k = +- reach / 2 in the log2 domain: each element reach ln 2 / (2 d scale)
    q = torch.full_like(q, reach * math.log(2) / (2 * d * d ** -0.5))
    _check_rows(q, c, table, lens)


@pytest.mark.parametrize("n,d,H", [(2, 32, 1), (2, 128, 2), (140, 32, 8), (140, 64, 8), (140, 128, 8)])
def test_rows_of_no_sequence_are_zeros(n, d, H):
    """Rows in front of the first and behind the last sequence, and those of a sequence longer than stated: zeros and
    -inf whatever the memory held, next to the results of the others."""
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    B = 40
    c = _cache(4, H, d, 16)
    table, lens = _i32([[0, 1, 2]] * B), _i32([40] * B)
    off = [3]
    for b in range(B):
        off.append(off[-1] + (n + 1 + b % 3 if b % 7 == 2 else n - b % 2))
    total = off[-1] + 5
    q = torch.randn(total, 2 * H, d, device=DEV).bfloat16()
    for lse_too in (True, False):
        junk = [torch.full_like(q, float("nan")), torch.full(q.shape[:2], float("nan"), device=DEV)]
        torch.cuda.synchronize()
        del junk                                                     # the next allocations find NaN
        out = paged_attention(q, c, table, lens, _i32(off), n, return_lse=lse_too)
        o = out[0] if lse_too else out
        with pytest.raises(RuntimeError, match="length"):
            c.check_errors()
        live = torch.zeros(total, dtype=torch.bool, device=DEV)
        for b in range(B):
            if b % 7 != 2:
                live[off[b]:off[b + 1]] = True
        assert (o[~live] == 0).all() and torch.isfinite(o).all()
        if lse_too:
            seen = torch.ones(total, dtype=torch.bool, device=DEV)       # rows that have keys
            for b in range(B):
                seen[off[b]:max(off[b], off[b + 1] - 40)] = False
            assert torch.equal((out[1] > -math.inf).all(1), live & seen) and torch.equal((out[1] > -math.inf).any(1), live & seen)
        # the others: within two roundings of bf16 and of the probabilities of a call without the long ones
        good = [b for b in range(B) if b % 7 != 2]
        cut = [0] + list(torch.tensor([off[b + 1] - off[b] for b in good]).cumsum(0))
        alone = paged_attention(q[live], c, table[good], lens[good], _i32(cut), n)
        c.check_errors()
        assert (o[live].float() - alone.float()).abs().max() <= 2.0 ** -6 * (c.v.float().abs().amax((1, 2, 3)) * c.v_scale.amax(1)).max()


def test_a_stated_most_of_zero_is_reported():
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(4, 1, 32, 16)
    before = _clone(c, DEV)
    x = torch.ones(3, 1, 32, device=DEV)
    c.append(x, x, _i32([[0]]), _i32([0]), _i32([0, 3]), 0)
    _same(c, before)
    with pytest.raises(RuntimeError, match="length"):
        c.check_errors()
    o = paged_attention(x.bfloat16(), c, _i32([[0]]), _i32([3]), _i32([0, 3]), 0)
    assert (o == 0).all()
    with pytest.raises(RuntimeError, match="length"):
        c.check_errors()
    c.append(x, x, _i32([[0]]), _i32([0]), _i32([0, 0]), 0)            # no tokens: nothing to report
    paged_attention(x.bfloat16(), c, _i32([[0]]), _i32([3]), _i32([0, 0]), 0)
    c.check_errors()


def test_tangents_are_refused():
    """Forward-mode derivatives do not go through the kernels: refused, not dropped."""
    import torch.autograd.forward_ad as fw
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    t, x = rope_table(4, 32, device=DEV), torch.randn(1, 4, 2, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    c = _cache(4, 2, 32, 16)
    with fw.dual_level():
        dual, dw, dt = (fw.make_dual(a, torch.ones_like(a)) for a in (x, w, t))
        for bad in (lambda: qk_norm_rope(dual, x, w, w, t), lambda: qk_norm_rope(x, dual, w, w, t),
                    lambda: qk_norm_rope(x, x, dw, w, t), lambda: qk_norm_rope(x, x, w, dw, t),
                    lambda: qk_norm_rope(x, x, w, w, dt)):
            with pytest.raises(RuntimeError, match="forward"):
                bad()
        qk_norm_rope(x, x, w, w, t)


def test_gradients_of_the_angles_are_refused():
    from primus_dlrm_b200.ops.rotary import qk_norm_rope, rope_table
    t, x = rope_table(4, 32, device=DEV).requires_grad_(), torch.randn(1, 4, 2, 32, device=DEV)
    with pytest.raises(RuntimeError, match="angle"):
        qk_norm_rope(x, x, None, None, t)
    with torch.no_grad():
        qk_norm_rope(x, x, None, None, t)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_has_no_gradient(n):
    """The output of a query that requires a gradient says so where the gradient is asked for."""
    import torch.autograd.forward_ad as fw
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    c = _cache(4, 2, 32, 16)
    table, lens = _i32([[0, 1, 2]]), _i32([45])
    q = torch.randn(1, n, 4, 32, device=DEV).bfloat16()
    want = paged_attention(q, c, table, lens)
    assert not want.requires_grad
    leaf = q.clone().requires_grad_()
    o, lse = paged_attention(leaf, c, table, lens, return_lse=True)
    assert torch.equal(o.detach(), want)
    for y in (o, lse):
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward(retain_graph=True)
    with torch.no_grad():
        assert not paged_attention(leaf, c, table, lens).requires_grad
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            paged_attention(fw.make_dual(q, torch.ones_like(q)), c, table, lens)


def test_training_after_inference_mode():
    """The angle table that a first call under inference mode built serves a training step too."""
    from test_onetrans_rotary import _model
    attn, x = _model("cuda", rotary=True, attention_impl="sdpa").blocks[0].attn, torch.randn(2, 30, 64, device=DEV)
    n_s = 30 - attn.n_ns
    with torch.inference_mode():
        attn(x, n_s, 20)
    attn(x, n_s, 20).sum().backward()
    assert attn.q_norm.weight.grad.abs().max() > 0


@pytest.mark.parametrize("q_len", [200, 77])
@pytest.mark.parametrize("impl,dtype,most", [("sdpa", torch.float32, 1e-4), ("fav4", torch.bfloat16, 0.06)])
def test_gradients_of_a_rotary_layer(impl, dtype, most, q_len):
    """Every parameter's gradient, the projection's among them, and the input's, against the CPU in 32 bits. 32 bits: sums
    of some 1600 products, 2^-24 each in random order, and differences that cancel by 10 or so; bf16: some eight roundings
    of 2^-8 on the way down and up again, that do not all point the same way."""
    from test_onetrans_rotary import _model
    gpu, cpu = (_model(d, rotary=True, attention_impl=impl).blocks[0].attn.train() for d in ("cuda", "cpu"))
    cpu.load_state_dict({k: v.cpu() for k, v in gpu.state_dict().items()})
    g = torch.Generator().manual_seed(q_len)
    x, dy = torch.randn(8, 200, 64, generator=g), torch.randn(8, q_len, 64, generator=g)
    grads = []
    for m, dev in ((gpu, "cuda"), (cpu, "cpu")):
        leaf = x.to(dev).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype != torch.float32 and dev == "cuda"):
            y = m(leaf.to(dtype if dev == "cuda" else torch.float32), 200 - m.n_ns, q_len)
        y.backward(dy.to(dev, y.dtype))
        grads.append({"x": leaf.grad, **{k: p.grad for k, p in m.named_parameters()}})
    assert {"s_qkv.weight", "ns_qkv_weight", "q_norm.weight", "k_norm.weight"} <= set(grads[0])
    for k, want in grads[1].items():
        got = grads[0][k].float().cpu()
        assert (got - want).norm() <= most * want.norm(), (k, ((got - want).norm() / want.norm()).item())
