"""Cases of the query/key norm with rotation, the 8-bit paged key/value cache and the attention over it.

Sizes follow the OneTrans configurations: 8 heads x 32 over 896 history + 16 candidate tokens, 16 heads x 64 over
1792 + 32 tokens, 6 heads x 64 over histories of 500 events; the head size of 128 with grouped heads is generic.
``run`` computes each operator in elementary torch operations in 32 bits, or (``own``) through the framework.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_THETA = 10000.0
_EPS = 1e-6
_MIN_EXP = -100          # the smallest scale of a page is 2^-100


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the next event of eight users: one token each, queries and keys of 8 heads x 32 (a call's latency)
        dict(name="rotary one token", op="rotary", batch=8, tokens=1, queries=1, heads=8, kv_heads=8, dim=32,
             rotary_dim=32, interleaved=False, dtype="bf16", backward=False),
        # a training step of the 8 x 32 model: 912 tokens, the second layer's 786 queries, forward and backward
        dict(name="rotary train 8x32", op="rotary", batch=256, tokens=912, queries=786, heads=8, kv_heads=8, dim=32,
             rotary_dim=32, interleaved=False, dtype="bf16", backward=True),
        # a training step at 6 x 64 with an odd batch and an odd history, pairs side by side, fp16
        dict(name="rotary train 6x64 odd", op="rotary", batch=37, tokens=517, queries=517, heads=6, kv_heads=6, dim=64,
             rotary_dim=64, interleaved=True, dtype="fp16", backward=True),
        # a prompt of grouped heads x 128 of which half the dims turn, in 32 bits
        dict(name="rotary grouped 128", op="rotary", batch=3, tokens=2049, queries=2049, heads=32, kv_heads=8, dim=128,
             rotary_dim=64, interleaved=False, dtype="fp32", backward=False),
        # one new event of 64 users with histories of very different lengths
        dict(name="append one token", op="append", seqs=64, held_lo=0, held_hi=1791, new_lo=1, new_hi=1, kv_heads=8,
             dim=32, page=32, dtype="bf16"),
        # the histories of 128 users enter the cache: 896 tokens each
        dict(name="append histories", op="append", seqs=128, held_lo=0, held_hi=0, new_lo=896, new_hi=896, kv_heads=8,
             dim=32, page=64, dtype="bf16"),
        # ragged pieces behind ragged histories: they begin and end inside pages
        dict(name="append ragged 128", op="append", seqs=48, held_lo=3, held_hi=2500, new_lo=1, new_hi=701, kv_heads=8,
             dim=128, page=16, dtype="fp16"),
        # one user's next event over a history of 897 (a call's latency)
        dict(name="attend one user", op="attend", seqs=1, queries_lo=1, queries_hi=1, held_lo=897, held_hi=897,
             shared=0, heads=8, kv_heads=8, dim=32, page=32, dtype="bf16"),
        # single tokens of 64 sequences, grouped heads x 128, lengths from short to 8191
        dict(name="attend tokens 128", op="attend", seqs=64, queries_lo=1, queries_hi=1, held_lo=300, held_hi=8191,
             shared=0, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # single tokens of three very long sequences: few rows, a long axis
        dict(name="attend tokens long", op="attend", seqs=3, queries_lo=1, queries_hi=1, held_lo=65537, held_hi=131071,
             shared=0, heads=16, kv_heads=4, dim=64, page=16, dtype="fp16"),
        # 1024 candidates of one user: 16 tokens each behind a history that they share
        dict(name="attend candidates", op="attend", seqs=1024, queries_lo=16, queries_hi=16, held_lo=912, held_hi=912,
             shared=896, heads=8, kv_heads=8, dim=32, page=64, dtype="bf16"),
        # whole histories of the 16 x 64 model as prompts, ragged up to its 1824 tokens
        dict(name="attend prompts 16x64", op="attend", seqs=12, queries_lo=911, queries_hi=1824, held_lo=911,
             held_hi=1824, shared=0, heads=16, kv_heads=16, dim=64, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; sizes are halved until it costs no more than the largest listed one."""
    op = rng.choice(["rotary", "append", "attend", "attend"])
    dim = rng.choice([32, 64, 128])
    if op == "rotary":
        tokens = _log(rng, 1, 2048)
        kv_heads = rng.choice([1, 2, 4, 6, 8, 16])
        c = dict(op=op, batch=_log(rng, 1, 512), tokens=tokens, queries=rng.choice([tokens, rng.randint(1, tokens)]),
                 heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads, dim=dim,
                 rotary_dim=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), backward=rng.random() < 0.5)
        while c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * dim > 1.1e8:
            c["batch"] = max(1, c["batch"] // 2)
            if c["batch"] == 1:
                c["tokens"] = max(1, c["tokens"] // 2)
                c["queries"] = min(c["queries"], c["tokens"])
        return c
    seqs = _log(rng, 1, 256)
    kv_heads = rng.choice([1, 2, 4, 6, 8, 16])
    page = rng.choice([16, 32, 64])
    if op == "append":
        held = rng.choice([0, _log(rng, 1, 8000)])
        new = rng.choice([1, _log(rng, 1, 1024)])
        c = dict(op=op, seqs=seqs, held_lo=held // rng.choice([1, 3]), held_hi=held,
                 new_lo=max(1, new // rng.choice([1, 4])), new_hi=new, kv_heads=kv_heads, dim=dim, page=page,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        while c["seqs"] > 1 and c["seqs"] * (c["held_hi"] + c["new_hi"]) * kv_heads * dim > 2.5e8:
            c["seqs"] //= 2
        return c
    if rng.random() < 0.5:
        q_hi = rng.choice([1, 1, 2, 5])
        held = _log(rng, max(1, q_hi), 60000)
    else:
        q_hi = _log(rng, 2, 1800)
        held = q_hi + rng.choice([0, _log(rng, 1, 4000)])
    q_lo = max(1, q_hi // rng.choice([1, 1, 3]))
    c = dict(op=op, seqs=seqs, queries_lo=q_lo, queries_hi=q_hi, held_lo=max(q_hi, held // rng.choice([1, 2, 8])),
             held_hi=held, shared=0, heads=kv_heads * rng.choice([1, 1, 2, 4, 5]), kv_heads=kv_heads, dim=dim, page=page,
             dtype=rng.choice(["bf16", "bf16", "fp16"]))
    # (padded) scores and expanded cache of the plain form, and the products of the largest listed case
    while c["seqs"] > 1 and (c["seqs"] * c["held_hi"] * kv_heads * dim > 3.5e8
                             or c["seqs"] * c["held_hi"] * c["heads"] * c["queries_hi"] > 4.5e8):
        c["seqs"] //= 2
    while c["held_hi"] * c["heads"] * c["queries_hi"] > 4.5e8:
        c["heads"] = c["kv_heads"] = 1
        c["held_hi"] //= 2
        c["held_lo"] = min(c["held_lo"], c["held_hi"])
        c["queries_hi"] = min(c["queries_hi"], c["held_lo"])
        c["queries_lo"] = min(c["queries_lo"], c["queries_hi"])
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, out of order."""
    step = next(s for s in (7919, 104729, 1299709, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(tokens in the cache before the call, new tokens or queries) of each sequence."""
    n = case["seqs"]
    held = _spread(case["held_lo"], case["held_hi"], n)
    if case["op"] == "append":
        return held, list(reversed(_spread(case["new_lo"], case["new_hi"], n)))
    return held, [min(h, q) for h, q in zip(held, reversed(_spread(case["queries_lo"], case["queries_hi"], n)))]


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    d = case["dim"]
    if case["op"] == "rotary":
        x = case["batch"] * (case["queries"] * case["heads"] + case["tokens"] * case["kv_heads"]) * d
        b, f = 2 * x * size + case["tokens"] * case["rotary_dim"] * 4 + 8 * d, 8 * x
        if case["backward"]:
            b, f = b + 3 * x * size + 8 * d, f + 14 * x
        return {"bytes": b, "flops": f}
    held, new = _lengths(case)
    h, p = case["kv_heads"], case["page"]
    if case["op"] == "append":
        touched = [(a + n - 1) // p - a // p + 1 for a, n in zip(held, new)]
        read = sum(a % p + n for a, n in zip(held, new))     # tokens of the touched pages, read back as values
        rows = len(held) * (max(new) + p)
        return {"bytes": 2 * h * (sum(new) * d * (size + 1) + sum(touched) * 4 + read * d + rows * d * 2),
                "flops": 2 * h * d * 10 * sum(new)}
    cached = sum(held) - (len(held) - 1) * case["shared"]
    pairs = sum(n * (a - n) + n * (n + 1) // 2 for a, n in zip(held, new))
    return {"bytes": 2 * cached * h * d + 2 * (-(-cached // p)) * h * 4 + 2 * sum(new) * case["heads"] * d * 2,
            "flops": 4 * pairs * case["heads"] * d}


# ---------------------------------------------------------------- what a program has in hand
def _angles(n_pos, rotary_dim, device):
    inv = _THETA ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], dim=1).float()


def _pow2_scale(amax):
    """The smallest power of two s (2^-100 at least) with amax / s <= 448 = 0.875 * 2^9."""
    f, e = torch.frexp(amax)
    e = torch.where(f > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, _MIN_EXP).clamp(min=_MIN_EXP))


def _pages(gen, n_pages, heads, page, dim, spread, device):
    """Pages as earlier calls left them: codes of normal values and each (page, head)'s scale."""
    codes = torch.empty(n_pages, heads, page, dim, dtype=_E4M3, device=device)
    scales = torch.empty(n_pages, heads, device=device)
    step = max(1, (1 << 27) // (heads * page * dim))
    for a in range(0, n_pages, step):
        x = torch.randn(min(step, n_pages - a), heads, page, dim, generator=gen, device=device)
        x = x * torch.exp(spread * torch.randn(x.shape[0], heads, 1, 1, generator=gen, device=device))
        s = _pow2_scale(x.abs().amax((2, 3)))
        scales[a:a + step] = s
        codes[a:a + step] = (x / s[..., None, None]).to(_E4M3)
    return codes, scales


def _table(gen, tokens, page, shared, device):
    """(page table [sequences, most pages], pages in all); the first shared // page pages are everybody's."""
    n = [-(-t // page) for t in tokens]
    both = shared // page
    total = both + sum(k - both for k in n)
    ids = torch.randperm(total + 3, generator=gen, device=device)[:total].int().cpu()
    table, at = torch.full((len(n), max(max(n), 1)), -1, dtype=torch.int32), both
    for i, k in enumerate(n):
        table[i, :both] = ids[:both]
        table[i, both:k] = ids[at:at + k - both]
        at += k - both
    return table.to(device), total + 3


def _offsets(new, device):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dt, d = _DTYPES[case["dtype"]], case["dim"]
    s = {"op": case["op"], "case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "rotary":
        B, T, Q, H, K = (case[k] for k in ("batch", "tokens", "queries", "heads", "kv_heads"))
        # as a projection leaves them: queries, keys and values of a token side by side
        qkv = torch.empty(B, T, (H + 2 * K) * d, dtype=dt, device=dev)
        for b in range(0, B, 64):
            qkv[b:b + 64] = (1.5 * randn(min(64, B - b), T, (H + 2 * K) * d)).to(dt)
        s["q"] = qkv[:, T - Q:, :H * d].unflatten(-1, (H, d))
        s["k"] = qkv[:, :, H * d:(H + K) * d].unflatten(-1, (K, d))
        s["q_weight"], s["k_weight"] = 1 + 0.2 * randn(d), 1 + 0.2 * randn(d)
        offset = int(torch.randint(0, 1000, (1,), generator=gen, device=dev))
        s["positions"] = torch.arange(T, device=dev, dtype=torch.int32) + offset
        s["table"] = _angles(T + 1000, case["rotary_dim"], dev)
        if case["backward"]:
            s["dq"], s["dk"] = randn(B, Q, H, d).to(dt), randn(B, T, K, d).to(dt)
        return s

    held, new = _lengths(case)
    K, page = case["kv_heads"], case["page"]
    after = [a + n for a, n in zip(held, new)] if case["op"] == "append" else held
    s["page_table"], n_pages = _table(gen, after, page, case.get("shared", 0), dev)
    k, ks = _pages(gen, n_pages, K, page, d, 0.1, dev)
    v, vs = _pages(gen, n_pages, K, page, d, 0.5, dev)
    s["kv"] = (k, v, ks, vs)
    s["lens"] = torch.tensor(held, dtype=torch.int32, device=dev)
    s["max_new"], s["max_len"] = max(new), max(held)
    s["uniform"] = min(new) == max(new)
    s["cu"] = _offsets(new, dev)
    N = sum(new)
    if case["op"] == "append":
        for name in ("new_k", "new_v"):
            s[name] = (randn(N, K, d) * torch.exp(0.5 * randn(N, 1, 1))).to(dt)
        s["k_weight"] = 1 + 0.2 * randn(d)
        s["table"] = _angles(max(after) + 1, d, dev)
        s["first"] = s["lens"] // page * page
        s["after"] = torch.tensor(after, dtype=torch.int32, device=dev)
        names = ("new_k", "new_v")
    else:
        s["q"] = (1.3 * randn(N, case["heads"], d)).to(dt)
        names = ("q",)
    if s["uniform"]:
        for name in names:
            s[name] = s[name].unflatten(0, (case["seqs"], max(new)))
    if own:
        from primus_dlrm_b200.ops.kv_cache import PagedKVCache
        s["cache"] = PagedKVCache.from_tensors(k, v, ks, vs)
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, interleaved):
    """x [..., heads, dim] by cos, sin [..., 1, rotary_dim / 2]."""
    h = cos.shape[-1]
    r, rest = x[..., :2 * h], x[..., 2 * h:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :h], r[..., h:])
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _norm_rotate(x, w, cos, sin, interleaved):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return _rotate(x * r * w, cos, sin, interleaved)


def _norm_rotate_grad(x, w, cos, sin, interleaved, dy):
    x, u = x.float(), _rotate(dy.float(), cos, -sin, interleaved)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xh = x * r
    g = u * w
    return r * (g - xh * (g * xh).mean(-1, keepdim=True)), (u * xh).sum((0, 1, 2))


def _rotary_plain(s):
    dt, il = s["q"].dtype, s["case"]["interleaved"]
    cs = s["table"][s["positions"].long()]
    cos, sin = cs.chunk(2, -1)
    cos, sin, Q = cos[:, None], sin[:, None], s["q"].shape[1]
    cq, sq = cos[-Q:], sin[-Q:]
    out = {"q": _norm_rotate(s["q"], s["q_weight"], cq, sq, il).to(dt),
           "k": _norm_rotate(s["k"], s["k_weight"], cos, sin, il).to(dt)}
    if s["case"]["backward"]:
        dq, dwq = _norm_rotate_grad(s["q"], s["q_weight"], cq, sq, il, s["dq"])
        dk, dwk = _norm_rotate_grad(s["k"], s["k_weight"], cos, sin, il, s["dk"])
        out |= {"dq": dq.to(dt), "dk": dk.to(dt), "dq_weight": dwq, "dk_weight": dwk}
    return out


def _rows(table, positions, page):
    """(page, row in it) of each position [sequences, n]; positions past the table go to its last page."""
    at = (positions // page).clamp(max=table.shape[1] - 1)
    return table.gather(1, at).long().clamp(min=0), positions % page


def _append_part(codes, scales, values, s, fresh, old, touched, page_of, token):
    """Puts `values` [N, heads, dim] (32 bits) into the pages of one of the two halves of the cache."""
    new = torch.where(fresh[..., None, None], values[token], 0.0)                      # [B, J, P, H, d]
    amax = new.abs().amax((2, 4))                                                       # [B, J, H]
    before = scales[page_of]
    has_old = old.any(-1)[..., None]
    scale = torch.where(has_old, torch.maximum(_pow2_scale(amax), before), _pow2_scale(amax))
    held = codes.view(torch.uint8)[page_of].view(_E4M3).float().transpose(2, 3) * before[:, :, None, :, None]
    x = torch.where(fresh[..., None, None], new, held) / scale[:, :, None, :, None]
    kept = codes.view(torch.uint8)[page_of].transpose(2, 3)
    x = torch.where((fresh | old)[..., None, None], x.to(_E4M3).view(torch.uint8), kept)
    codes.view(torch.uint8)[page_of[touched]] = x[touched].transpose(1, 2)
    scales[page_of[touched]] = scale[touched]


def _append_plain(s):
    page = s["case"]["page"]
    k, v, ks, vs = s["kv"]
    dev = k.device
    lens, n = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    new_k, new_v = s["new_k"], s["new_v"]
    if s["uniform"]:
        new_k, new_v = new_k.flatten(0, 1), new_v.flatten(0, 1)
    seq = torch.repeat_interleave(torch.arange(len(n), device=dev), n, output_size=new_k.shape[0])
    pos = lens[seq] + torch.arange(new_k.shape[0], device=dev) - s["cu"].long()[seq]
    cos, sin = s["table"][pos].chunk(2, -1)
    new_k = _norm_rotate(new_k, s["k_weight"], cos[:, None], sin[:, None], False)
    # the pages that new tokens can fall into, as [sequence, page, row]
    j = torch.arange((s["max_new"] + page - 2) // page + 1, device=dev)
    at = (lens // page)[:, None] + j
    place = at[..., None] * page + torch.arange(page, device=dev)
    i = place - lens[:, None, None]
    fresh = (i >= 0) & (i < n[:, None, None])
    touched = fresh.any(-1)
    old = (i < 0) & touched[..., None]
    token = torch.where(fresh, i + s["cu"].long()[:-1, None, None], 0)
    page_of = s["page_table"].gather(1, at.clamp(max=s["page_table"].shape[1] - 1)).long().clamp(min=0)
    _append_part(k, ks, new_k, s, fresh, old, touched, page_of, token)
    _append_part(v, vs, new_v.float(), s, fresh, old, touched, page_of, token)
    # the touched pages' tokens as the values that they stand for
    where = s["first"].long()[:, None] + torch.arange(s["max_new"] + page, device=dev)
    p, r = _rows(s["page_table"], where, page)
    there = (where < (lens + n)[:, None])[..., None, None]
    out = {}
    for name, c, f in (("k", k, ks), ("v", v, vs)):
        x = c.view(torch.uint8)[p, :, r].view(_E4M3).float() * f[p][..., None]
        out[name] = torch.where(there, x, 0.0).to(torch.bfloat16)
    return out


def _attend_plain(s):
    k, v, ks, vs = s["kv"]
    page, H, d = s["case"]["page"], s["case"]["heads"], s["case"]["dim"]
    K, dev = k.shape[1], k.device
    G, q = H // K, s["q"]
    lens, n = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    B, most = len(n), s["max_new"]
    i = torch.arange(most, device=dev)
    if not s["uniform"]:
        q = q[(s["cu"].long()[:-1, None] + i).clamp(max=q.shape[0] - 1)]               # padded to [B, most, H, d]
    ids = s["page_table"].long().clamp(min=0)
    L = ids.shape[1] * page
    kf = (k.view(torch.uint8)[ids].view(_E4M3).float() * ks[ids][..., None, None]).transpose(1, 2).reshape(B, K, L, d)
    vf = (v.view(torch.uint8)[ids].view(_E4M3).float() * vs[ids][..., None, None]).transpose(1, 2).reshape(B, K, L, d)
    q = q.float().unflatten(2, (K, G)).permute(0, 2, 1, 3, 4).reshape(B, K, most * G, d)
    w = (q @ kf.transpose(2, 3)) * d ** -0.5
    last = (lens - n)[:, None] + i                                                       # the last key of each query
    last = torch.where(i < n[:, None], last, -1).repeat_interleave(G, 1)
    w = w.masked_fill(torch.arange(L, device=dev) > last[:, None, :, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e30))
    total = w.sum(-1, keepdim=True)
    vf = vf * (torch.arange(L, device=dev) < lens[:, None])[:, None, :, None]
    o = (w @ vf) / torch.where(total > 0, total, 1.0)
    o = o.unflatten(2, (most, G)).permute(0, 2, 1, 3, 4).reshape(B, most, H, d)
    if not s["uniform"]:
        seq = torch.repeat_interleave(torch.arange(B, device=dev), n, output_size=s["q"].shape[0])
        o = o[seq, torch.arange(s["q"].shape[0], device=dev) - s["cu"].long()[seq]]
    return o.to(s["q"].dtype)


# ---------------------------------------------------------------- through the framework
def _rotary_own(s):
    from primus_dlrm_b200.ops.rotary import qk_norm_rope
    il = s["case"]["interleaved"]
    if not s["case"]["backward"]:
        q, k = qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], s["positions"], eps=_EPS,
                            interleaved=il)
        return {"q": q, "k": k}
    leaf = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["q_weight"], s["k_weight"])]
    q, k = qk_norm_rope(*leaf, s["table"], s["positions"], eps=_EPS, interleaved=il)
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaf, (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dq_weight": dwq, "dk_weight": dwk}


def _append_own(s):
    cu = None if s["uniform"] else s["cu"]
    s["cache"].append(s["new_k"], s["new_v"], s["page_table"], s["lens"], cu, s["max_new"], k_weight=s["k_weight"],
                      norm_eps=_EPS, rope=s["table"])
    k, v = s["cache"].read(s["page_table"], s["after"], s["first"], s["max_new"] + s["case"]["page"])
    return {"k": k, "v": v}


def _attend_own(s):
    from primus_dlrm_b200.ops.kv_cache import paged_attention
    cu = None if s["uniform"] else s["cu"]
    return paged_attention(s["q"], s["cache"], s["page_table"], s["lens"], cu, s["max_new"], max_len=s["max_len"])


def run(state):
    op = state["op"]
    if own:
        return (_rotary_own if op == "rotary" else _append_own if op == "append" else _attend_own)(state)
    return (_rotary_plain if op == "rotary" else _append_plain if op == "append" else _attend_plain)(state)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(x, w):
    x = x.double()
    return x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * w.double()


def _exact_turn(x, table, interleaved, back=False):
    """Pairs as complex numbers times exp(i angle) (or exp(-i angle)): x [n, heads, dim], table [n, rotary_dim]."""
    h = table.shape[-1] // 2
    z = torch.complex(table[:, :h].double(), table[:, h:].double())[:, None]
    z = z.conj() if back else z
    y = x.clone()
    if interleaved:
        t = torch.complex(x[..., 0:2 * h:2].contiguous(), x[..., 1:2 * h:2].contiguous()) * z
        y[..., 0:2 * h:2], y[..., 1:2 * h:2] = t.real, t.imag
    else:
        t = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous()) * z
        y[..., :h], y[..., h:2 * h] = t.real, t.imag
    return y


def _exact_rotary(s):
    il, Q = s["case"]["interleaved"], s["q"].shape[1]
    table = s["table"][s["positions"].long()]
    out = {}
    for name, x, w, t in (("q", s["q"], s["q_weight"], table[-Q:]), ("k", s["k"], s["k_weight"], table)):
        y, dx = torch.empty(x.shape, dtype=torch.float64, device=x.device), torch.empty(x.shape, dtype=torch.float64, device=x.device)
        dw = torch.zeros(x.shape[-1], dtype=torch.float64, device=x.device)
        for b in range(x.shape[0]):
            y[b] = _exact_turn(_exact_norm(x[b], w), t, il)
            if s["case"]["backward"]:
                xd, u = x[b].double(), _exact_turn(s["d" + name][b].double(), t, il, back=True)
                m = torch.sqrt((xd ** 2).sum(-1, keepdim=True) / xd.shape[-1] + _EPS)
                g = u * w.double()
                dx[b] = g / m - xd * (g * xd).sum(-1, keepdim=True) / (xd.shape[-1] * m ** 3)
                dw += (u * xd / m).sum((0, 1))
        out[name] = y
        if s["case"]["backward"]:
            out["d" + name], out["d" + name + "_weight"] = dx, dw
    return out


def _exact_append(s, held, new):
    page = s["case"]["page"]
    table, at = s["page_table"].tolist(), 0
    out = {n: torch.zeros(len(held), s["max_new"] + page, *s["kv"][0].shape[1::2], dtype=torch.float64, device="cuda")
           for n in ("k", "v")}
    for b, (a, n) in enumerate(zip(held, new)):
        for name, c, f in (("k", s["kv"][0], s["kv"][2]), ("v", s["kv"][1], s["kv"][3])):
            x = s["new_" + name].reshape(-1, *s["new_" + name].shape[-2:])[at:at + n]
            x = _exact_turn(_exact_norm(x, s["k_weight"]), s["table"][a:a + n], False) if name == "k" else x.double()
            start, old = a % page, table[b][a // page]
            if start:
                x = torch.cat([c[old, :, :start].double().transpose(0, 1) * f[old].double()[:, None], x])
            pages = -(-x.shape[0] // page)
            full = torch.zeros(pages * page, *x.shape[1:], dtype=torch.float64, device=x.device)
            full[:x.shape[0]] = x
            full = full.unflatten(0, (pages, page))
            mine = full.clone()
            mine[0, :start] = 0                                     # an old row does not raise its own page's scale
            scale = torch.exp2(torch.ceil(torch.log2(mine.abs().amax((1, 3)) / 448)).clamp(min=_MIN_EXP))
            if start:
                scale[0] = torch.maximum(scale[0], f[old].double())
            code = (full / scale[:, None, :, None]).to(_E4M3).double()
            out[name][b, :x.shape[0]] = (code * scale[:, None, :, None]).flatten(0, 1)[:x.shape[0]]
        at += n
    return out


def _exact_attend(s, held, new):
    page, H, d = s["case"]["page"], s["case"]["heads"], s["case"]["dim"]
    k, v, ks, vs = s["kv"]
    q, out, at = s["q"].reshape(-1, H, d), [], 0
    G = H // k.shape[1]
    for b, (a, n) in enumerate(zip(held, new)):
        ids = s["page_table"][b, :-(-a // page)].long()
        kd, vd = ((c[ids].double() * f[ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :a]
                  for c, f in ((k, ks), (v, vs)))
        qd = q[at:at + n].double().transpose(0, 1)
        sees = torch.arange(a, device=q.device) <= (a - n + torch.arange(n, device=q.device))[:, None]
        o = torch.empty(H, n, d, dtype=torch.float64, device=q.device)
        for h in range(H):
            w = (qd[h] @ kd[h // G].T / math.sqrt(d)).masked_fill(~sees, -math.inf)
            o[h] = torch.softmax(w, -1) @ vd[h // G]
        out.append(o.transpose(0, 1))
        at += n
    return torch.cat(out).reshape(s["q"].shape)


def exact(case, seed):
    if case["op"] == "attend" and case["seqs"] * case["heads"] > 8192 and case["shared"] == 0:
        return None                                                 # over about 20 seconds
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s)
    held, new = _lengths(case)
    return _exact_append(s, held, new) if case["op"] == "append" else _exact_attend(s, held, new)
