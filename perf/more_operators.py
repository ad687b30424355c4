"""Cases of the 8-bit integer products and of the training layers that keep their activations in 8 bits.

Sizes follow the OneTrans configurations (256 wide with 16 NS tokens over 896 events, 384 wide over 500 events, 1024
wide with 32 NS tokens over 1792 events; FFNs four times as wide), with odd sizes and batches among them.
``run`` computes each operator in elementary torch operations in 32 bits, or (``own``) through the framework.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 32              # values that share a power-of-two scale


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one token through a wide up projection (a call's latency)
        dict(name="int8 one token", op="linear", rows=1, groups=1, inner=1024, outer=4096, bias=True, act="gelu",
             residual=False, dtype="bf16"),
        # the 16 NS tokens of one candidate through a narrow projection
        dict(name="int8 16 tokens narrow", op="linear", rows=16, groups=1, inner=256, outer=768, bias=False, act="",
             residual=False, dtype="bf16"),
        # the next token of 96 users through a down projection, added to the residual stream
        dict(name="int8 96 tokens down", op="linear", rows=96, groups=1, inner=4096, outer=1024, bias=False, act="",
             residual=True, dtype="bf16"),
        # 1024 candidates of 16 NS tokens each, a weight of its own for each token
        dict(name="int8 candidates", op="linear", rows=1024, groups=16, inner=256, outer=1024, bias=False, act="gelu",
             residual=False, dtype="bf16"),
        # histories as prompts: nine of 1792 events and a piece
        dict(name="int8 prompts", op="linear", rows=16417, groups=1, inner=1024, outer=4096, bias=False, act="gelu",
             residual=False, dtype="bf16"),
        # an odd layer in 32 bits: neither dim a multiple of 16
        dict(name="int8 odd", op="linear", rows=2069, groups=1, inner=333, outer=1001, bias=True, act="relu",
             residual=False, dtype="fp32"),
        # the saved input of a training step's projection, and back
        dict(name="pack 256 wide", op="pack", rows=233472, width=256, dtype="bf16"),
        # odd rows whose last block is short, in 32 bits
        dict(name="pack odd", op="pack", rows=7919, width=1001, dtype="fp32"),
        # a training step's QKV projection of the 256 wide model: 912 tokens of 128 samples, forward and backward
        dict(name="projection 256", op="projection", batch=128, tokens=912, ns=16, inner=256, outer=768),
        # the 384 wide model with an odd batch and an odd history
        dict(name="projection 384 odd", op="projection", batch=37, tokens=517, ns=16, inner=384, outer=1152),
        # a training step's FFN of the 256 wide model, the second layer's 786 rows
        dict(name="ffn 256", op="ffn", batch=128, tokens=786, ns=16, inner=256, outer=1024),
        # a training step's FFN of the 1024 wide model, an odd batch
        dict(name="ffn 1024", op="ffn", batch=7, tokens=1312, ns=32, inner=1024, outer=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges; its rows are halved until it costs no more than the largest listed one."""
    op = rng.choice(["linear", "linear", "linear", "pack", "projection", "ffn"])
    if op == "linear":
        groups = rng.choice([1, 1, 1, 8, 16, 32])
        c = dict(op=op, rows=_log(rng, 1, 32768), groups=groups, inner=_log(rng, 64, 4096), outer=_log(rng, 64, 4096),
                 bias=rng.random() < 0.5, act=rng.choice(["", "gelu", "relu"]), residual=rng.random() < 0.3,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if rng.random() < 0.6:
            c["inner"], c["outer"] = -(-c["inner"] // 64) * 64, -(-c["outer"] // 64) * 64
        while c["rows"] > 1 and c["rows"] * groups * max(c["inner"] * c["outer"] / 6.8e10,
                                                         max(c["inner"], c["outer"]) / 1.3e8) > 1:
            c["rows"] //= 2
        return c
    if op == "pack":
        c = dict(op=op, rows=_log(rng, 1, 262144), width=_log(rng, 1, 4096),
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        while c["rows"] * c["width"] > 6e7:
            c["rows"] //= 2
        return c
    inner = 64 * rng.randint(1, 16)
    outer = 4 * inner if op == "ffn" else 64 * rng.randint(1, 48)
    ns = rng.choice([0, 8, 16, 32])
    c = dict(op=op, batch=_log(rng, 1, 128), tokens=max(ns, 1) + _log(rng, 1, 1792), ns=ns, inner=inner, outer=outer)
    while c["batch"] > 1 and c["batch"] * c["tokens"] * max(inner * outer / 3.8e10, outer / 1.0e8) > 1:
        c["batch"] //= 2
    return c


def work(case):
    size = 4 if case.get("dtype") == "fp32" else 2
    if case["op"] == "pack":
        n, b = case["rows"] * case["width"], case["rows"] * -(-case["width"] // _BLOCK)
        return {"bytes": 2 * (n * (size + 1) + b), "flops": 5 * n}
    k, n = case["inner"], case["outer"]
    if case["op"] == "linear":
        m, g = case["rows"] * case["groups"], case["groups"]
        b = m * k * size + m * n * size * (2 if case["residual"] else 1) + g * n * (k + 4) + (4 * n if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * n * k}
    m, w = case["batch"] * case["tokens"], (1 + case["ns"]) * k * n
    eighths = 33 / 32                                        # a saved value's bytes
    if case["op"] == "projection":                           # x, y, dy, dx, x saved and loaded, W, dW
        return {"bytes": m * (4 * k + 4 * n + 2 * k * eighths) + 2 * 2 * w, "flops": 6 * m * n * k}
    # x, z, y, dy, dx, x and the pre-activation saved and loaded, both weights and their gradients
    return {"bytes": m * (10 * k + 2 * (k + n) * eighths) + 2 * 2 * 2 * w, "flops": 12 * m * n * k}


# ---------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def filled(rows, width, dt, spread):
        """Rows of normal values of their own sizes, a few channels larger than the others."""
        out = torch.empty(rows, width, dtype=dt, device=dev)
        channel = torch.exp(0.5 * randn(width))
        for a in range(0, rows, 65536):
            n = min(65536, rows - a)
            out[a:a + n] = randn(n, width) * channel * torch.exp(spread * randn(n, 1))
        return out

    s = {"op": case["op"], "case": case}
    if case["op"] == "pack":
        s["x"] = filled(case["rows"], case["width"], _DTYPES[case["dtype"]], 1.0)
        return s
    k, n = case["inner"], case["outer"]
    if case["op"] == "linear":
        dt, m, g = _DTYPES[case["dtype"]], case["rows"], case["groups"]
        s["x"] = filled(m * g, k, dt, 0.5)
        w = randn(g, n, k) / math.sqrt(k)
        s["scale"] = w.abs().amax(-1) / 127
        s["codes"] = torch.round(w / s["scale"][..., None]).clamp(-127, 127).to(torch.int8)
        s["bias"] = 0.2 * randn(n) if case["bias"] else None
        s["residual"] = randn(m * g, n).to(dt) if case["residual"] else None
        if g > 1:                                            # [candidates, tokens, inner], a weight for each token
            s["x"] = s["x"].view(m, g, k)
            s["residual"] = s["residual"].view(m, g, n) if case["residual"] else None
        else:
            s["codes"], s["scale"] = s["codes"][0], s["scale"][0]
        if own:
            from primus_dlrm_b200.ops.int8 import Int8Weight
            s["weight"] = Int8Weight.from_tensors(s["codes"], s["scale"])
        return s
    b, t, ns = case["batch"], case["tokens"], case["ns"]

    def weight(o, i):
        return ((randn(o, i) / math.sqrt(i)).bfloat16(), (randn(ns, o, i) / math.sqrt(i)).bfloat16())

    s["x"] = filled(b * t, k, torch.bfloat16, 0.3).view(b, t, k)
    s["w"], s["wn"] = weight(n, k)
    if case["op"] == "ffn":
        s["z"] = filled(b * t, k, torch.bfloat16, 0.3).view(b, t, k)
        s["w2"], s["wn2"] = weight(k, n)
    s["dy"] = filled(b * t, k if case["op"] == "ffn" else n, torch.bfloat16, 0.3).view(b, t, -1)
    return s


# ---------------------------------------------------------------- plain forms
def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))


def _gelu_grad(x):
    return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def _linear_plain(s):
    x, w, t = s["x"].float(), s["codes"].float(), s["scale"]
    sx = (x.abs().amax(-1, keepdim=True) / 127).clamp(min=2.0 ** -126)
    a = torch.round(x * (1 / sx))
    if w.dim() == 3:
        y = (a.transpose(0, 1) @ w.transpose(1, 2)).transpose(0, 1)
    else:
        y = a @ w.t()
    y = y * (sx * t)
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    y = _gelu(y) if act == "gelu" else y.clamp(min=0) if act == "relu" else y
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _pack(x, top):
    """(codes, bytes of the scales' exponents, values) of x [rows, width] in 32 bits; `top`: the largest scale byte."""
    rows, width = x.shape
    blocks = -(-width // _BLOCK)
    if width < blocks * _BLOCK:
        x = torch.cat([x, x.new_zeros(rows, blocks * _BLOCK - width)], 1)
    x = x.view(rows, blocks, _BLOCK)
    f, e = torch.frexp(x.abs().amax(-1))                     # amax = f 2^e, 0.5 <= f < 1
    e = torch.where(f > 127 / 128, e - 6, e - 7)             # the least power with amax <= 127 * 2^e
    e = torch.where(f > 0, e, -126).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(f), e)[..., None]
    most = torch.where(e + 127 == top, 63.0, 127.0)[..., None]
    codes = torch.minimum(torch.maximum(torch.round(x / scale), -most), most)
    flat = lambda v: v.reshape(rows, blocks * _BLOCK)[:, :width]  # noqa: E731
    return flat(codes).to(torch.int8), (e + 127).to(torch.uint8), flat(codes * scale)


def _top(dtype):
    """Byte of the scale whose code 64 would be past the type's largest value."""
    return 10 + 127 if dtype == torch.float16 else 122 + 127


def _pack_plain(s):
    codes, exponents, values = _pack(s["x"].float(), _top(s["x"].dtype))
    return {"codes": codes, "exponents": exponents, "values": values.to(s["x"].dtype)}


def _saved(x):
    return _pack(x.reshape(-1, x.shape[-1]), _top(torch.float32))[2].view(x.shape)


def _mixed(x, w, wn):
    """Rows x [B, T, K] by w [N, K], the last rows of each sample by their own wn [ns, N, K]."""
    y, ns = x @ w.t(), wn.shape[0]
    if ns:
        y[:, -ns:] = (x[:, -ns:].transpose(0, 1) @ wn.transpose(1, 2)).transpose(0, 1)
    return y


def _mixed_grads(dy, x, wn):
    """Gradients of w and wn."""
    ns, s = wn.shape[0], x.shape[1] - wn.shape[0]
    dw = dy[:, :s].reshape(-1, dy.shape[-1]).t() @ x[:, :s].reshape(-1, x.shape[-1])
    return dw, dy[:, s:].permute(1, 2, 0) @ x[:, s:].transpose(0, 1)


def _projection_plain(s):
    x, w, wn, dy = (s[k].float() for k in ("x", "w", "wn", "dy"))
    y = _mixed(x, w, wn)
    dx = _mixed(dy, w.t(), wn.transpose(1, 2))
    dw, dwn = _mixed_grads(dy, _saved(x), wn)
    return {k: v.bfloat16() for k, v in dict(y=y, dx=dx, dw=dw, dwn=dwn).items()}


def _ffn_plain(s):
    x, z, w1, wn1, w2, wn2, dy = (s[k].float() for k in ("x", "z", "w", "wn", "w2", "wn2", "dy"))
    p = _mixed(x, w1, wn1)
    y = z + _mixed(_gelu(p), w2, wn2)
    p = _saved(p)
    dp = _mixed(dy, w2.t(), wn2.transpose(1, 2)) * _gelu_grad(p)
    dw2, dwn2 = _mixed_grads(dy, _gelu(p), wn2)
    dw1, dwn1 = _mixed_grads(dp, _saved(x), wn1)
    dx = _mixed(dp, w1.t(), wn1.transpose(1, 2))
    out = dict(y=y, dx=dx, dz=dy, dw1=dw1, dwn1=dwn1, dw2=dw2, dwn2=dwn2)
    return {k: v.bfloat16() for k, v in out.items()}


# ---------------------------------------------------------------- through the framework
def _linear_own(s):
    from primus_dlrm_b200.ops.int8 import int8_linear
    return int8_linear(s["x"], s["weight"], s["bias"], act=s["case"]["act"] or None, residual=s["residual"])


def _pack_own(s):
    from primus_dlrm_b200.ops.saved8 import load8, save8
    saved = save8(s["x"])
    return {"codes": saved.codes, "exponents": saved.exponents, "values": load8(saved)}


def _projection_own(s):
    from primus_dlrm_b200.ops import dense
    leaf = [s[k].detach().requires_grad_() for k in ("x", "w", "wn")]
    y = dense.mixed_linear(leaf[0], s["x"].shape[1] - s["wn"].shape[0], leaf[1], leaf[2], save8=True)
    dx, dw, dwn = torch.autograd.grad(y, leaf, s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "dwn": dwn}


def _ffn_own(s):
    from primus_dlrm_b200.ops import dense
    leaf = [s[k].detach().requires_grad_() for k in ("x", "z", "w", "w2", "wn", "wn2")]
    y = dense.mixed_ffn(leaf[0], leaf[1], s["x"].shape[1] - s["wn"].shape[0], *leaf[2:], save8=True)
    dx, dz, dw1, dw2, dwn1, dwn2 = torch.autograd.grad(y, leaf, s["dy"])
    return {"y": y.detach(), "dx": dx, "dz": dz, "dw1": dw1, "dwn1": dwn1, "dw2": dw2, "dwn2": dwn2}


def run(state):
    name = state["op"]
    if own:
        return {"linear": _linear_own, "pack": _pack_own, "projection": _projection_own, "ffn": _ffn_own}[name](state)
    return {"linear": _linear_plain, "pack": _pack_plain, "projection": _projection_plain, "ffn": _ffn_plain}[name](state)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_linear(s):
    case = s["case"]
    x, w, t = s["x"].double(), s["codes"].double(), s["scale"].double()
    # a token's scale, its reciprocal and the product that a code is nearest to are 32-bit numbers by definition
    sx = torch.clamp(s["x"].float().abs().max(-1, keepdim=True).values / 127, min=2.0 ** -126)
    a = torch.round(s["x"].float() * torch.reciprocal(sx)).double()
    y = torch.einsum("mk,nk->mn", a, w) if w.dim() == 2 else torch.einsum("mgk,gnk->mgn", a, w)
    y = y * sx.double() * t
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "gelu":
        y = torch.special.ndtr(y) * y
    elif case["act"] == "relu":
        y = torch.relu(y)
    return y + s["residual"].double() if s["residual"] is not None else y


def _exact_values(x):
    """What the 8-bit form of x (64 bits, last dim) stands for: the whole number of steps nearest to each value."""
    pad = -x.shape[-1] % _BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, _BLOCK))
    amax = b.abs().max(-1, keepdim=True).values
    step = torch.exp2(torch.ceil(torch.log2(amax / 127)))
    step = torch.where(amax > 127 * step, 2 * step, torch.where(amax <= 127 * step / 2, step / 2, step))   # log2's rounding
    step = torch.where(amax > 0, step, 1.0).clamp(min=2.0 ** -126)
    return (torch.round(b / step) * step).flatten(-2)[..., :x.shape[-1]]


def _exact_rows(x, w, wn):
    s = x.shape[1] - wn.shape[0]
    return torch.cat([torch.einsum("btk,nk->btn", x[:, :s], w), torch.einsum("btk,tnk->btn", x[:, s:], wn)], 1)


def _exact_weights(dy, x, ns):
    s = x.shape[1] - ns
    return (torch.einsum("btn,btk->nk", dy[:, :s], x[:, :s]), torch.einsum("btn,btk->tnk", dy[:, s:], x[:, s:]))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s)
    if case["op"] == "pack":
        return {"codes": None, "exponents": None, "values": _exact_values(s["x"].double())}
    x, w, wn, dy = (s[k].double() for k in ("x", "w", "wn", "dy"))
    ns = wn.shape[0]
    if case["op"] == "projection":
        dw, dwn = _exact_weights(dy, _exact_values(x), ns)
        return {"y": _exact_rows(x, w, wn), "dx": _exact_rows(dy, w.mT, wn.mT), "dw": dw, "dwn": dwn}
    w2, wn2 = s["w2"].double(), s["wn2"].double()
    p = _exact_rows(x, w, wn)
    y = s["z"].double() + _exact_rows(p * torch.special.ndtr(p), w2, wn2)
    p = _exact_values(p)
    h = p * torch.special.ndtr(p)
    dp = _exact_rows(dy, w2.mT, wn2.mT) * (torch.special.ndtr(p) + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi))
    dw2, dwn2 = _exact_weights(dy, h, ns)
    dw1, dwn1 = _exact_weights(dp, _exact_values(x), ns)
    return {"y": y, "dx": _exact_rows(dp, w.mT, wn.mT), "dz": dy, "dw1": dw1, "dwn1": dwn1, "dw2": dw2, "dwn2": dwn2}
