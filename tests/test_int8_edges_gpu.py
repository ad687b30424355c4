"""Products of 8-bit integers and layers with activations in 8 bits, where they meet values and calls at the edge."""
import math

import pytest
import torch

from primus_dlrm_b200.ops import dense
from primus_dlrm_b200.ops.int8 import Int8Weight, _linear_ref, int8_linear, quantize_rows
from primus_dlrm_b200.ops.saved8 import load8, save8

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_gelu_of_minus_infinity(rows, dtype):
    """GELU of a bias of minus infinity, and of a sum that overflows to it, is 0 in every form of the product (chosen by the
    rows), beside channels without a number too; NaN stays NaN and plus infinity stays."""
    g = _gen(rows)
    codes = torch.randint(-127, 128, (300, 256), generator=g, device=DEV, dtype=torch.int8)
    scale = torch.full((300,), 1e-6, device=DEV)
    codes[[3, 70]] = 127
    scale[[3, 70]] = 1e33                                    # 127 * 127 * 256 * (1e4 / 127) * 1e33 passes every type
    scale[4] = math.nan
    bias = torch.zeros(300, device=DEV)
    bias[[7, 133, 299]] = -math.inf
    w = Int8Weight.from_tensors(codes, scale)
    sign = torch.where(torch.arange(rows, device=DEV) % 2 == 0, -1.0, 1.0)[:, None]
    x = (sign * 1e4).expand(rows, 256).to(dtype)
    for b in (bias, None):
        y, ref = int8_linear(x, w, b, act="gelu"), _linear_ref(x, w, b, "gelu", None)
        assert y[:, 4].isnan().all() and torch.equal(y.isnan(), ref.isnan())
        low = (sign < 0).expand(rows, 1)
        for c in (3, 70):
            assert torch.equal(y[:, c:c + 1], torch.where(low, 0.0, math.inf).to(dtype))
        if b is not None:
            assert y[:, [7, 133, 299]].eq(0).all()
        assert torch.equal(y.isinf(), ref.isinf())


def test_row_codes_refuse_tangents():
    from torch.autograd import forward_ad
    x = torch.randn(4, 20, device=DEV)
    with forward_ad.dual_level():
        for bad in (lambda t: quantize_rows(t), lambda t: Int8Weight.from_float(t)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                bad(forward_ad.make_dual(x, x))


def test_error_word_follows_the_current_stream():
    """The code is that of the calls before it on the current stream, a stream of its own too; and 0 on a fresh word."""
    from primus_dlrm_b200.ops.int8 import _err_word, int8_error_code
    assert int8_error_code(DEV) == 0
    word, side = _err_word(DEV), torch.cuda.Stream()
    assert word.shape == (1,) and word.dtype == torch.int32 and not word.is_inference()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                    # some 10 ms
            word.fill_(2)
            assert int8_error_code(DEV) == 2
    finally:
        word.zero_()
    assert int8_error_code(DEV) == 0


@pytest.mark.parametrize("kv_cache", [None, "fp8"])
def test_scoring_reports_a_product_that_gave_up(kv_cache):
    from primus_dlrm_b200.ops.int8 import _err_word
    from test_models_cpu import _batch
    from test_onetrans_rotary import _model, _split
    model = _model(DEV, rotary=True, attention_impl="fav4")
    user, cand, _ = _split({k: v.cuda() for k, v in _batch(B=9, L=40, windows=2, seed=5).items()}, 9)
    w8 = model.int8_weights()
    want = model.score_candidates(user, cand, "listen_plus", kv_cache=kv_cache, weights=w8)
    _err_word(DEV).fill_(2)
    with pytest.raises(RuntimeError, match="int8_linear: a bounded wait"):
        model.score_candidates(user, cand, "listen_plus", kv_cache=kv_cache, weights=w8)
    assert torch.equal(model.score_candidates(user, cand, "listen_plus", kv_cache=kv_cache, weights=w8), want)


@pytest.mark.parametrize("D,F_", [(64, 128), (40, 72)])
@pytest.mark.parametrize("dtype,ztype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_layers_under_autocast(dtype, ztype, D, F_):
    """Output types are those of the 16-bit layers. Values differ by the roundings to bf16 (2^-8) of pre-activation, GELU,
    result and sum, at other places: 2^-6 of the output's size; gradients by those and the 8-bit values' (0.04 together)."""
    g = _gen(1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, z = r(2, 9, D).to(dtype), r(2, 9, D).to(ztype)
    leaves = [t.requires_grad_() for t in (x, z, r(F_, D) / D ** 0.5, r(D, F_) / F_ ** 0.5, r(3, F_, D) / D ** 0.5,
                                           r(3, D, F_) / F_ ** 0.5)]
    x, z, w1, w2, wn1, wn2 = leaves
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for act in (None, "gelu"):
            a, b = (dense.mixed_linear(x, 6, w1, wn1, act=act, save8=s) for s in (False, True))
            assert a.dtype == b.dtype and (a - b).norm() <= 2.0 ** -6 * a.norm()
        a = z + dense.mixed_linear(dense.mixed_linear(x, 6, w1, wn1, act="gelu"), 6, w2, wn2)
        b = dense.mixed_ffn(x, z, 6, w1, w2, wn1, wn2, save8=True)
        with torch.no_grad():
            c = dense.mixed_ffn(x, z, 6, w1, w2, wn1, wn2, save8=True)
    assert a.dtype == b.dtype == c.dtype and (a - b).norm() <= 2.0 ** -6 * a.norm() and (a - c).norm() <= 2.0 ** -6 * a.norm()
    for u, v, t in zip(*(torch.autograd.grad(y, leaves, torch.ones_like(y)) for y in (a, b)), leaves):
        assert v.dtype == t.dtype and (u.double() - v.double()).norm() <= 0.04 * u.double().norm()


def test_training_with_sharded_parameters():
    """FSDP frees a block's bf16 weights after its forward and gathers them again for its backward, which the layers' nodes
    hold: gradients are those of the same model unsharded. They leave it in bf16, and the norms' weights enter in bf16: some
    roundings of 2^-8 in each of two blocks, for which 2^-5 leaves room. One rank, in a process of its own."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    code = """
import os, sys
sys.path[:0] = [%r, %r]
import datetime, socket, torch, torch.distributed as dist
with socket.socket() as s:
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
torch.cuda.set_device(0)
dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1, timeout=datetime.timedelta(seconds=60),
                        device_id=torch.device("cuda", 0))
from primus_dlrm_b200.parallel.fsdp import DTensor, full_tensor, shard_dense
from test_models_cpu import _batch
from test_onetrans_rotary import _model
kw = dict(dropout=0.0, attention_impl="fav4", d_model=64, heads=2, activation_bits=8)
a, b = _model("cuda", **kw).train(), _model("cuda", **kw).train()
b.load_state_dict(a.state_dict())
shard_dense(b, torch.device("cuda", 0), dist.group.WORLD, torch.bfloat16)
batch = {k: v.cuda() for k, v in _batch(B=32, windows=2).items()}
grads = []
for m in (a, b):
    for again in range(2):
        m.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            total, _, _ = m.forward_loss(batch, {"listen_plus": 1.0}, [])
        total.backward()
    grads.append((total.item(), {n: full_tensor(p.grad).float() for n, p in m.named_parameters() if p.grad is not None and n.startswith("blocks")}))
(la, ga), (lb, gb) = grads
assert isinstance(b.blocks[0].ffn.s_w1.weight, DTensor) and ga.keys() == gb.keys() and len(ga) > 10
print("LOSS", abs(la - lb) <= 2.0 ** -8 * abs(la))
worst = max((float((ga[n] - gb[n]).norm() / (ga[n].norm() + 1e-12)), n) for n in ga)
print("GRADS", worst[0] <= 2.0 ** -5, worst)
torch.cuda.synchronize()
dist.destroy_process_group()
""" % (str(root), str(root / "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "LOSS True" in r.stdout and "GRADS True" in r.stdout, r.stdout + r.stderr[-2000:]


def test_calls_at_once_all_end():
    """Two threads with streams of their own, forward and backward through every form: each of their calls ends, with the
    results of a call by itself; what a thread raises is seen."""
    import threading
    g = _gen(11)
    w = Int8Weight.from_float(torch.randn(300, 640, generator=g, device=DEV))
    xs = [torch.randn(m, 640, generator=g, device=DEV).bfloat16() for m in (1, 16, 90, 3000)]
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    # at most 64 rows a sum, in one block: no order of additions changes a weight's gradient
    layer = [r(4, 9, 64), r(4, 9, 64), r(128, 64), r(64, 128), r(3, 128, 64), r(3, 64, 128)]
    dy = r(4, 9, 64)

    def once(leaves):
        out = [int8_linear(x, w, act="gelu") for x in xs] + [load8(save8(x)) for x in xs]
        y = dense.mixed_ffn(leaves[0], leaves[1], 6, *leaves[2:], save8=True)
        return out + [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = once([t.clone().requires_grad_() for t in layer])
    torch.cuda.synchronize()
    bad, done = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                leaves = [t.clone().requires_grad_() for t in layer]
                for _ in range(20):
                    for a, b in zip(once(leaves), want):
                        if not torch.equal(a, b):
                            bad.append(a.shape)
                    done.append(1)
        except Exception as e:  # noqa: BLE001 - any of them is a failure of this test
            bad.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and len(done) == 40


def test_a_backward_captured_beside_an_eager_graph_ends_in_an_error_or_a_result():
    """A backward pass captured while an eager graph of the same leaves lives: PyTorch may refuse it, for its own operations
    alike. Either way the process goes on, and exits as it should."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys
sys.path.insert(0, %r)
import torch
from primus_dlrm_b200.ops import dense
r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
p = [t.requires_grad_() for t in (r(2, 9, 64), r(2, 9, 64), r(128, 64), r(64, 128), r(3, 128, 64), r(3, 64, 128))]
dy = r(2, 9, 64)
layer = lambda: dense.mixed_ffn(p[0], p[1], 6, *p[2:], save8=True)
want = torch.autograd.grad(layer(), p, dy)
alive = layer()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(layer(), p, dy)
    graph.replay()
    print("CAPTURED", all(torch.equal(a, b) for a, b in zip(got, want)))
except RuntimeError as e:
    print("REFUSED True", str(e)[:200])
torch.cuda.synchronize()
print("AFTER", all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, p, dy), want)))
""" % str(Path(__file__).resolve().parent.parent)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr[-1500:]
    assert ("CAPTURED True" in r.stdout) != ("REFUSED True" in r.stdout) and "AFTER True" in r.stdout, r.stdout
