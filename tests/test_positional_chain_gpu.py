"""The position-aware operators together, as a model uses them: rotary positions, a windowed
prompt pass into a cache, decoding steps from it; a batch behind a shared prefix; a training
step through rotary and windowed attention. Against fp64."""
import math

import pytest
import torch

import positional_ref as ref

pytestmark = pytest.mark.gpu


def rotary_bound(x, amplitude):
    """Half a bf16 step of the turned value, plus what fp32 arithmetic adds (test_rotary_gpu)."""
    return ref.half_step(x.dtype) * 1.001 * amplitude


def test_prompt_then_steps_match_one_pass():
    """A prompt of 300 tokens, then 5 steps, one of two tokens; the window (64) and the sinks (4)
    leave most of the cache behind. The same rotated Q, K go into the fp64 statement."""
    from blackflash_b200 import rotary, rotary_frequencies, window_attention, window_decode
    b, hq, hkv, d, window, sinks, cap = 2, 8, 2, 128, 64, 4, 400
    freqs, amp = rotary_frequencies(96, 500000.0, "by-parts", 4.0, 128)
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = 306
    q, k, v = (torch.randn(b, n, h, d, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2) for h in (hq, hkv, hkv))
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    qr, kr = rotary(q, k, pos, freqs, amplitude=amp)
    err = (qr.double() - ref.rotary64(q, pos, freqs, False, amp)).abs()
    assert (err <= rotary_bound(q, 1.0) * qr.double().abs() + 1e-5).all()
    o64, _, pv = ref.window_ref(qr, kr, v, window, sinks, 1 / math.sqrt(d))

    kc, vc = (torch.full((b, hkv, cap, d), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    done = 300
    kc[:, :, :done], vc[:, :, :done] = kr[:, :, :done], v[:, :, :done]
    o = window_attention(qr[:, :, :done], kc[:, :, :done], vc[:, :, :done], window, sinks)  # views of the cache
    ref.check_o(o, o64[:, :, :done], pv[:, :, :done])
    for t in (1, 1, 2, 1, 1):
        step = slice(done, done + t)
        qs, ks = rotary(q[:, :, step], k[:, :, step], pos[step], freqs, amplitude=amp)
        assert torch.equal(qs, qr[:, :, step]) and torch.equal(ks, kr[:, :, step])
        kc[:, :, step], vc[:, :, step] = ks, v[:, :, step]
        done += t
        o = window_decode(qs, kc, vc, torch.full((b,), done, dtype=torch.int32, device="cuda"), window, sinks)
        ref.check_o(o, o64[:, :, step], pv[:, :, step])
    assert done == n


def test_prefix_steps_match_one_cache():
    """Behind a shared prefix: the step equals one against caches that hold the prefix each, and
    the two results agree within their bounds; then a chunk of the prompt through the window."""
    from blackflash_b200 import prefix_decode, window_attention, window_decode
    b, hq, hkv, d, p, c = 3, 6, 2, 64, 500, 40
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda").to(torch.bfloat16)
    kp, vp, k, v, q = rnd(hkv, p, d), rnd(hkv, p, d), rnd(b, hkv, c, d), rnd(b, hkv, c, d), rnd(b, hq, 2, d)
    n = torch.tensor([40, 2, 17], dtype=torch.int32, device="cuda")
    full_k, full_v = (torch.cat([x.expand(b, -1, -1, -1), y], 2) for x, y in ((kp, k), (vp, v)))
    o64, _, pv = ref.decode_ref(q, k, v, n, 1 << 40, 0, 0.125, kp, vp)
    shared = prefix_decode(q, kp, vp, k, v, n)
    apart = window_decode(q, full_k, full_v, n + p, p + c)
    ref.check_o(shared, o64, pv)
    ref.check_o(apart, o64, pv)
    for i in range(b):  # the prompt's last two rows
        m = p + int(n[i])
        o = window_attention(q[i: i + 1], full_k[i: i + 1, :, :m], full_v[i: i + 1, :, :m], m)
        ref.check_o(o, o64[i: i + 1], pv[i: i + 1])


def test_training_step_through_rotary_and_window():
    """Gradients of the chain for the projections' outputs, against fp64 autograd.

    Two roundings more than the attention's own bound: dQ and dK are rounded to bf16 before the
    inverse turn (their bound holds elementwise and a turn mixes a pair, so the pair's bounds add
    up), and the turned Q, K that the statement starts from are the rounded ones."""
    from blackflash_b200 import rotary, rotary_frequencies, rotary_with_grad, window_attention_with_grad
    b, hq, hkv, n, d, window, sinks = 1, 4, 2, 260, 64, 100, 3
    freqs, _ = rotary_frequencies(d)
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(b, n, h, d, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2).requires_grad_(True)
               for h in (hq, hkv, hkv))
    pos = torch.arange(n, device="cuda")
    do = torch.randn(b, hq, n, d, generator=gen, device="cuda").to(torch.bfloat16)
    qr, kr = rotary_with_grad(q, k, pos, freqs)
    o = window_attention_with_grad(qr, kr, v, window, sinks)
    gq, gk, gv = torch.autograd.grad(o, (q, k, v), do)
    with torch.no_grad():
        qr, kr = rotary(q, k, pos, freqs)
        want = ref.window_grad_ref(qr, kr, v, do, window, sinks, 1 / math.sqrt(d))
        for got, name in ((gq, "dq"), (gk, "dk")):
            g, lim = want[name]
            back = ref.rotary64(g, pos, freqs, False, 1.0, -1.0)
            pair = lim[..., : d // 2] + lim[..., d // 2:]
            lim2 = torch.cat([pair, pair], -1) + ref.half_step(torch.bfloat16) * back.abs() * 1.01 + 1e-5
            assert ((got.double() - back).abs() <= lim2).all(), name
        g, lim = want["dv"]
        assert ((gv.double() - g).abs() <= lim).all()


def test_differentiable_once():
    from blackflash_b200 import rotary_frequencies, rotary_with_grad, window_attention_with_grad
    x = torch.randn(1, 2, 8, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
    freqs, _ = rotary_frequencies(64)
    outs = [window_attention_with_grad(x, x, x, 4), rotary_with_grad(x, x, torch.arange(8, device="cuda"), freqs)[0]]
    for o in outs:
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(o.float().sum(), x, create_graph=True)
    h = x.detach().half().requires_grad_(True)
    with pytest.raises(RuntimeError, match="bfloat16"):
        window_attention_with_grad(h, h, h, 4)


def test_refusals_on_the_gpu():
    """Layouts and sizes that only a CUDA tensor can have; each leaves the context usable."""
    import blackflash_b200 as bf
    q = torch.randn(2, 4, 16, 64, device="cuda").to(torch.bfloat16)
    k = q[:, :2]
    n = torch.tensor([16, 16], dtype=torch.int32, device="cuda")
    freqs, _ = bf.rotary_frequencies(64)
    pos = torch.arange(16, device="cuda")
    kp = q[0, :2]
    odd = torch.randn(2, 4, 16, 68, device="cuda").to(torch.bfloat16)[..., 2:66]
    bad = [
        lambda: bf.window_attention(q, q[:, :3], q[:, :3], 4), lambda: bf.window_attention(q, k, k[:, :, :8], 4),
        lambda: bf.window_attention(q, k, k, 0), lambda: bf.window_attention(q, k, k, 4, -1),
        lambda: bf.window_attention(q, k, k, 4, 0, 0.0), lambda: bf.window_attention(q, k, k, 4, 0, math.inf),
        lambda: bf.window_attention(q.half(), k, k, 4), lambda: bf.window_attention(q.float(), q.float(), q.float(), 4),
        lambda: bf.window_attention(q[..., :32], k[..., :32], k[..., :32], 4), lambda: bf.window_attention(q[..., ::2], k, k, 4),
        lambda: bf.window_attention(odd, odd, odd, 4), lambda: bf.window_attention(q, k[:, :1].expand(2, 2, 16, 64), k, 4),
        lambda: bf.window_attention(q.transpose(2, 3), k, k, 4), lambda: bf.window_attention(q, k.cpu(), k, 4),
        lambda: bf.window_decode(q, k, k, n.long(), 4), lambda: bf.window_decode(q, k, k, n[:1], 4),
        lambda: bf.window_decode(q, k, k, n.cpu(), 4), lambda: bf.window_decode(q, odd[:, :2], odd[:, :2], n, 4),
        lambda: bf.prefix_decode(q, kp[:1], kp[:1], k, k, n), lambda: bf.prefix_decode(q, kp, kp[:, :4], k, k, n),
        lambda: bf.prefix_decode(q, kp.half(), kp, k, k, n),
        lambda: bf.rotary(q, k, pos[:4], freqs), lambda: bf.rotary(q, k, pos.float(), freqs), lambda: bf.rotary(q, k, pos, freqs.float()),
        lambda: bf.rotary(q, k, pos.cpu(), freqs), lambda: bf.rotary(q, k, pos, freqs[:0]),
        lambda: bf.rotary(q[..., :32], k[..., :32], pos, freqs), lambda: bf.rotary(q, k, pos, freqs, False, math.nan),
        lambda: bf.window_attention_backward(q, k, k, q, q, torch.zeros(2, 4, 15, device="cuda"), 4),
        lambda: bf.window_attention_backward(q, k, k, q.transpose(0, 1).contiguous().transpose(0, 1), q,
                                             torch.zeros(2, 4, 16, device="cuda"), 4),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
    assert torch.isfinite(bf.window_attention(q, k, k, 4)).all()


FIRST_CALLS = """
import torch
import blackflash_b200 as bf
q = torch.randn(2, 4, 200, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
k, n = q.detach()[:, :2], torch.tensor([200, 77], dtype=torch.int32, device="cuda")
freqs, _ = bf.rotary_frequencies(64)
pos = torch.arange(200, device="cuda")
def calls():
    o = bf.window_attention_with_grad(q, k, k, 50, 4)
    return [o.detach(), torch.autograd.grad(o, q, torch.ones_like(o))[0], *bf.rotary(q.detach(), k, pos, freqs),
            bf.window_decode(q.detach()[:, :, :1], k, k, n, 50, 4), bf.prefix_decode(q.detach()[:, :, :1], k[0], k[0], k, k, n)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
print("captured")
"""


def test_first_calls_of_a_process_under_capture():
    """Set-up that a first call does (kernel attributes, entry points) is allowed in a capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


CAPTURED_LEAF = """
import torch
import blackflash_b200 as bf
q = torch.randn(2, 4, 200, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
k = torch.randn(2, 2, 200, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
freqs, _ = bf.rotary_frequencies(64)
pos = torch.arange(200, device="cuda")
forms = {"window": lambda: bf.window_attention_with_grad(q, k, k, 50, 4),
         "rotary": lambda: bf.rotary_with_grad(q, k, pos, freqs)[0]}
grad = torch.ones_like(q)
def step(form):
    return torch.autograd.grad(form(), [q, k], grad)
for name, form in forms.items():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(form)
    torch.cuda.current_stream().wait_stream(side)
    alive = form()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            step(form)
    except RuntimeError as e:
        assert "graph of its inputs" in str(e), e
        print("refused", name, flush=True)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(form)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step(form)))
    print("captured", name, flush=True)
"""


def test_captured_backward_beside_an_eager_graph_of_its_leaves():
    """Refused, in words, and captured once that graph is gone; in a process of its own, which
    the engine's failure would end."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", CAPTURED_LEAF], cwd=root, capture_output=True, text=True, timeout=300)
    lines = [f"{what} {name}" for name in ("window", "rotary") for what in ("refused", "captured")]
    assert out.returncode == 0 and out.stdout.split("\n")[:-1] == lines, out.stdout + out.stderr[-2000:]


CAPTURED_PROJECTION = """
import torch
import blackflash_b200 as bf
x = torch.randn(2, 200, 6, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)  # [B, N, H, d]
w = torch.randn(2, 2, 200, 64, device="cuda").to(torch.bfloat16).requires_grad_(True)
freqs, _ = bf.rotary_frequencies(64)
pos = torch.arange(200, device="cuda")
grad = torch.ones(2, 4, 200, 64, device="cuda", dtype=torch.bfloat16)
def window(a=x):
    h = a.transpose(1, 2)
    return bf.window_attention_with_grad(h[:, :4], h[:, 4:], h[:, 4:], 50, 4)
def chain(a=x):
    q, k = bf.rotary_with_grad(a[:, :, :4].transpose(1, 2), a[:, :, 4:].transpose(1, 2), pos, freqs)
    return bf.window_attention_with_grad(q, k, k * 2, 50, 4)
def beside(a=x):
    return bf.window_attention_with_grad(a[:, :, :4].transpose(1, 2), w, w, 50, 4)
def warm(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
def captured(step):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    return [t.clone() for t in got]
def check(name, form, leaves, alive):
    step = lambda: torch.autograd.grad(form(), leaves, grad)
    warm(step)
    alive = alive()
    try:
        captured(step)
        print("captured", name, flush=True)
    except RuntimeError as e:
        assert "graph of its inputs" in str(e), e
        print("refused", name, flush=True)
    del alive
    assert all(torch.equal(a, b) for a, b in zip(captured(step), step())), name
    print("alone", name, flush=True)
check("window", window, [x], lambda: x * 1)
check("chain", chain, [x], lambda: x * 1)
# A leaf that this backward does not reach may keep its graph.
check("beside", beside, [x], lambda: w * 1)
"""


def test_captured_backward_through_other_operations():
    """The leaf lies behind a transposed view or a slice: refused in words all the same, and only
    where the backward reaches a leaf whose graph lives."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", CAPTURED_PROJECTION], cwd=root, capture_output=True, text=True, timeout=300)
    lines = ["refused window", "alone window", "refused chain", "alone chain", "captured beside", "alone beside"]
    assert out.returncode == 0 and out.stdout.split("\n")[:-1] == lines, out.stdout + out.stderr[-2000:]


@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed_step_and_no_grad_modes(reentrant):
    """Recomputed in the backward, the step has the same gradients; without gradients the same output."""
    from torch.utils.checkpoint import checkpoint

    from blackflash_b200 import rotary_frequencies, rotary_with_grad, window_attention, window_attention_with_grad
    freqs, _ = rotary_frequencies(64)
    pos = torch.arange(150, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 150, 6, 64, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_(True)
    do = torch.randn(2, 4, 150, 64, generator=gen, device="cuda").to(torch.bfloat16)

    def layer(a):
        q, k = rotary_with_grad(a[:, :, :4].transpose(1, 2), a[:, :, 4:].transpose(1, 2), pos, freqs)
        return window_attention_with_grad(q, k, k, 40, 2)
    o = layer(x)
    want, = torch.autograd.grad(o, x, do)
    layer_o = checkpoint(layer, x, use_reentrant=reentrant)
    layer_o.backward(do)
    assert torch.equal(layer_o, o) and torch.equal(x.grad, want)
    with torch.no_grad():
        assert torch.equal(layer(x), o)
    with torch.inference_mode():
        assert torch.equal(layer(x), o)
        q = x[:, :, :4].transpose(1, 2)
        assert torch.equal(window_attention(q, q, q, 40), window_attention_with_grad(q, q, q, 40))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current():
    import blackflash_b200 as bf
    q = torch.randn(1, 4, 200, 64, device="cuda:1").to(torch.bfloat16)
    o = bf.window_attention(q, q, q, 50, 4)
    o64, _, pv = ref.window_ref(q, q, q, 50, 4, 0.125)
    ref.check_o(o, o64, pv)
