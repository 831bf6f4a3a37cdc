"""Sliding-window attention with sinks on the GPU, against fp64 with counted roundings."""
import math

import pytest
import torch

import positional_ref as ref

pytestmark = pytest.mark.gpu


def make(b, hq, hkv, nq, nkv, d, t=torch.bfloat16, seed=0, heads_last=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def one(h, n):
        if heads_last:
            return torch.randn(b, n, h, d, generator=gen, device="cuda").to(t).transpose(1, 2)
        return torch.randn(b, h, n, d, generator=gen, device="cuda").to(t)
    return one(hq, nq), one(hkv, nkv), one(hkv, nkv)


def run_and_check(q, k, v, window, sinks, scale=None):
    from blackflash_b200 import wait_status, window_attention, window_attention_lse
    o, lse = window_attention_lse(q, k, v, window, sinks, scale)
    torch.cuda.synchronize()
    assert wait_status() == 0
    o64, lse64, pv = ref.window_ref(q, k, v, window, sinks, 1 / math.sqrt(q.shape[3]) if scale is None else scale)
    ref.check_o(o, o64, pv)
    ref.check_lse(lse, lse64)
    assert o.is_contiguous() and torch.equal(window_attention(q, k, v, window, sinks, scale), o)
    return o, lse


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,nkv,window,sinks", [
    (1, 1, 1, 0), (2, 2, 1, 1), (7, 7, 3, 0), (128, 128, 128, 0), (129, 129, 1, 0), (255, 255, 64, 4),
    (257, 257, 128, 128), (300, 300, 129, 1), (640, 640, 127, 129), (1000, 1000, 100, 300), (1000, 1000, 5000, 0),
    (777, 777, 1, 4), (1, 700, 50, 3), (5, 513, 128, 0), (130, 1000, 200, 16), (300, 100, 20, 2), (600, 1, 4, 0),
    (400, 129, 1, 1000000),
])
def test_window_parity(d, nq, nkv, window, sinks):
    run_and_check(*make(2, 4, 2, nq, nkv, d, seed=nq + nkv), window, sinks)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (3, 1), (6, 2), (8, 1), (10, 5), (12, 4)])
def test_window_head_groups(hq, hkv, t):
    for d in (64, 128):
        run_and_check(*make(2, hq, hkv, 333, 461, d, t, seed=hq), 150, 5)


def test_window_types_and_peaked_scores():
    """Scores of +-40: the lazy maximum moves, weights underflow, in both types."""
    for t in (torch.bfloat16, torch.float16):
        q, k, v = make(1, 2, 2, 700, 700, 64, t, seed=5)
        run_and_check((q * 3).to(t), (k * 3).to(t), v, 400, 4)
        run_and_check(q, k, v, 400, 4, scale=1e-3)


def test_window_strided_views():
    """[B, N, H, d] projections, a slice of a wider cache, and one of its rows per head."""
    from blackflash_b200 import window_attention
    q, k, v = make(2, 4, 2, 300, 300, 128, seed=1, heads_last=True)
    assert not q.is_contiguous()
    o, _ = run_and_check(q, k, v, 90, 7)
    assert torch.equal(o, window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 90, 7))
    wide = torch.randn(3, 5, 1000, 192, device="cuda").to(torch.bfloat16)
    run_and_check(wide[1:, :4, 100:400, 64:128], wide[1:, 2:4, 200:500, :64], wide[:2, 1:3, 500:800, 128:], 77, 3)


def test_window_many_items():
    """More items than multiprocessors: query buffers, rings and phases reused."""
    for d, hq, hkv in ((64, 16, 4), (128, 16, 4), (64, 15, 15), (128, 9, 3)):
        run_and_check(*make(3, hq, hkv, 1500, 1500, d, seed=d), 200, 4)


def test_window_causal_equals_dense_causal():
    """window >= N is the library's causal forward, within both kernels' roundings."""
    from blackflash_b200 import blackflash, window_attention
    q, k, v = make(2, 3, 3, 900, 900, 64, seed=3)
    a, b = blackflash(q, k, v, causal=True), window_attention(q, k, v, 900)
    o, _, pv = ref.window_ref(q, k, v, 900, 0, 0.125)
    assert ((a.double() - b.double()).abs() <= 2 * ref.o_bound(o, pv, q.dtype)).all()


def test_window_is_deterministic_and_leaves_neighbours():
    """Two calls agree bit for bit; rows around a view are not written."""
    from blackflash_b200 import window_attention
    q, k, v = make(1, 4, 2, 500, 500, 128, seed=9)
    assert torch.equal(window_attention(q, k, v, 130, 4), window_attention(q, k, v, 130, 4))


def test_window_other_stream_graph_and_autograd_thread():
    from blackflash_b200 import window_attention
    q, k, v = make(1, 4, 2, 400, 400, 64, seed=2)
    want = window_attention(q, k, v, 100, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = window_attention(q, k, v, 100, 4)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(window_attention(q, k, v, 100, 4))
        graphs.append(g)
    q2, k2, v2 = make(1, 4, 2, 400, 400, 64, seed=22)
    q.copy_(q2), k.copy_(k2), v.copy_(v2)
    want = window_attention(q, k, v, 100, 4)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_window_empty_problems():
    from blackflash_b200 import window_attention_lse
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    o, lse = window_attention_lse(z(2, 4, 3, 64), z(2, 2, 0, 64), z(2, 2, 0, 64), 5)
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = window_attention_lse(z(2, 4, 0, 64), z(2, 2, 9, 64), z(2, 2, 9, 64), 5)
    assert o.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)


def test_window_nan_query_row_stays_its_own():
    from blackflash_b200 import window_attention
    q, k, v = make(1, 2, 1, 300, 300, 64, seed=4)
    want = window_attention(q, k, v, 100, 4)
    q[0, 1, 150] = math.nan
    got = window_attention(q, k, v, 100, 4)
    assert torch.isnan(got[0, 1, 150]).all()
    got[0, 1, 150] = want[0, 1, 150]
    assert torch.equal(got, want)


# ---------------------------------------------------------------- gradients

def check_grads(got, q, k, v, do, window, sinks, scale=None):
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = ref.window_grad_ref(q, k, v, do, window, sinks, scale)
    for name, x in zip(("dq", "dk", "dv"), got):
        g, lim = want[name]
        err = (x.double() - g).abs()
        bad = int((err > lim).sum())
        assert bad == 0 and torch.isfinite(x).all(), (name, bad, x.numel(), float((err / lim).max()))


def grads_of(q, k, v, do, window, sinks, scale=None):
    from blackflash_b200 import wait_status, window_attention_backward, window_attention_lse
    o, lse = window_attention_lse(q, k, v, window, sinks, scale)
    got = window_attention_backward(q, k, v, o, do, lse, window, sinks, scale)
    torch.cuda.synchronize()
    assert wait_status() == 0
    return got


def upstream(q, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(q.shape, generator=gen, device="cuda").to(q.dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nq,nkv,window,sinks", [
    (1, 1, 1, 0), (3, 3, 2, 1), (64, 64, 64, 0), (65, 65, 10, 2), (128, 128, 128, 0), (129, 129, 1, 0), (255, 255, 64, 4),
    (300, 300, 129, 1), (640, 640, 127, 129), (1000, 1000, 100, 300), (1000, 1000, 5000, 0), (777, 777, 1, 4),
    (1, 700, 50, 3), (130, 1000, 200, 16), (300, 100, 20, 2), (600, 1, 4, 0), (2500, 2500, 64, 4),
])
def test_window_backward_parity(d, nq, nkv, window, sinks):
    q, k, v = make(2, 4, 2, nq, nkv, d, seed=nq + nkv)
    do = upstream(q)
    check_grads(grads_of(q, k, v, do, window, sinks), q, k, v, do, window, sinks)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (3, 1), (8, 1), (10, 5)])
def test_window_backward_head_groups_and_views(hq, hkv):
    for d in (64, 128):
        q, k, v = make(2, hq, hkv, 333, 461, d, seed=hq, heads_last=True)
        do = upstream(q.transpose(1, 2)).transpose(1, 2)
        check_grads(grads_of(q, k, v, do, 150, 5), q, k, v, do, 150, 5)


def test_window_backward_many_items_and_parts():
    """More items than multiprocessors, sink tiles in many parts, and a second run bit for bit."""
    for d, hq, hkv, n, w, s in ((64, 8, 2, 2000, 200, 4), (128, 8, 2, 2000, 200, 140), (64, 16, 16, 1300, 100, 1)):
        q, k, v = make(3, hq, hkv, n, n, d, seed=d)
        do = upstream(q)
        got = grads_of(q, k, v, do, w, s)
        check_grads(got, q, k, v, do, w, s)
        for a, b in zip(got, grads_of(q, k, v, do, w, s)):
            assert torch.equal(a, b)


def test_window_autograd_broadcast_and_differences():
    """Through autograd: K and V shared by expansion, a broadcast upstream, and a difference."""
    from blackflash_b200 import window_attention, window_attention_with_grad
    q, k, v = make(2, 4, 1, 300, 300, 64, seed=11)
    do = upstream(q)
    a = [x.clone().requires_grad_(True) for x in (q, k, v)]
    got = torch.autograd.grad(window_attention_with_grad(*a, 90, 4), a, do)
    check_grads(got, q, k, v, do, 90, 4)
    # One K/V head for all batches: the expanded leaf gets the sum over the batch.
    leaf = k[:1].clone().requires_grad_(True)
    kk = leaf.expand(2, 1, 300, 64).contiguous()
    g, = torch.autograd.grad(window_attention_with_grad(q, kk, v, 90, 4), leaf, do)
    full = torch.autograd.grad(window_attention_with_grad(q, kk, v, 90, 4), kk, do)[0]
    assert torch.equal(g, full.sum(0, keepdim=True))
    # A sum's gradient is one expanded number.
    x = q.clone().requires_grad_(True)
    g, = torch.autograd.grad(window_attention_with_grad(x, k, v, 90, 4).sum(), x)
    check_grads((g,), q, k, v, torch.ones_like(q), 90, 4)
    # A difference along a direction of V, in which O is linear: <dO, O(V + e) - O(V)> = <dV, e>.
    e = upstream(v, 5)
    v2 = (v + e).to(v.dtype)
    e = v2.double() - v.double()
    left = (do.double() * (window_attention(q, k, v2, 90, 4).double() - window_attention(q, k, v, 90, 4).double())).sum()
    right = (got[2].double() * e).sum()
    # Both sides are sums of 76800 and 38400 rounded terms; each term's bound adds up, in size.
    o1, _, pv1 = ref.window_ref(q, k, v, 90, 4, 0.125)
    o2, _, pv2 = ref.window_ref(q, k, v2, 90, 4, 0.125)
    lim = (do.double().abs() * (ref.o_bound(o1, pv1, q.dtype) + ref.o_bound(o2, pv2, q.dtype))).sum()
    lim = lim + (ref.window_grad_ref(q, k, v, do, 90, 4, 0.125)["dv"][1] * e.abs()).sum()
    assert abs(left - right) <= lim


def test_window_training_step_in_a_graph():
    """Forward and backward captured, replayed on new data, on a stream of their own."""
    from blackflash_b200 import window_attention_with_grad
    q, k, v = (x.requires_grad_(True) for x in make(1, 4, 2, 300, 300, 128, seed=12))
    do = upstream(q)

    def step():
        o = window_attention_with_grad(q, k, v, 100, 4)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        for x, y in zip((q, k, v), make(1, 4, 2, 300, 300, 128, seed=13)):
            x.copy_(y)
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_window_backward_empty():
    from blackflash_b200 import window_attention_backward
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, k = z(2, 4, 3, 64), z(2, 2, 0, 64)
    dq, dk, dv = window_attention_backward(q, k, k, q, q, torch.zeros(2, 4, 3, device="cuda"), 5)
    assert (dq == 0).all() and dk.shape == dv.shape == k.shape


@pytest.mark.parametrize("d,n,window,sinks", [(64, 300, 200, 4), (128, 618, 568, 0), (64, 700, 64, 65)])
def test_one_key_has_no_score_gradient(d, n, window, sinks):
    """The first row sees one key: P = 1, so dP - D is 0 whatever O was rounded to. In fp32,
    D = (P dP) / P is dP to three roundings of 2^-24 (two products, one quotient; P is 1 to a
    few 2^-22 and cancels), and dS = P (dP - D) rounds once more: 2^-21 |dP| holds them."""
    import blackflash_b200 as bf
    q, k, v = make(2, 6, 2, n, n, d)
    do = make(2, 6, 2, n, n, d, seed=1)[0]
    o, lse = bf.window_attention_lse(q, k, v, window, sinks)
    dq, _, _ = bf.window_attention_backward(q, k, v, o, do, lse, window, sinks)
    k0, v0 = (x[:, :, :1].double().repeat_interleave(3, 1) for x in (k, v))
    dp = (do[:, :, :1].double() * v0).abs().sum(-1, keepdim=True)  # at least |dP|, in either sweep's sum
    bound = d ** -0.5 * dp * k0.abs() * 2.0 ** -21
    assert (dq[:, :, :1].double().abs() <= bound).all()


@pytest.mark.parametrize("b,h,n,window,sinks", [
    (2, 20, 1500, 100, 3),    # fewer sink tiles than blocks, each as long as six others
    (1, 150, 700, 65, 1),     # two blocks have a second sink tile
    (3, 50, 513, 129, 130),   # two sink tiles a head
    (1, 80, 257, 30, 257),    # nothing but sink tiles
    (1, 140, 300, 30, 2),     # blocks without a sink tile are few
])
def test_window_backward_late_blocks(b, h, n, window, sinks):
    """Items of unlike length dealt to the blocks: every tile has its gradient, each time the same."""
    q, k, v = make(b, h, h, n, n, 64)
    do = upstream(q)
    got = grads_of(q, k, v, do, window, sinks)
    check_grads(got, q, k, v, do, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(got, grads_of(q, k, v, do, window, sinks)))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sinks", [1, 32, 33])
@pytest.mark.parametrize("window", [512, 513])
def test_window_sides_of_the_narrow_sink_step(t, sinks, window):
    """At d = 128 the sinks have a step of 32 columns up to window 512."""
    run_and_check(*make(1, 4, 2, 1100, 1100, 128, t, seed=sinks), window, sinks)
