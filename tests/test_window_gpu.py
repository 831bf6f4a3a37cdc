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
