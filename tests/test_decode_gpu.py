"""Decoding steps against a cache (window with sinks, shared prefix) on the GPU, against
fp64 with counted roundings."""
import math

import pytest
import torch

import positional_ref as ref

pytestmark = pytest.mark.gpu


def make(b, hq, hkv, t, cap, d, ty=torch.bfloat16, seed=0, prefix=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda").to(ty)
    out = [rnd(b, hq, t, d), rnd(b, hkv, cap, d), rnd(b, hkv, cap, d)]
    if prefix is not None:
        out += [rnd(hkv, prefix, d), rnd(hkv, prefix, d)]
    return out


def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def poison(k, v, lengths):
    """NaN and infinities in every cache row that is not in use."""
    for i, n in enumerate(lengths.tolist()):
        n = max(n, 0)
        k[i, :, n:] = math.nan
        v[i, :, n:] = math.inf


def check_window(q, k, v, lengths, window, sinks, scale=None):
    from blackflash_b200 import window_decode
    poison(k, v, lengths)
    o, lse = window_decode(q, k, v, lengths, window, sinks, scale, want_lse=True)
    o64, lse64, pv = ref.decode_ref(q, k, v, lengths, window, sinks, scale or 1 / math.sqrt(q.shape[3]))
    ref.check_o(o, o64, pv)
    ref.check_lse(lse, lse64)
    assert torch.equal(window_decode(q, k, v, lengths, window, sinks, scale), o)
    return o


def check_prefix(q, k, v, kp, vp, lengths):
    from blackflash_b200 import prefix_decode, wait_status
    poison(k, v, lengths)
    o, lse = prefix_decode(q, kp, vp, k, v, lengths, want_lse=True)
    torch.cuda.synchronize()
    assert wait_status() == 0
    o64, lse64, pv = ref.decode_ref(q, k, v, lengths, 1 << 40, 0, 1 / math.sqrt(q.shape[3]), kp, vp)
    ref.check_o(o, o64, pv)
    ref.check_lse(lse, lse64)
    assert torch.equal(prefix_decode(q, kp, vp, k, v, lengths), o)
    return o


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ty", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 1), (100, 0), (257, 16), (10 ** 9, 0), (5, 10 ** 9),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window_decode_ragged(d, ty, window, sinks):
    q, k, v = make(8, 8, 2, 1, 700, d, ty, seed=window % 97)
    check_window(q, k, v, lens(0, 1, 2, 31, 128, 333, 699, 700), window, sinks)


@pytest.mark.parametrize("hq,hkv,t", [(1, 1, 1), (3, 3, 2), (16, 1, 1), (17, 1, 1), (32, 4, 5), (40, 1, 3), (6, 2, 33)])
def test_window_decode_rows(hq, hkv, t):
    """Row tiles that are full, ragged and several; tokens before the first key see nothing."""
    for d in (64, 128):
        q, k, v = make(4, hq, hkv, t, 300, d, seed=t)
        check_window(q, k, v, lens(300, t - 1, 0, 150), 90, 4)


def test_window_decode_long_splits():
    """Enough keys for many splits; some sequences far shorter than the longest."""
    q, k, v = make(3, 8, 2, 2, 20011, 64, seed=3)
    check_window(q, k, v, lens(20011, 700, 1), 15001, 9)
    q, k, v = make(1, 8, 1, 1, 30000, 128, seed=4)
    check_window(q, k, v, lens(29999), 10 ** 6, 0)


def test_window_decode_matches_prompt_row():
    """The step at position n is row n of the prompt pass."""
    from blackflash_b200 import window_attention
    n, w, s = 500, 120, 4
    q, k, v = make(2, 8, 2, n, n, 128, seed=6)
    full = window_attention(q, k, v, w, s)
    o64, _, pv = ref.window_ref(q, k, v, w, s, 1 / math.sqrt(128))
    for pos in (0, 1, 119, 120, 124, 499):
        o = check_window(q[:, :, pos: pos + 1], k.clone(), v.clone(), lens(pos + 1, pos + 1), w, s)
        ref.check_o(o, o64[:, :, pos: pos + 1], pv[:, :, pos: pos + 1])
        ref.check_o(full[:, :, pos: pos + 1], o64[:, :, pos: pos + 1], pv[:, :, pos: pos + 1])


def test_window_decode_strides_lengths_past_the_cache_and_offsets():
    """Token-major caches, lengths held to 0 .. C, and a cache whose offsets pass 2^31 elements."""
    from blackflash_b200 import window_decode
    gen = torch.Generator(device="cuda").manual_seed(0)
    cache = torch.randn(2, 4, 300, 2, 3, 64, generator=gen, device="cuda").to(torch.bfloat16)  # [2, B, C, ., H, d]
    k, v = (x[:, :, 1].transpose(1, 2) for x in cache)
    q = torch.randn(4, 2, 6, 64, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2)
    n = lens(-5, 301, 2 ** 31 - 1, 150)
    o = window_decode(q, k, v, n, 60, 2)
    o64, _, pv = ref.decode_ref(q, k, v, n, 60, 2, 0.125)
    ref.check_o(o, o64, pv)
    big = torch.empty(2, 1, (1 << 24) + 100, 128, dtype=torch.bfloat16, device="cuda")  # 2^32 elements
    big[:, :, -600:].normal_(generator=gen)
    big[:, :, :8].normal_(generator=gen)
    q = torch.randn(2, 4, 1, 128, generator=gen, device="cuda").to(torch.bfloat16)
    full = big.shape[2]
    o = window_decode(q, big, big, lens(full, full - 1), 500, 4)
    for i, n in enumerate((full, full - 1)):
        kk = torch.cat([big[i, :, :4], big[i, :, n - 500: n]], 1)[None]
        o64, _, pv = ref.decode_ref(q[i: i + 1], kk, kk, lens(504), 1 << 40, 0, 1 / math.sqrt(128))
        ref.check_o(o[i: i + 1], o64, pv)


@pytest.mark.parametrize("d,ty", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float16), (128, torch.float16)])
@pytest.mark.parametrize("b,hq,hkv,t,prefix,cap", [
    (1, 1, 1, 1, 1, 1), (4, 8, 2, 1, 1000, 128), (33, 8, 2, 1, 129, 40), (5, 10, 2, 1, 300, 17), (70, 4, 1, 3, 257, 9),
    (2, 16, 1, 9, 200, 30), (3, 6, 3, 1, 5000, 64), (130, 4, 4, 1, 128, 5),
])
def test_prefix_decode_parity(d, ty, b, hq, hkv, t, prefix, cap):
    q, k, v, kp, vp = make(b, hq, hkv, t, cap, d, ty, seed=b + prefix, prefix=prefix)
    lengths = torch.randint(0, cap + 1, (b,), device="cuda", dtype=torch.int32,
                            generator=torch.Generator(device="cuda").manual_seed(b))
    check_prefix(q, k, v, kp, vp, lengths)


@pytest.mark.parametrize("d,ty", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("b,hq,hkv,t,prefix", [
    (1, 1, 1, 1, 1), (4, 8, 2, 1, 1000), (33, 8, 2, 1, 129), (5, 10, 2, 1, 300), (70, 4, 1, 3, 257),
    (2, 16, 1, 9, 200), (3, 6, 3, 1, 5000), (130, 4, 4, 1, 128),
])
def test_prefix_decode_large_caches(d, ty, b, hq, hkv, t, prefix):
    """Capacities for which the prefix is read by a kernel of its own, whatever the lengths are."""
    cap = (33 << 20) // (b * hkv * ((hq // hkv * t + 15) // 16) * d * 4) + 1
    q, k, v, kp, vp = make(b, hq, hkv, t, cap, d, ty, seed=b + prefix, prefix=prefix)
    lengths = torch.randint(0, 60, (b,), device="cuda", dtype=torch.int32,
                            generator=torch.Generator(device="cuda").manual_seed(b))
    check_prefix(q, k, v, kp, vp, lengths)


@pytest.mark.parametrize("t", [1, 4])
def test_prefix_decode_sides_of_the_rule(t):
    """The same step just below and just above the size from which the prefix has its own kernel."""
    from blackflash_b200 import prefix_decode
    below = (32 << 20) // (4 * 2 * 128 * 4) - 900
    q, k, v, kp, vp = make(4, 8, 2, t, below + 1, 128, seed=t, prefix=900)
    n = lens(0, 2, 1000, below)
    for cap in (below, below + 1):
        o64, _, pv = ref.decode_ref(q, k[:, :, :cap], v[:, :, :cap], n, 1 << 40, 0, 1 / math.sqrt(128), kp, vp)
        ref.check_o(prefix_decode(q, kp, vp, k[:, :, :cap], v[:, :, :cap], n), o64, pv)


def test_prefix_decode_without_prefix_or_cache():
    from blackflash_b200 import prefix_decode, window_decode
    q, k, v, kp, vp = make(3, 4, 2, 2, 50, 64, seed=1, prefix=77)
    n = lens(50, 0, 1)
    assert torch.equal(prefix_decode(q, kp[:, :0], vp[:, :0], k, v, n), window_decode(q, k, v, n, 50))
    check_prefix(q, k[:, :, :0], v[:, :, :0], kp, vp, lens(0, 0, 0))
    o, lse = prefix_decode(q, kp[:, :0], vp[:, :0], k[:, :, :0], v[:, :, :0], n, want_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()


def test_prefix_decode_strided_prefix_and_big_batch():
    gen = torch.Generator(device="cuda").manual_seed(8)
    pages = torch.randn(2, 400, 4, 128, generator=gen, device="cuda").to(torch.bfloat16)  # [2, P, Hkv, d]
    q, k, v, _, _ = make(64, 16, 4, 1, 30, 128, seed=8, prefix=1)
    check_prefix(q, k, v, pages[0].transpose(0, 1), pages[1].transpose(0, 1),
                 torch.randint(1, 31, (64,), device="cuda", dtype=torch.int32))


def test_steps_on_other_streams_and_in_two_graphs():
    """Workspaces are the call's own: two graphs replayed at once do not share one."""
    from blackflash_b200 import prefix_decode, window_decode
    q, k, v, kp, vp = make(4, 8, 2, 1, 3000, 64, seed=2, prefix=2000)
    n = lens(3000, 2999, 17, 1024)
    side = torch.cuda.Stream()
    calls = [lambda: window_decode(q, k, v, n, 2500, 4), lambda: prefix_decode(q, kp, vp, k, v, n)]
    for call in calls:
        want = call()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call()
        side.synchronize()
        assert torch.equal(got, want)
    graphs, outs = [], []
    for call in calls * 2:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    q.copy_(torch.randn_like(q))
    n.copy_(lens(5, 3000, 2048, 333))
    want = [call() for call in calls * 2]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@pytest.mark.parametrize("d,ty", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("b,hq,hkv,t,cap,window,sinks", [
    (1, 8, 2, 1, 130, 999, 0), (1, 8, 2, 1, 384, 100, 6), (1, 8, 2, 1, 385, 999, 0), (1, 8, 2, 1, 769, 999, 0),
    (2, 6, 3, 7, 700, 300, 5), (37, 4, 4, 1, 1100, 1024, 4), (37, 8, 4, 1, 1025, 9999, 0), (149, 1, 1, 2, 384, 380, 1),
    (13, 6, 6, 1, 513, 257, 1),
])
def test_decode_few_keys(d, ty, b, hq, hkv, t, cap, window, sinks):
    """Around the sizes up to which one block, of four warps or of eight, takes all keys of a head."""
    q, k, v = make(b, hq, hkv, t, cap, d, ty, seed=cap)
    lengths = torch.randint(0, cap + 1, (b,), device="cuda", dtype=torch.int32,
                            generator=torch.Generator(device="cuda").manual_seed(b))
    lengths[-1] = cap
    check_window(q, k, v, lengths, window, sinks)
