"""Position-aware operators on values at the edge of their types, against fp64."""
import math

import pytest
import torch

import positional_ref as ref
from test_window_gpu import check_grads, grads_of, make, upstream

pytestmark = pytest.mark.gpu


def same_outside(got, want, rows):
    """Rows in `rows` are NaN in every column, all others as they were, bit for bit."""
    assert torch.isnan(got[rows]).all(), f"{int((~torch.isnan(got[rows])).sum())} numbers where a row sees a NaN"
    assert torch.equal(got[~rows], want[~rows])


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (3, 3)])
@pytest.mark.parametrize("base,sinks", [(0, 4), (64, 0), (130, 130), (184, 40)])
def test_a_key_of_nan_reaches_the_rows_that_see_it(t, d, hq, hkv, base, sinks):
    """At every index of 16: none may hide in columns that another form of the exponential takes."""
    from blackflash_b200 import window_attention_lse
    n, window = 200, 60
    q, k, v = make(16, hq, hkv, n, n, d, t, seed=base)
    want, want_lse = window_attention_lse(q, k, v, window, sinks)
    seen = ref.visible(n, n, window, sinks, "cuda")
    rows = torch.zeros(16, hq, n, dtype=torch.bool, device="cuda")
    for i in range(16):
        k[i, -1, base + i] = math.nan  # of the last KV head
        rows[i, -(hq // hkv):] = seen[:, base + i]
    got, lse = window_attention_lse(q, k, v, window, sinks)
    same_outside(got, want, rows)
    same_outside(lse, want_lse, rows)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sinks", [0, 100])
def test_infinite_scores(t, d, sinks):
    """A score of +inf (or of inf times 0) makes its row NaN, as the definition does; one of -inf
    has weight 0."""
    from blackflash_b200 import window_attention_lse
    n, window, base = 300, 90, 64
    q, k, v = make(16, 2, 2, n, n, d, t, seed=7)
    seen = ref.visible(n, n, window, sinks, "cuda").repeat(16, 2, 1, 1)
    rows = torch.zeros(16, 2, n, dtype=torch.bool, device="cuda")
    for i in range(16):
        rows[i] = seen[i, :, :, base + i] & (q[i, :, :, 5] >= 0)
        k[i, :, base + i, 5] = 0  # for the statement, which leaves that key out
        seen[i, :, :, base + i] = False
    o64, lse64, _, pv = ref.attention64(q.double(), k.double(), v.double(), seen, 1 / math.sqrt(d))
    for i in range(16):
        k[i, :, base + i, 5] = math.inf
    got, lse = window_attention_lse(q, k, v, window, sinks)
    assert torch.isnan(got[rows]).all() and torch.isnan(lse[rows]).all()
    ref.check_o(got[~rows], o64[~rows], pv[~rows])
    ref.check_lse(lse[~rows], lse64[~rows])


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
def test_a_prefix_key_of_nan_reaches_every_row(t, d):
    """In the prefix's own kernel (a large cache, hardly used), at every index of 16."""
    from blackflash_b200 import prefix_decode, wait_status
    b, hq, hkv, p = 4, 8, 2, 300
    cap = (33 << 20) // (b * hkv * d * 4) + 1
    gen = torch.Generator(device="cuda").manual_seed(d)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda").to(t)
    q, kp, vp = rnd(b, hq, 1, d), rnd(hkv, p, d), rnd(hkv, p, d)
    k, v = torch.zeros(2, b, hkv, cap, d, dtype=t, device="cuda")
    k[:, :, :9], v[:, :, :9] = rnd(b, hkv, 9, d), rnd(b, hkv, 9, d)
    n = torch.tensor([0, 1, 9, 4], dtype=torch.int32, device="cuda")
    want, want_lse = prefix_decode(q, kp, vp, k, v, n, want_lse=True)
    rows = torch.zeros(b, hq, 1, dtype=torch.bool, device="cuda")
    rows[:, hq // hkv:] = True
    for key in range(140, 156):
        bad = kp.clone()
        bad[1, key] = math.nan
        got, lse = prefix_decode(q, bad, vp, k, v, n, want_lse=True)
        same_outside(got, want, rows)
        same_outside(lse, want_lse, rows)
    torch.cuda.synchronize()
    assert wait_status() == 0


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_bits_do_not_depend_on_the_alignment(t, interleaved):
    """A view that starts on a pair and one that starts on 16 bytes give the same bits."""
    from blackflash_b200 import rotary, rotary_frequencies
    freqs, amp = rotary_frequencies(128, 500000.0, "by-parts", 4.0, 8192)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 6, 200, 128, generator=gen, device="cuda").to(t)
    pos = torch.randint(0, 1 << 20, (2, 200), generator=gen, device="cuda")
    wide = torch.zeros(2, 6, 200, 136, dtype=t, device="cuda")
    wide[..., 2:130] = x
    outs = [rotary(v, v[:, :2], pos, freqs, interleaved, amp) for v in (x, wide[..., 2:130])]
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def largest(shape, t, seed):
    """Random signs of the type's largest number."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    sign = torch.randint(0, 2, shape, generator=gen, device="cuda") * 2 - 1
    return (sign * torch.finfo(t).max).to(t)


def unseen_keys(t, d, nq, window, sinks):
    """A chunk of queries, its keys, and which of these no query sees (zero so far)."""
    n = 256
    q, k, v = make(2, 4, 2, nq, n, d, t, seed=nq)
    unseen = ~ref.visible(nq, n, window, sinks, "cuda").any(0)
    assert unseen.sum() > 50
    k[:, :, unseen], v[:, :, unseen] = 0, 0
    return q, k, v, unseen


CHUNKS = pytest.mark.parametrize("nq,window,sinks", [(8, 16, 4), (8, 16, 0), (130, 16, 0), (1, 1, 0), (40, 60, 100)])


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@CHUNKS
def test_masked_keys_of_the_largest_size(t, d, nq, window, sinks):
    """Finite keys and values that no query sees have weight 0, however large: what a cache may
    hold between the sinks and the window."""
    from blackflash_b200 import window_attention_lse
    q, k, v, unseen = unseen_keys(t, d, nq, window, sinks)
    o64, lse64, pv = ref.window_ref(q, k, v, window, sinks, 1 / math.sqrt(d))
    k[:, :, unseen], v[:, :, unseen] = (largest(k[:, :, unseen].shape, t, s) for s in (1, 2))
    o, lse = window_attention_lse(q, k, v, window, sinks)
    ref.check_o(o, o64, pv)
    ref.check_lse(lse, lse64)


@pytest.mark.parametrize("d", [64, 128])
@CHUNKS
def test_gradients_beside_masked_keys_of_the_largest_size(d, nq, window, sinks):
    """dO V^T of such a key passes fp32; its weight is 0 all the same."""
    q, k, v, unseen = unseen_keys(torch.bfloat16, d, nq, window, sinks)
    do = upstream(q)
    plain = (q, k.clone(), v.clone(), do)
    k[:, :, unseen], v[:, :, unseen] = (largest(k[:, :, unseen].shape, k.dtype, s) for s in (1, 2))
    check_grads(grads_of(q, k, v, do, window, sinks), *plain, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
def test_upstream_of_rows_that_see_nothing(d):
    """Queries before the first key have no weight, whatever (finite) gradient comes for them."""
    q, k, v = make(2, 4, 2, 300, 100, d, seed=3)
    do = upstream(q)
    do[:, :, :200] = 0
    plain = (q, k, v, do.clone())
    do[:, :, :200] = largest(do[:, :, :200].shape, do.dtype, 3)
    check_grads(grads_of(q, k, v, do, 30, 2), *plain, 30, 2)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(16, 4), (60, 0), (500, 0)])
def test_backward_beside_partly_masked_keys_of_the_largest_size(d, window, sinks):
    """Key 150 carries a value whose product with some upstream rows passes fp32: the rows that
    see it are lost, as in the definition, and no other row is."""
    n = 300
    q, k, v = make(1, 2, 2, n, n, d, seed=5)
    do = upstream(q)
    want = ref.window_grad_ref(q, k, v, do, window, sinks, 1 / math.sqrt(d))
    v[:, :, 150] = torch.finfo(v.dtype).max
    dq, _, _ = grads_of(q, k, v, do, window, sinks)
    away = ~ref.visible(n, n, window, sinks, "cuda")[:, 150]
    g, lim = (x[:, :, away] for x in want["dq"])
    assert ((dq[:, :, away].double() - g).abs() <= lim).all()


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hkv,cap,window", [(16, 1, 300, 400), (16, 2, 3000, 2900), (16, 16, 60, 50), (16, 1, 12000, 11000)])
def test_a_cache_key_of_nan_or_infinity_reaches_the_tokens_that_see_it(t, d, b, hkv, cap, window):
    """One split and several, four warps a block and eight; three tokens, the last of which alone
    see the key. It may hold the largest value where they do not."""
    from blackflash_b200 import window_decode
    tokens, base = 3, cap - 17
    gen = torch.Generator(device="cuda").manual_seed(cap)

    def rnd(*s):
        return torch.randn(s, generator=gen, device="cuda").to(t)
    q, k, v = rnd(b, 2 * hkv, tokens, d), rnd(b, hkv, cap, d), rnd(b, hkv, cap, d)
    n = torch.full((b,), cap, dtype=torch.int32, device="cuda")
    n[::2] = cap // 2
    want, want_lse = window_decode(q, k, v, n, window, want_lse=True)
    for value in (math.nan, math.inf):
        bad = k.clone()
        rows = torch.zeros(b, 2 * hkv, tokens, dtype=torch.bool, device="cuda")
        for i in range(b):
            key = (base + i) if i % 2 else cap // 2 - 1 - i % 3
            bad[i, -1, key, 7] = value
            pos = int(n[i]) - tokens + torch.arange(tokens, device="cuda")
            seen = (key <= pos) & (key > pos - window)
            # inf times a negative number is -inf, a weight of 0: looked at in the other test alone.
            rows[i, -2:] = seen
            if value == math.inf:
                q[i, -2:, :, 7] = q[i, -2:, :, 7].abs() + 0.01
        if value == math.inf:
            want, want_lse = window_decode(q, k, v, n, window, want_lse=True)
        got, lse = window_decode(q, bad, v, n, window, want_lse=True)
        same_outside(got, want, rows)
        same_outside(lse, want_lse, rows)
    # The newest token's key and value at their largest: the tokens before it do not see them.
    k2, v2 = k.clone(), v.clone()
    for i in range(b):
        k2[i, :, int(n[i]) - 1], v2[i, :, int(n[i]) - 1] = (torch.finfo(t).max * s for s in (-1, 1))
    got = window_decode(q, k2, v2, n, window)
    assert torch.equal(got[:, :, :-1], want[:, :, :-1])
