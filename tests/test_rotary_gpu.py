"""Rotary positions on the GPU, against fp64 with counted roundings."""
import pytest
import torch

import positional_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def bound(x, want, positions, freqs, interleaved, rot, amplitude):
    """Output rounding, and per product: cos and sin within 3 steps of fp32 (sincospi, its
    first-order correction, the amplitude), the two products and their sum half a step each.

    The angle n * f itself is rounded to fp64: once here (half a step, n f 2^-53), and three
    times in the kernel (1 / 2 pi, f / 2 pi, the product), so the two angles differ by up to
    4 n f 2^-53. That is 5e-5 at n = 10^11, where it exceeds fp32's step; below n = 10^7 it
    does not count."""
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    size = torch.zeros_like(want)
    pair = (x[..., lo].double().abs() + x[..., hi].double().abs()) * abs(amplitude)
    angle = 4 * 2.0 ** -53 * (positions.double().abs()[..., None] * freqs)[..., None, :, :]
    each = pair * (5 * 2.0 ** -23 + angle)
    size[..., lo], size[..., hi] = each, each
    return ref.half_step(x.dtype) * want.abs() + size + 1e-30


def check(got, x, positions, freqs, interleaved, amplitude=1.0, sign=1.0):
    want = ref.rotary64(x, positions, freqs, interleaved, amplitude, sign)
    err = (got.double() - want).abs()
    lim = bound(x, want, positions, freqs, interleaved, 2 * freqs.numel(), amplitude)
    assert got.is_contiguous() and got.dtype == x.dtype
    # An fp16 or bf16 result below the normal range is off by half its least step.
    lim = lim + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    bad = int((err > lim).sum())
    assert bad == 0, (bad, float((err / lim).max()))
    rot = 2 * freqs.numel()
    assert torch.equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (128, 64), (128, 32), (64, 42), (80, 2), (2, 2), (96, 90),
                                   (1024, 1024), (12, 8), (10, 6)])
def test_rotary_layouts(t, interleaved, d, rot):
    from blackflash_b200 import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(rot, 500000.0)
    gen = torch.Generator(device="cuda").manual_seed(d + rot)
    for b, hq, hk, n in ((1, 1, 1, 1), (3, 5, 2, 17), (2, 4, 1, 301)):
        q, k = (torch.randn(b, h, n, d, generator=gen, device="cuda").to(t) for h in (hq, hk))
        pos = torch.randint(0, 1 << 20, (b, n), generator=gen, device="cuda", dtype=torch.int32)
        a, c = rotary(q, k, pos, freqs, interleaved, 1.25)
        check(a, q, pos, freqs, interleaved, 1.25)
        check(c, k, pos, freqs, interleaved, 1.25)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_views_positions_and_inverse(interleaved):
    """Token-major views, odd offsets, shared [N] and int64 positions, far and negative ones."""
    from blackflash_b200 import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(32)
    for t in TYPES:
        x = torch.randn(2, 50, 6, 130, device="cuda").to(t)
        views = [x[..., :64].transpose(1, 2), x[..., 2:66].transpose(1, 2), x[:, ::2, :, 66:].transpose(1, 2),
                 x[:, :1, :1, :64].expand(2, 50, 6, 64).transpose(1, 2)]
        for v in views:
            n = v.shape[2]
            for pos in (torch.arange(n, device="cuda"), torch.arange(n, device="cuda", dtype=torch.int32) - 25,
                        (torch.arange(2 * n, device="cuda") * 1234567891).view(2, n)):
                a, b = rotary(v, v[:, :1], pos, freqs, interleaved)
                check(a, v, pos, freqs, interleaved)
                check(b, v[:, :1], pos, freqs, interleaved)
            a, b = rotary(v, v[:, :0], pos, freqs, interleaved, inverse=True)
            check(a, v, pos, freqs, interleaved, sign=-1.0)
            assert b.shape == v[:, :0].shape


def test_rotary_gradient_formula_and_differences():
    from blackflash_b200 import rotary_frequencies, rotary_with_grad
    freqs, amp = rotary_frequencies(32, scaling="by-parts", factor=4.0, original_length=64)
    gen = torch.Generator(device="cuda").manual_seed(0)
    for interleaved in (False, True):
        q, k = (torch.randn(2, h, 9, 40, generator=gen, device="cuda").requires_grad_(True) for h in (3, 1))
        pos = torch.arange(100, 109, device="cuda")
        a, b = rotary_with_grad(q, k, pos, freqs, interleaved, amp)
        ga, gb = (torch.randn(x.shape, generator=gen, device="cuda") for x in (a, b))
        gq, gk = torch.autograd.grad((a, b), (q, k), (ga, gb))
        check(gq, ga, pos, freqs, interleaved, amp, -1.0)
        check(gk, gb, pos, freqs, interleaved, amp, -1.0)
        # The map is linear: a difference of any size gives the gradient, but for fp32 rounding.
        dq = torch.randn(q.shape, generator=gen, device="cuda")
        a2, _ = rotary_with_grad(q + dq, k, pos, freqs, interleaved, amp)
        left, right = ((a2 - a).double() * ga.double()).sum(), (dq.double() * gq.double()).sum()
        # Each of the 2160 terms carries a few steps of values of about 5.
        assert abs(left - right) <= 2160 * 5 * 8 * 2.0 ** -24
        # A gradient that is one number for all (a sum's), and a broadcast leaf.
        row = torch.randn(1, 1, 9, 40, generator=gen, device="cuda").requires_grad_(True)
        out = rotary_with_grad(row.expand(2, 3, 9, 40), k, pos, freqs, interleaved, amp)[0]
        g, = torch.autograd.grad(out.sum(), row)
        one = ref.rotary64(torch.ones(2, 3, 9, 40, device="cuda"), pos, freqs, interleaved, amp, -1.0).sum((0, 1))
        assert (g[0, 0].double() - one).abs().max() <= 6 * 8 * 2.0 ** -23


def test_rotary_graph_and_stream():
    from blackflash_b200 import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(64)
    q = torch.randn(4, 8, 1, 64, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([[3], [1000], [0], [77777]], device="cuda", dtype=torch.int32)
    rotary(q, q, pos, freqs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a, b = rotary(q, q, pos, freqs)
    pos += 5
    g.replay()
    torch.cuda.synchronize()
    check(a, q, pos, freqs, False)
    assert torch.equal(a, b)


def test_rotary_empty():
    from blackflash_b200 import rotary, rotary_frequencies
    freqs, _ = rotary_frequencies(64)
    q = torch.zeros(0, 8, 3, 64, device="cuda")
    a, b = rotary(q, q, torch.arange(3, device="cuda"), freqs)
    assert a.shape == b.shape == q.shape
