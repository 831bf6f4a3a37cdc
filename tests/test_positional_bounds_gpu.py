"""Every entry point of the position-aware operators, called through the C ABI with each output
and workspace exactly as large as documented and set between guard bytes, and each input a view
whose neighbours are NaN: nothing outside is written, nothing outside counts."""
import ctypes
import math

import pytest
import torch

import positional_ref as ref

pytestmark = pytest.mark.gpu

GUARD, FILL = 4096, 0xA5


class Guarded:
    """A buffer of `count` elements between two guards; data at an `align`-byte boundary and no more."""

    def __init__(self, count, t, align):
        self.bytes = count * torch.empty(0, dtype=t).element_size()
        self.raw = torch.full((2 * GUARD + self.bytes + 256,), FILL, dtype=torch.uint8, device="cuda")
        assert self.raw.data_ptr() % 256 == 0
        self.at = GUARD + align
        self.data = self.raw[self.at: self.at + self.bytes].view(t)
        self.ptr = self.data.data_ptr()
        assert not self.bytes or (self.ptr % align == 0 and self.ptr % (2 * align) != 0)

    def check(self, name):
        torch.cuda.synchronize()
        assert (self.raw[: self.at] == FILL).all(), f"{name}: bytes before it"
        assert (self.raw[self.at + self.bytes:] == FILL).all(), f"{name}: bytes after it"


def inside(shape, t, gen, pad=3):
    """A random [b, h, n, d] view with `pad` rows and heads of NaN on every side."""
    b, h, n, d = shape
    big = torch.full((b + 2, h + 2, n + 2 * pad, d), math.nan, dtype=t, device="cuda")
    view = big[1: b + 1, 1: h + 1, pad: pad + n]
    view.copy_(torch.randn(shape, generator=gen, device="cuda"))
    return view


def bf_view(x):
    from blackflash_b200 import _lib
    return _lib.View(x.data_ptr(), (ctypes.c_longlong * 3)(*x.stride()[-4:-1] if x.dim() == 4 else (0, *x.stride()[:2])))


@pytest.fixture(scope="module")
def lib():
    from blackflash_b200 import _lib
    return _lib.load()


def ok(lib, rc):
    assert rc == 0, lib.blackflash_last_error()
    torch.cuda.synchronize()


STREAM = ctypes.c_void_p(0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 1), (3, 3)])
@pytest.mark.parametrize("n,window,sinks", [(1, 1, 0), (129, 40, 2), (300, 100, 130), (1500, 64, 4)])
def test_window_forward_and_backward_stay_in_their_buffers(lib, d, hq, hkv, n, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(n)
    b, t = 2, torch.bfloat16
    q, do = inside((b, hq, n, d), t, gen), inside((b, hq, n, d), t, gen)
    k, v = inside((b, hkv, n, d), t, gen), inside((b, hkv, n, d), t, gen)
    scale = 1 / math.sqrt(d)
    o, lse = Guarded(b * hq * n * d, t, 32), Guarded(b * hq * n, torch.float32, 4)
    sizes = (b, hq, hkv, n, n, d, window, sinks)
    torch.cuda.synchronize()
    views = [bf_view(x) for x in (q, k, v)]
    ok(lib, lib.blackflash_window_fwd(*views, o.ptr, lse.ptr, *sizes, scale, 0, STREAM))
    o64, lse64, pv = ref.window_ref(q, k, v, window, sinks, scale)
    ref.check_o(o.data.view(b, hq, n, d), o64, pv)
    ref.check_lse(lse.data.view(b, hq, n), lse64)
    outs = {"dq": Guarded(b * hq * n * d, t, 32), "dk": Guarded(b * hkv * n * d, t, 32), "dv": Guarded(b * hkv * n * d, t, 32)}
    ws = Guarded(lib.blackflash_window_bwd_workspace_bytes(*sizes), torch.uint8, 32)
    ok(lib, lib.blackflash_window_bwd(*views, o.ptr, bf_view(do), lse.ptr, *(x.ptr for x in outs.values()), ws.ptr, ws.bytes,
                                      *sizes, scale, STREAM))
    want = ref.window_grad_ref(q, k, v, do, window, sinks, scale)
    for name, buf in {**outs, "o": o, "lse": lse, "workspace": ws}.items():
        buf.check(name)
        if name in want:
            g, lim = want[name]
            assert ((buf.data.view(g.shape).double() - g).abs() <= lim).all(), name


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("b,hq,hkv,t,cap,window,sinks", [
    (3, 2, 1, 1, 1, 1, 0), (3, 6, 2, 3, 129, 40, 2), (2, 17, 1, 1, 300, 300, 0), (3, 8, 2, 2, 5000, 4000, 9),
    (1, 8, 1, 1, 30000, 29000, 0),
])
def test_window_decode_stays_in_its_buffers(lib, d, dtype, b, hq, hkv, t, cap, window, sinks):
    gen = torch.Generator(device="cuda").manual_seed(cap)
    q = torch.randn(b, hq, t, d, generator=gen, device="cuda").to(dtype)
    k, v = inside((b, hkv, cap, d), dtype, gen), inside((b, hkv, cap, d), dtype, gen)
    n = torch.tensor([cap, cap // 2, 0][:b], dtype=torch.int32, device="cuda")
    scale = 1 / math.sqrt(d)
    need = lib.blackflash_decode_workspace_bytes(b, hq, hkv, t, 0, cap, d, window, sinks)
    o, lse, ws = Guarded(b * hq * t * d, dtype, 16), Guarded(b * hq * t, torch.float32, 4), Guarded(need, torch.uint8, 32)
    torch.cuda.synchronize()
    ok(lib, lib.blackflash_window_decode(q.data_ptr(), bf_view(k), bf_view(v), n.data_ptr(), o.ptr, lse.ptr,
                                         ws.ptr if need else None, need, b, hq, hkv, t, cap, d, window, sinks, scale,
                                         int(dtype == torch.float16), STREAM))
    o64, lse64, pv = ref.decode_ref(q, k, v, n, window, sinks, scale)
    ref.check_o(o.data.view(b, hq, t, d), o64, pv)
    ref.check_lse(lse.data.view(b, hq, t), lse64)
    for name, buf in (("o", o), ("lse", lse), ("workspace", ws)):
        buf.check(name)


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("b,hq,hkv,t,p,cap", [
    (3, 4, 2, 1, 1, 1), (5, 10, 2, 1, 300, 17), (3, 4, 2, 2, 77, 0),  # the prefix read with the cache
    (5, 10, 2, 3, 300, None), (70, 4, 1, 3, 257, None), (2, 16, 1, 9, 200, None),  # by a kernel of its own
])
def test_prefix_decode_stays_in_its_buffers(lib, d, dtype, b, hq, hkv, t, p, cap):
    gen = torch.Generator(device="cuda").manual_seed(p)
    if cap is None:
        cap = (33 << 20) // (b * hkv * ((hq // hkv * t + 15) // 16) * d * 4) + 1
    q = torch.randn(b, hq, t, d, generator=gen, device="cuda").to(dtype)
    kp, vp = inside((1, hkv, p, d), dtype, gen)[0], inside((1, hkv, p, d), dtype, gen)[0]
    k, v = (torch.full((b + 2, hkv, max(cap, 1) + 1, d), math.nan, dtype=dtype, device="cuda")[1:-1, :, :cap] for _ in range(2))
    n = torch.randint(0, min(cap, 60) + 1, (b,), device="cuda", dtype=torch.int32, generator=gen)
    k[:, :, :60] = torch.randn(k[:, :, :60].shape, generator=gen, device="cuda")
    v[:, :, :60] = torch.randn(v[:, :, :60].shape, generator=gen, device="cuda")
    scale = 1 / math.sqrt(d)
    need = lib.blackflash_decode_workspace_bytes(b, hq, hkv, t, p, cap, d, 2 ** 31 - 1, 0)
    o, lse, ws = Guarded(b * hq * t * d, dtype, 16), Guarded(b * hq * t, torch.float32, 4), Guarded(need, torch.uint8, 32)
    torch.cuda.synchronize()
    ok(lib, lib.blackflash_prefix_decode(q.data_ptr(), bf_view(kp), bf_view(vp), bf_view(k), bf_view(v), n.data_ptr(), o.ptr,
                                         lse.ptr, ws.ptr if need else None, need, b, hq, hkv, t, p, cap, d, scale,
                                         int(dtype == torch.float16), STREAM))
    o64, lse64, pv = ref.decode_ref(q, k, v, n, 1 << 40, 0, scale, kp, vp)
    ref.check_o(o.data.view(b, hq, t, d), o64, pv)
    ref.check_lse(lse.data.view(b, hq, t), lse64)
    for name, buf in (("o", o), ("lse", lse), ("workspace", ws)):
        buf.check(name)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("n,d,rot", [(1, 64, 64), (7, 80, 20), (301, 12, 6), (33, 2, 2), (130, 1024, 1024)])
def test_rotary_stays_in_its_buffers(lib, t, interleaved, n, d, rot):
    """Outputs at the least alignment, a pair; then at 16 bytes, where whole vectors are written."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    b, hq, hk = 2, 3, 1
    q, k = inside((b, hq, n, d), t, gen), inside((b, hk, n, d), t, gen)
    pos = torch.randint(0, 1 << 20, (b, n), generator=gen, device="cuda", dtype=torch.int32)
    freqs = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    size = q.element_size()
    code = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[t]
    outs = []
    for align in (2 * size, 16):
        qo, ko = Guarded(b * hq * n * d, t, align), Guarded(b * hk * n * d, t, align)
        torch.cuda.synchronize()
        ok(lib, lib.blackflash_rotary(bf_view(q), bf_view(k), qo.ptr, ko.ptr, pos.data_ptr(), 0, 1, freqs.data_ptr(), b, hq, hk,
                                      n, d, rot, interleaved, 1.25, 0, code, STREAM))
        qo.check("Q_out"), ko.check("K_out")
        outs.append((qo.data.view(q.shape), ko.data.view(k.shape)))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    for got, x in zip(outs[0], (q, k)):
        want = ref.rotary64(x, pos, freqs, bool(interleaved), 1.25)
        # Output rounding; five fp32 steps of the pair's size for cos, sin and the sum (|x| < 6 here).
        lim = ref.half_step(t) * want.abs() + 12 * 1.25 * 5 * 2.0 ** -23 + torch.finfo(t).smallest_normal
        assert ((got.double() - want).abs() <= lim).all()


def test_backward_on_the_engines_thread_and_another_stream():
    """A training step on a side stream: the backward runs on the engine's thread, on that stream."""
    from blackflash_b200 import window_attention_with_grad
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(2, h, 400, 64, generator=gen, device="cuda").to(torch.bfloat16) for h in (4, 2, 2, 4))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(window_attention_with_grad(*leaves, 100, 4), leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
        o = window_attention_with_grad(*leaves, 100, 4)
        o.backward(do)
    side.synchronize()
    for x, y in zip(leaves, want):
        assert torch.equal(x.grad, y)
