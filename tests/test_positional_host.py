"""Position-aware operators on the CPU: argument checks of the C ABI and of the Python
layer, workspace plans, frequency tables."""
import math

import pytest
import torch


def view(lib, data=16, strides=(64, 64, 64)):
    import ctypes

    from blackflash_b200 import _lib
    return _lib.View(data, (ctypes.c_longlong * 3)(*strides))


@pytest.fixture(scope="module")
def lib():
    from blackflash_b200 import _lib
    from blackflash_b200.build import build_lib
    build_lib()
    yield _lib.load()
    _lib.load().blackflash_decode_workspace_bytes(1, 1, 1, 1, 0, 1, 64, 1, 0)  # clears the thread's last error


@pytest.mark.parametrize("change", [dict(B=0), dict(Hkv=3), dict(d=32), dict(window=0), dict(sinks=-2)])
def test_window_backward_plans(lib, change):
    ok = dict(B=1, Hq=4, Hkv=2, Nq=300, Nkv=300, d=64, window=50, sinks=0)
    ws = lib.blackflash_window_bwd_workspace_bytes
    assert ws(*ok.values()) == 4 * 6 * 4 * 384            # six words a row of 4 heads, 300 rows padded to 384
    # Sinks that 100 query tiles see come in parts: 128-row fp32 pieces of dV and dK.
    many = ws(*{**ok, "Nq": 12800, "Nkv": 12800, "sinks": 4}.values()) - 4 * 6 * 4 * 12800
    assert many > 0 and many % (2 * 128 * 64 * 4) == 0
    assert ws(*{**ok, **change}.values()) == -1 and lib.blackflash_last_error()
    # Long, and with a whole length of sinks: the parts stay bounded, whatever the length.
    for n, sinks in ((1 << 20, 4), (1 << 20, 128), (1 << 16, 1 << 16), (1 << 20, 1 << 20)):
        parts = ws(1, 8, 8, n, n, 128, 64, sinks) - 4 * 6 * 8 * n
        assert 0 <= parts <= (8 * 148 + 8 * 148) * 2 * 128 * 128 * 4


def test_window_backward_refusals(lib):
    ok, sizes = view(lib), (1, 2, 2, 8, 8, 64, 4, 0, 0.125, None)
    need = lib.blackflash_window_bwd_workspace_bytes(*sizes[:8])
    good = [ok, ok, ok, 32, ok, 16, 32, 32, 32, 32, need]
    for i, bad, text in ((0, None, b"Q:"), (4, view(lib, strides=(64, 3, 64)), b"dO"), (3, None, b"O, dQ"), (5, None, b"lse"),
                         (8, 16, b"O, dQ"), (9, None, b"workspace"), (10, need - 1, b"workspace")):
        args = list(good)
        args[i] = bad
        assert lib.blackflash_window_bwd(*args, *sizes) == 1 and text in lib.blackflash_last_error()
    assert lib.blackflash_window_bwd(*good, *sizes[:8], -1.0, None) == 1


WINDOW = dict(B=1, Hq=2, Hkv=1, Nq=8, Nkv=8, d=64, window=4, sinks=0, scale=0.125, dtype=0)


@pytest.mark.parametrize("change,text", [
    (dict(B=0), b"empty"), (dict(Nkv=0), b"empty"), (dict(Hq=3, Hkv=2), b"multiple"), (dict(d=96), b"d=64"),
    (dict(window=0), b"window"), (dict(sinks=-1), b"sinks"), (dict(scale=0.0), b"scale"),
    (dict(scale=math.nan), b"scale"), (dict(scale=-1.0), b"scale"), (dict(dtype=2), b"dtype"),
    (dict(Nq=(1 << 30) + 1), b"2^30"), (dict(B=70000, Hq=40000, Hkv=40000), b"too large"),
])
def test_window_fwd_refuses_sizes(lib, change, text):
    a = {**WINDOW, **change}
    v = view(lib, strides=(1 << 20, 1 << 14, 64))
    rc = lib.blackflash_window_fwd(v, v, v, 32, None, *(a[x] for x in WINDOW), None)
    assert rc == 1 and text in lib.blackflash_last_error(), lib.blackflash_last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(data=0), b"null"), (dict(data=24), b"aligned"), (dict(strides=(64, 64, 60)), b"strides"),
    (dict(strides=(64, 0, 64)), b"strides"), (dict(strides=(64, 64, -64)), b"strides"),
])
def test_views_are_checked(lib, bad, text):
    ok = view(lib)
    for i in range(3):
        views = [ok, ok, ok]
        views[i] = view(lib, **bad)
        rc = lib.blackflash_window_fwd(*views, 32, None, *{**WINDOW, "Hkv": 2}.values(), None)
        assert rc == 1 and text in lib.blackflash_last_error()
    rc = lib.blackflash_window_fwd(ok, ok, ok, 16, None, *WINDOW.values(), None)
    assert rc == 1 and b"O must" in lib.blackflash_last_error()


def test_decode_plans_and_refusals(lib):
    ws = lib.blackflash_decode_workspace_bytes
    assert ws(1, 8, 2, 1, 0, 64, 64, 64, 0) == 0          # one split: no workspace
    assert ws(1, 8, 2, 1, 0, 100000, 64, 512, 4) == 0     # few keys: one block each
    assert ws(1, 8, 2, 1, 0, 100000, 64, 5000, 4) > 0
    # The plan follows the window, not the capacity.
    assert ws(1, 8, 2, 1, 0, 1 << 30, 128, 512, 4) == ws(1, 8, 2, 1, 0, 1000, 128, 512, 4)
    assert ws(64, 32, 8, 1, 16384, 1024, 128, 2 ** 31 - 1, 0) % 4 == 0
    for bad in ((0, 8, 2, 1, 0, 64, 64, 64, 0), (1, 8, 3, 1, 0, 64, 64, 64, 0), (1, 8, 2, 0, 0, 64, 64, 64, 0),
                (1, 8, 2, 1, 0, 0, 64, 64, 0), (1, 8, 2, 1, -1, 64, 64, 64, 0), (1, 8, 2, 1, 0, 64, 80, 64, 0),
                (1, 8, 2, 1, 0, 64, 64, 0, 0), (1, 8, 2, 1, 0, 64, 64, 4, -1), (1, 1 << 20, 1, 2, 0, 64, 64, 4, 0),
                (65536, 65536, 65536, 1, 0, 64, 64, 4, 0)):
        assert ws(*bad) == -1 and lib.blackflash_last_error(), bad
    v = view(lib)
    need = ws(1, 8, 2, 1, 0, 100000, 64, 5000, 4)
    sizes = (1, 8, 2, 1, 100000, 64, 5000, 4, 0.125, 0, None)
    for args, text in (((None, v, v, 16, 16, None, 16, need), b"Q and O"), ((16, v, v, None, 16, None, 32, need), b"lengths"),
                       ((16, v, v, 16, 16, None, 32, need - 1), b"workspace"), ((16, v, v, 16, 16, None, None, need), b"workspace"),
                       ((16, v, v, 16, 16, None, 16, need), b"workspace"), ((16, None, v, 16, 16, None, 32, need), b"K_cache")):
        assert lib.blackflash_window_decode(*args, *sizes) == 1
        assert text in lib.blackflash_last_error()
    big = 1 << 30
    p = (1, 8, 2, 1, 9000, 50, 64)  # enough keys to be split: with a workspace
    for args, text in (((16, None, v, v, v, 16, 16, None, 32, big), b"prefix"), ((16, v, v, v, None, 16, 16, None, 32, big), b"V_cache"),
                       ((16, v, v, v, v, 16, 16, None, None, big), b"workspace")):
        assert lib.blackflash_prefix_decode(*args, *p, 0.125, 0, None) == 1
        assert text in lib.blackflash_last_error()
    assert lib.blackflash_prefix_decode(16, v, v, v, v, 16, 16, None, 16, big, *p, math.inf, 0, None) == 1


def test_rotary_refusals(lib):
    v = view(lib)
    ok = dict(B=1, Hq=2, Hk=1, N=3, d=64, rot=64, inter=0, amp=1.0, inv=0, dtype=0)
    for change in (dict(B=0), dict(N=0), dict(Hq=0, Hk=0), dict(Hq=-1), dict(Hq=70000), dict(d=65), dict(d=2048),
                   dict(rot=0), dict(rot=66), dict(rot=7), dict(amp=math.inf), dict(dtype=3)):
        a = {**ok, **change}
        assert lib.blackflash_rotary(v, v, 16, 16, 16, 0, 0, 16, *a.values(), None) == 1, change
        assert lib.blackflash_last_error()
    for args in ((None, v, 16, 16, 16, 0, 0, 16), (v, v, None, 16, 16, 0, 0, 16), (v, v, 16, 16, None, 0, 0, 16),
                 (v, v, 16, 16, 16, 0, 0, None), (view(lib, data=18), v, 16, 16, 16, 0, 0, 16), (v, v, 16, 18, 16, 0, 0, 16),
                 (view(lib, strides=(64, 63, 64)), v, 16, 16, 16, 0, 0, 16), (view(lib, strides=(64, -64, 64)), v, 16, 16, 16, 0, 0, 16)):
        assert lib.blackflash_rotary(*args, *ok.values(), None) == 1
        assert lib.blackflash_last_error()


def test_python_checks():
    import blackflash_b200 as bf
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    q, n = z(1, 2, 4, 64), torch.zeros(1, dtype=torch.int32)
    f = torch.zeros(32, dtype=torch.float64)
    from blackflash_b200.build import build_torch_ext
    build_torch_ext()
    for call in (lambda: bf.window_attention(q, q, q, 4), lambda: bf.window_attention(q.float(), q, q, 4),
                 lambda: bf.window_attention_lse(None, q, q, 4), lambda: bf.window_decode(q, q, q, n, 4),
                 lambda: bf.prefix_decode(q, q[0], q[0], q, q, n), lambda: bf.rotary(q, q, n, f)):
        with pytest.raises(RuntimeError, match="must be a"):
            call()
    with pytest.raises(RuntimeError, match="must have 4 axes"):  # a message with a number in it
        bf.window_attention(q[0], q, q, 4)
    for kw in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=4, base=1.0), dict(rotary_dim=4, factor=0.5),
               dict(rotary_dim=4, scaling="cubic"), dict(rotary_dim=2, scaling="ntk", factor=2.0),
               dict(rotary_dim=4, scaling="by-parts", factor=2.0)):
        with pytest.raises(RuntimeError):
            bf.rotary_frequencies(**kw, device="cpu")


def test_rotary_frequency_scalings():
    from blackflash_b200 import rotary_frequencies
    f, a = rotary_frequencies(64, 10000.0, device="cpu")
    assert a == 1.0 and f.dtype == torch.float64 and f[0] == 1.0 and abs(f[1] / 10000 ** (-1 / 32) - 1) < 1e-15
    assert torch.equal(rotary_frequencies(64, 10000.0, "linear", 8.0, device="cpu")[0], f / 8)
    g, _ = rotary_frequencies(64, 10000.0, "ntk", 8.0, device="cpu")
    assert g[0] == 1.0 and abs(g[-1] * 8 / f[-1] - 1) < 1e-12
    g, a = rotary_frequencies(64, 10000.0, "by-parts", 8.0, 4096, device="cpu")
    assert torch.equal(g[:5], f[:5]) and torch.allclose(g[-5:], f[-5:] / 8, rtol=1e-14, atol=0)
    assert (g[1:] < g[:-1]).all() and abs(a - (1 + 0.1 * math.log(8))) < 1e-15


@pytest.mark.parametrize("rot,base,length,fast,slow", [
    (64, 1e4, 100, 64.0, 32.0),    # every pair turns less than beta_slow times: the fastest 15.9
    (64, 1e4, 4, 32.0, 1.0),       # 0.64 turns
    (64, 1e4, 150, 32.0, 1.0),     # the fastest pair (23.9 turns) lies inside the ramp
    (32, 1e4, 1 << 24, 32.0, 1.0),  # every pair turns more than beta_fast times: the slowest 475
    (16, 100.0, 4096, 32.0, 8.0),  # the slowest pair (11.6 turns) lies inside the ramp
    (2, 1e4, 4096, 32.0, 1.0), (128, 5e5, 8192, 32.0, 1.0),
])
def test_by_parts_follows_the_turns_of_each_pair(rot, base, length, fast, slow):
    """Pairs above beta_fast turns stay, those below beta_slow are divided by the factor, and
    between them the share of the divided frequency rises by equal steps."""
    from blackflash_b200 import rotary_frequencies
    factor = 8.0
    f = rotary_frequencies(rot, base, device="cpu")[0]
    g = rotary_frequencies(rot, base, "by-parts", factor, length, fast, slow, device="cpu")[0]
    turns = length * f / (2 * math.pi)
    share = (1 - g / f) / (1 - 1 / factor)  # 0: kept, 1: divided; fp64 rounding alone is off
    assert (share[turns > fast].abs() < 1e-12).all() and ((share[turns < slow] - 1).abs() < 1e-12).all()
    assert ((share > -1e-12) & (share < 1 + 1e-12)).all()
    inside = (share > 1e-9) & (share < 1 - 1e-9)
    steps = share[inside].diff()
    assert (steps > 0).all() and (steps.numel() < 2 or (steps - steps[0]).abs().max() < 1e-12)
    # The ramp spans the whole pairs around the two bounds, so its step is known.
    ends = [rot * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
    if steps.numel():
        assert abs(steps[0] * (math.ceil(ends[1]) - math.floor(ends[0])) - 1) < 1e-9


HUGE_SIZES = """
from blackflash_b200 import _lib
lib = _lib.load()
def refused(x):
    assert x == -1 and lib.blackflash_last_error(), x
big = 1 << 30
for b, hq, hkv, t in ((big, big, big, 256), (big, big, big, 16), (big, big, big, 1), (1 << 16, 1 << 16, 1 << 16, 1 << 20),
                      (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 1), (1 << 11, 1 << 10, 1 << 10, 1 << 10)):
    for p, c in ((0, 64), (big, 0), (big, big)):
        refused(lib.blackflash_decode_workspace_bytes(b, hq, hkv, t, p, c, 64, 4, 0))
# The most rows, and the most keys, that are taken.
assert lib.blackflash_decode_workspace_bytes(2 ** 31 - 1, 1, 1, 1, big, big, 128, 2 ** 31 - 1, 2 ** 31 - 1) > 0
assert lib.blackflash_decode_workspace_bytes(1 << 20, 1 << 10, 1 << 10, 1, big, big, 128, 2 ** 31 - 1, 0) > 0
for b, hq, hkv, nq, nkv, w, s in ((big, big, big, big, big, 4, 0), (1 << 16, 1 << 16, 1 << 16, big, 1, 4, 0),
                                  (1 << 20, 1 << 20, 1, big, big, big, big), (1 << 16, 1, 1, big, 1, 4, 0),
                                  (1 << 20, 1, 1, 1, big, 4, 0)):
    refused(lib.blackflash_window_bwd_workspace_bytes(b, hq, hkv, nq, nkv, 64, w, s))
assert lib.blackflash_window_bwd_workspace_bytes(1, 8, 8, big, big, 64, big, big) >= 4 * 6 * 8 * big
assert lib.blackflash_window_bwd_workspace_bytes(1, 1, 1, 1, big, 128, big, big) > 0
print("refused")
"""


def test_sizes_whose_products_pass_64_bits():
    """Refused, not divided by: in a process of its own, which a division by zero would end."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", HUGE_SIZES], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "refused" in out.stdout, (out.returncode, out.stderr[-2000:])
