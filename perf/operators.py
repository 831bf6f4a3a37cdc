"""Measured cases of the position-aware attention operators.

Three operators are measured, each in the forms that training and serving use:

  window   causal attention with a sliding window and a few first tokens that stay
           visible (sinks), grouped KV heads: the prompt pass ("window_fwd"), the
           training step ("window_train": output and gradients) and the step of one or
           a few new tokens against a cache ("window_decode");
  prefix   a decoding step of a batch whose sequences share one long prefix
           ("prefix_decode");
  rotary   rotary positions applied to Q and K ("rotary"), with the gradients of a
           training step ("rotary_train").

`run` computes a case in plain fp32 torch operations, or, where `own` is true, by the
public calls of blackflash_b200. `exact` computes the same outputs in fp64.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A short prompt, small grid: the library's B=4 H=8 N=1024 configuration with grouped KV heads.
        dict(name="window_fwd_prompt_1k", op="window_fwd", b=4, hq=8, hkv=2, nq=1024, nkv=1024, d=64, window=256,
             sinks=4, type="bf16"),
        # A long prompt, the B=8 H=16 N=8192 configuration's length at head dimension 128.
        dict(name="window_fwd_prompt_8k", op="window_fwd", b=4, hq=16, hkv=4, nq=8192, nkv=8192, d=128, window=1024,
             sinks=4, type="bf16"),
        # One chunk of a chunked prompt: fewer queries than keys, odd sizes, fp16, no sinks.
        dict(name="window_fwd_chunk_odd", op="window_fwd", b=3, hq=12, hkv=12, nq=777, nkv=5001, d=64, window=2047,
             sinks=0, type="fp16"),
        # A training step of a windowed layer, one KV head per query head.
        dict(name="window_train_4k", op="window_train", b=2, hq=16, hkv=16, nq=4096, nkv=4096, d=64, window=1024,
             sinks=4, type="bf16"),
        # A training step with grouped KV heads, odd length, a whole tile of sinks.
        dict(name="window_train_gqa_odd", op="window_train", b=1, hq=32, hkv=8, nq=6143, nkv=6143, d=128, window=2048,
             sinks=128, type="bf16"),
        # One sequence, one token: the smallest serving step.
        dict(name="window_decode_single", op="window_decode", b=1, hq=8, hkv=2, t=1, cap=4096, d=64, window=512,
             sinks=4, type="bf16"),
        # A full serving batch, one token each, ragged lengths.
        dict(name="window_decode_batch", op="window_decode", b=64, hq=32, hkv=8, t=1, cap=8192, d=128, window=4096,
             sinks=4, type="bf16"),
        # Three drafted tokens a sequence over a long cache, odd capacity, one KV head per query head, fp16.
        dict(name="window_decode_draft", op="window_decode", b=5, hq=16, hkv=16, t=3, cap=30001, d=64, window=10000,
             sinks=16, type="fp16"),
        # A few requests behind one system prompt.
        dict(name="prefix_decode_few", op="prefix_decode", b=4, hq=8, hkv=2, t=1, prefix=1000, cap=128, d=64,
             type="bf16"),
        # A serving batch behind one long document.
        dict(name="prefix_decode_batch", op="prefix_decode", b=64, hq=32, hkv=8, t=1, prefix=16384, cap=1024, d=128,
             type="bf16"),
        # Positions of one decoding step, far out in a long context.
        dict(name="rotary_decode", op="rotary", b=64, hq=32, hkv=8, n=1, d=128, rot=128, interleaved=False,
             type="bf16", heads_last=False),
        # Positions of a training step on the projections' own [B, N, H, d] layout, part of the head, interleaved.
        dict(name="rotary_train_partial", op="rotary_train", b=4, hq=32, hkv=8, n=4095, d=128, rot=64,
             interleaved=True, type="bf16", heads_last=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges, no dearer than the largest of its kind."""
    op = rng.choice(["window_fwd", "window_train", "window_decode", "prefix_decode", "rotary", "rotary_train"])
    d = rng.choice([64, 128])
    hkv = rng.choice([1, 2, 3, 4, 8])
    g = rng.choice([1, 1, 2, 3, 4, 8])
    half = rng.choice(["bf16", "bf16", "fp16"])
    sinks = rng.choice([0, 1, 4, 16, 100, 128])
    if op == "window_fwd":
        nq = _log_int(rng, 1, 8192)
        nkv = nq + rng.choice([0, 0, _log_int(rng, 1, 8192)])
        b = max(1, min(rng.choice([1, 2, 3, 4]), 64 * 8192 // (hkv * g * nq)))
        return dict(op=op, b=b, hq=hkv * g, hkv=hkv, nq=nq, nkv=nkv, d=d, window=_log_int(rng, 1, 1024), sinks=sinks,
                    type=half)
    if op == "window_train":
        nq = _log_int(rng, 1, 6143)
        g = min(g, 4)
        b = max(1, min(rng.choice([1, 2, 3]), 32 * 6143 // (hkv * g * nq)))
        return dict(op=op, b=b, hq=hkv * g, hkv=hkv, nq=nq, nkv=nq, d=d, window=_log_int(rng, 1, 2048), sinks=sinks,
                    type="bf16")
    if op == "window_decode":
        cap = _log_int(rng, 1, 32768)
        b = max(1, min(_log_int(rng, 1, 64), 64 * 8192 // cap))
        return dict(op=op, b=b, hq=hkv * g, hkv=hkv, t=rng.choice([1, 1, 1, 2, 3, 5]), cap=cap, d=d,
                    window=_log_int(rng, 1, 4096), sinks=sinks, type=half)
    if op == "prefix_decode":
        return dict(op=op, b=_log_int(rng, 1, 64), hq=hkv * min(g, 4), hkv=hkv, t=rng.choice([1, 1, 1, 2, 5]),
                    prefix=_log_int(rng, 1, 8192), cap=_log_int(rng, 8, 512), d=d, type=half)
    n = _log_int(rng, 1, 4095)
    b = max(1, min(_log_int(rng, 1, 64), 4 * 4095 // n))
    return dict(op=op, b=b, hq=hkv * min(g, 4), hkv=hkv, n=n, d=d, rot=rng.choice([d, d // 2, d // 4, 3 * d // 4 - 6]),
                interleaved=rng.random() < 0.5, type=rng.choice(["bf16", "fp16", "fp32"]),
                heads_last=rng.random() < 0.5)


def _visible(p, window, sinks):
    """Keys that the query at position p sees: the last `window` up to itself, and the sinks before those."""
    return min(window, p + 1) + min(sinks, max(0, p + 1 - window))


def _lengths(case):
    """Tokens in each sequence's cache: spread evenly from a sixteenth of the capacity to all of it."""
    b, cap, t = case["b"], case["cap"], case["t"]
    lo = max(min(t, cap), cap // 16)
    return [lo + (cap - lo) * (i + 1) // b for i in range(b)]


def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    if op in ("window_fwd", "window_train"):
        nq, nkv = case["nq"], case["nkv"]
        pairs = b * hq * sum(_visible(p, case["window"], case["sinks"]) for p in range(nkv - nq, nkv))
        # Keys that some query sees: the first query's window on, and the sinks before it.
        first = max(0, nkv - nq - case["window"] + 1)
        keys = nkv - first + min(case["sinks"], first)
        q, kv = b * hq * nq * d * size, b * hkv * keys * d * size
        if op == "window_fwd":
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * d}
        # Forward: two products. Backward: five (the scores again, dP, dV, dK, dQ).
        return {"bytes": 4 * q + 4 * kv, "flops": (4 + 10) * pairs * d}
    if op == "window_decode":
        keys = pairs = 0
        for n in _lengths(case):
            first = max(0, n - case["t"] - case["window"] + 1)
            keys += n - first + min(case["sinks"], first)
            pairs += sum(_visible(p, case["window"], case["sinks"]) for p in range(n - case["t"], n) if p >= 0)
        return {"bytes": 2 * b * hq * case["t"] * d * size + 2 * hkv * keys * d * size, "flops": 4 * hq * pairs * d}
    if op == "prefix_decode":
        keys = sum(_lengths(case))
        pairs = sum(max(0, n - case["t"] + 1 + i) for n in _lengths(case) for i in range(case["t"]))
        pairs += b * case["t"] * case["prefix"]
        return {"bytes": 2 * b * hq * case["t"] * d * size + 2 * hkv * (keys + case["prefix"]) * d * size,
                "flops": 4 * hq * pairs * d}
    elements = b * (hq + hkv) * case["n"] * d
    passes = 2 if op == "rotary_train" else 1
    # Each rotated pair takes four products and two sums.
    return {"bytes": passes * 2 * elements * size, "flops": passes * 3 * b * (hq + hkv) * case["n"] * case["rot"]}


# ------------------------------------------------------------------ inputs

def _randn(gen, *shape, type):
    return torch.randn(shape, generator=gen, device=_DEV).to(_TYPES[type])


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    op, ty = case["op"], case["type"]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    st = {"case": case}
    if op in ("window_fwd", "window_train"):
        st["q"] = _randn(gen, b, hq, case["nq"], d, type=ty)
        st["k"] = _randn(gen, b, hkv, case["nkv"], d, type=ty)
        st["v"] = _randn(gen, b, hkv, case["nkv"], d, type=ty)
        if op == "window_train":
            st["do"] = _randn(gen, b, hq, case["nq"], d, type=ty)
            for x in ("q", "k", "v"):
                st[x].requires_grad_(True)
    elif op in ("window_decode", "prefix_decode"):
        order = torch.randperm(b, generator=gen, device=_DEV)
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=_DEV)[order].contiguous()
        st["q"] = _randn(gen, b, hq, case["t"], d, type=ty)
        st["k"] = _randn(gen, b, hkv, case["cap"], d, type=ty)
        st["v"] = _randn(gen, b, hkv, case["cap"], d, type=ty)
        if op == "prefix_decode":
            st["kp"] = _randn(gen, hkv, case["prefix"], d, type=ty)
            st["vp"] = _randn(gen, hkv, case["prefix"], d, type=ty)
    else:
        n = case["n"]
        for x, h in (("q", hq), ("k", hkv)):
            if case["heads_last"]:  # the projection's output, seen as [B, H, N, d]
                st[x] = _randn(gen, b, n, h, d, type=ty).transpose(1, 2)
            else:
                st[x] = _randn(gen, b, h, n, d, type=ty)
            if op == "rotary_train":
                st[x].requires_grad_(True)
                st["d" + x] = _randn(gen, b, h, n, d, type=ty)
        # Each sequence starts somewhere in a context of a million tokens.
        start = torch.randint(0, 1 << 20, (b, 1), generator=gen, device=_DEV)
        st["positions"] = (start + torch.arange(n, device=_DEV)).to(torch.int32)
        # Angle per position of each rotated pair, base 500000, stretched fourfold for the long context.
        pair = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=_DEV)
        st["freqs"] = 500000.0 ** (-pair / case["rot"]) / 4.0
        st["amplitude"] = 0.1 * math.log(4.0) + 1.0
    return st


# ------------------------------------------------------------------ the pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    import blackflash_b200 as bf
    case = st["case"]
    op = case["op"]
    if op == "window_fwd":
        return bf.window_attention(st["q"], st["k"], st["v"], case["window"], case["sinks"])
    if op == "window_train":
        o = bf.window_attention_with_grad(st["q"], st["k"], st["v"], case["window"], case["sinks"])
        return (o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]))
    if op == "window_decode":
        return bf.window_decode(st["q"], st["k"], st["v"], st["lengths"], case["window"], case["sinks"])
    if op == "prefix_decode":
        return bf.prefix_decode(st["q"], st["kp"], st["vp"], st["k"], st["v"], st["lengths"])
    args = (st["positions"], st["freqs"], case["interleaved"], st["amplitude"])
    if op == "rotary":
        return bf.rotary(st["q"], st["k"], *args)
    q, k = bf.rotary_with_grad(st["q"], st["k"], *args)
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"])))


def _plain_softmax(s):
    """Softmax over the last axis, its masked scores -inf; a row that sees nothing gets zeros."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p))


def _window_blocks(case):
    """Blocks of queries with the keys that some query of the block sees (as index ranges)."""
    nq, nkv, window, sinks = case["nq"], case["nkv"], case["window"], case["sinks"]
    step = 1024
    for a in range(0, nq, step):
        e = min(nq, a + step)
        lo = max(0, a + nkv - nq - window + 1)
        yield a, e, min(sinks, lo), lo, e + nkv - nq


def _window_scores(case, q, k, a, e, s0, lo, hi, dev):
    """Masked scores of queries [a, e) of one KV head's group against keys [0, s0) and [lo, hi)."""
    keys = torch.cat([torch.arange(s0, device=dev), torch.arange(lo, hi, device=dev)])
    pos = torch.arange(a, e, device=dev) + case["nkv"] - case["nq"]
    seen = (keys <= pos[:, None]) & ((keys > pos[:, None] - case["window"]) | (keys < case["sinks"]))
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(case["d"])
    return torch.where(seen, s, torch.full_like(s, -math.inf))


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "window_fwd":
        return _plain_window(case, st["q"], st["k"], st["v"], None)[0]
    if op == "window_train":
        return _plain_window(case, st["q"].detach(), st["k"].detach(), st["v"].detach(), st["do"])
    if op == "window_decode":
        return _plain_decode(case, st["q"], st["k"], st["v"], st["lengths"], None, None, case["window"], case["sinks"])
    if op == "prefix_decode":
        return _plain_decode(case, st["q"], st["k"], st["v"], st["lengths"], st["kp"], st["vp"], None, 0)
    turn = (st["positions"], st["freqs"], case["interleaved"], st["amplitude"])
    out = tuple(_plain_rotary(st[x].detach(), *turn, 1.0) for x in ("q", "k"))
    if op == "rotary_train":
        out += tuple(_plain_rotary(st[x], *turn, -1.0) for x in ("dq", "dk"))
    return out


def _plain_window(case, q, k, v, do):
    b, hq, nq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    q, k, v = q.float().view(b, hkv, g, nq, d), k.float(), v.float()
    o = torch.empty_like(q)
    if do is not None:
        do = do.float().view(b, hkv, g, nq, d)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        for a, e, s0, lo, hi in _window_blocks(case):
            kk = torch.cat([k[i, :, :s0], k[i, :, lo:hi]], 1)[:, None]
            vv = torch.cat([v[i, :, :s0], v[i, :, lo:hi]], 1)[:, None]
            qq = q[i, :, :, a:e]
            p = _plain_softmax(_window_scores(case, qq, kk, a, e, s0, lo, hi, q.device))
            oo = torch.matmul(p, vv)
            o[i, :, :, a:e] = oo
            if do is not None:
                dd = do[i, :, :, a:e]
                gv = torch.matmul(p.transpose(-1, -2), dd).sum(1)
                ds = p * (torch.matmul(dd, vv.transpose(-1, -2)) - (dd * oo).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, :, :, a:e] = torch.matmul(ds, kk)
                gk = torch.matmul(ds.transpose(-1, -2), qq).sum(1)
                dk[i, :, :s0] += gk[:, :s0]
                dk[i, :, lo:hi] += gk[:, s0:]
                dv[i, :, :s0] += gv[:, :s0]
                dv[i, :, lo:hi] += gv[:, s0:]
    ty = _TYPES[case["type"]]
    outs = (o.view(b, hq, nq, d),) if do is None else (o.view(b, hq, nq, d), dq.view(b, hq, nq, d), dk, dv)
    return tuple(x.to(ty) for x in outs)


def _plain_decode(case, q, k, v, lengths, kp, vp, window, sinks):
    b, hq, t, d = q.shape
    hkv, cap = k.shape[1], k.shape[2]
    q = q.float().view(b, hkv, hq // hkv * t, d)
    keys = torch.arange(cap, device=q.device)
    pos = (lengths[:, None] - t + torch.arange(t, device=q.device))[:, None, :, None]
    seen = keys <= pos
    if window is not None:
        seen = seen & ((keys > pos - window) | (keys < sinks))
    seen = seen.expand(b, hq // hkv, t, cap).reshape(b, 1, hq // hkv * t, cap)
    s = torch.matmul(q, k.float().transpose(-1, -2)) / math.sqrt(d)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    if kp is None:
        o = torch.matmul(_plain_softmax(s), v.float())
    else:
        n = kp.shape[1]
        p = _plain_softmax(torch.cat([torch.matmul(q, kp.float().transpose(-1, -2)) / math.sqrt(d), s], -1))
        o = torch.matmul(p[..., :n], vp.float()) + torch.matmul(p[..., n:], v.float())
    return o.view(b, hq, t, d).to(_TYPES[case["type"]])


def _plain_rotary(x, positions, freqs, interleaved, amplitude, sign):
    """Pairs turned by position times frequency: angles in fp64, products in fp32."""
    angle = positions.double()[..., None] * freqs
    cos = (torch.cos(angle) * amplitude).float()[:, None]
    sin = (torch.sin(angle) * (amplitude * sign)).float()[:, None]
    r = 2 * freqs.numel()
    y = x.float().contiguous()
    if interleaved:
        u, w = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([u * cos - w * sin, u * sin + w * cos], -1).flatten(-2)
    else:
        u, w = y[..., : r // 2], y[..., r // 2: r]
        turned = torch.cat([u * cos - w * sin, u * sin + w * cos], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


# ------------------------------------------------------------------ the definition in fp64

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("window_fwd", "window_train"):
        return _exact_window(case, st)
    if op in ("window_decode", "prefix_decode"):
        return _exact_decode(case, st)
    return _exact_rotary(case, st)


def _exact_window(case, st):
    """Head by head over the full score matrix."""
    nq, nkv = case["nq"], case["nkv"]
    group = case["hq"] // case["hkv"]
    scale = case["d"] ** -0.5
    q, k, v = (st[x].detach() for x in ("q", "k", "v"))
    i = torch.arange(nq, device=_DEV)[:, None] + (nkv - nq)
    j = torch.arange(nkv, device=_DEV)[None, :]
    hidden = (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
    grads = case["op"] == "window_train"
    o = torch.empty(q.shape, dtype=torch.float64, device=_DEV)
    if grads:
        dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device=_DEV) for x in (q, k, v))
    for b in range(case["b"]):
        for h in range(case["hq"]):
            c = h // group
            qh, kh, vh = q[b, h].double(), k[b, c].double(), v[b, c].double()
            p = torch.softmax((qh @ kh.T).mul_(scale).masked_fill_(hidden, -math.inf), -1)
            o[b, h] = p @ vh
            if grads:
                g = st["do"][b, h].double()
                dv[b, c] += p.T @ g
                ds = (g @ vh.T).sub_((g * o[b, h]).sum(1, keepdim=True)).mul_(p).mul_(scale)
                dq[b, h] = ds @ kh
                dk[b, c] += ds.T @ qh
    return (o, dq, dk, dv) if grads else o


def _exact_decode(case, st):
    """Sequence by sequence, token by token, over the keys that the token sees."""
    b, hq, hkv, t, d = (case[x] for x in ("b", "hq", "hkv", "t", "d"))
    if b * t * hkv > 4096:
        return None
    o = torch.zeros((b, hq, t, d), dtype=torch.float64, device=_DEV)
    lengths = st["lengths"].tolist()
    shared = case["op"] == "prefix_decode"
    if shared:
        kp, vp = st["kp"].double(), st["vp"].double()
    for s in range(b):
        for x in range(t):
            pos = lengths[s] - t + x
            near = range(max(0, pos + 1 - (case.get("window") or pos + 1)), pos + 1)
            idx = list(range(min(case.get("sinks", 0), max(0, near.start)))) + list(near)
            ks, vs = st["k"][s][:, idx].double(), st["v"][s][:, idx].double()
            if shared:
                ks, vs = torch.cat([kp, ks], 1), torch.cat([vp, vs], 1)
            if ks.shape[1] == 0:
                continue
            qs = st["q"][s, :, x].double().view(hkv, hq // hkv, d)
            w = torch.einsum("hgd,hnd->hgn", qs, ks) * d ** -0.5
            o[s, :, x] = torch.einsum("hgn,hnd->hgd", torch.softmax(w, -1), vs).reshape(hq, d)
    return o


def _exact_rotary(case, st):
    """Each pair as a complex number times amplitude e^(i angle)."""
    r = case["rot"]
    unit = torch.polar(torch.full_like(st["freqs"], st["amplitude"]).expand(*st["positions"].shape, r // 2).contiguous(),
                       st["positions"].double()[..., None] * st["freqs"])[:, None]

    def turn(x, factor):
        y = x.detach().double().contiguous()
        if case["interleaved"]:
            at = (slice(0, r, 2), slice(1, r, 2))
        else:
            at = (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(y[..., at[0]], y[..., at[1]]) * factor
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
        return y

    out = (turn(st["q"], unit), turn(st["k"], unit))
    if case["op"] == "rotary_train":
        out += (turn(st["dq"], unit.conj()), turn(st["dk"], unit.conj()))
    return out
