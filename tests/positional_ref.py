"""fp64 statements of the position-aware operators, and elementwise error bounds.

Every bound counts roundings: a value rounded to type t is off by at most eps(t) / 2 of
itself, where eps(bf16) = 2^-7 and eps(fp16) = 2^-10."""
import math

import torch


def half_step(t):
    return torch.finfo(t).eps / 2


def visible(n_q, n_kv, window, sinks, device):
    p = torch.arange(n_q, device=device)[:, None] + n_kv - n_q
    j = torch.arange(n_kv, device=device)[None, :]
    return (j <= p) & ((j > p - window) | (j < sinks))


def softmax64(s, seen):
    """Rows of probabilities (zero where nothing is seen) and their logsumexp."""
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - lse[..., None]), torch.zeros_like(s))
    return torch.nan_to_num(p, nan=0.0), lse


def attention64(q, k, v, seen, scale):
    """O, lse, P and the bound's P @ |V|, for q [..., n_q, d] and k, v [..., n_kv, d]."""
    p, lse = softmax64(torch.matmul(q, k.transpose(-1, -2)) * scale, seen)
    return torch.matmul(p, v), lse, p, torch.matmul(p, v.abs())


# What the exponentials add, relative to each weight: the FMA-pipe exponential is off by at
# most 7.5e-5 (its minimax error); scores of a few tens in fp32 and ex2.approx (2^-22) add
# less than 2.5e-5. Weights and their sum are both off by that, hence twice.
EXP_REL = 2e-4


def o_bound(o, pv, t):
    """Weights rounded to t (half a step of P|V|), output rounded to t, exponentials."""
    return half_step(t) * (pv + o.abs()) + EXP_REL * pv + 1e-7


def check_o(got, o, pv):
    err = (got.double() - o).abs()
    bound = o_bound(o, pv, got.dtype)
    bad = err > bound
    assert not bad.any() and torch.isfinite(got).all(), (
        f"{int(bad.sum())} of {bad.numel()} outside, worst {float((err / bound).max()):.3g} of the bound")


def check_lse(got, lse):
    """The sum's relative error is EXP_REL at most, so its logarithm's absolute one is too;
    the fp32 value and log2 add 2^-22 of a value below 100."""
    inf = lse == -math.inf
    assert torch.equal(got == -math.inf, inf)
    err = (got.double() - lse).masked_fill(inf, 0).abs()
    assert float(err.max()) <= EXP_REL + 100 * 2.0 ** -22, float(err.max())


def window_ref(q, k, v, window, sinks, scale):
    """q [B, Hq, Nq, d], k, v [B, Hkv, Nkv, d] -> O, lse, bound term, all fp64."""
    g = q.shape[1] // k.shape[1]
    k, v = (x.double().repeat_interleave(g, 1) for x in (k, v))
    seen = visible(q.shape[2], k.shape[2], window, sinks, q.device)
    o, lse, _, pv = attention64(q.double(), k, v, seen, scale)
    return o, lse, pv


def window_grad_ref(q, k, v, do, window, sinks, scale):
    """Gradients in fp64 and the elementwise bound of each.

    With h half a bf16 step and e = EXP_REL: P enters dV rounded (h) and off by e; dS is
    P (dP - D), off by e of itself, by P times D's error, and rounded (h). D comes from the
    rounded O, itself within o_bound, so its error is sum |dO| o_bound. Each gradient is
    rounded once more (h)."""
    b, hq, nq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    h = half_step(torch.bfloat16)
    q6, do6 = q.double(), do.double()
    k6, v6 = (x.double().repeat_interleave(g, 1) for x in (k, v))
    seen = visible(nq, k.shape[2], window, sinks, q.device)
    o, _, p, pv = attention64(q6, k6, v6, seen, scale)
    dv = p.transpose(-1, -2) @ do6
    dp = do6 @ v6.transpose(-1, -2)
    ds = p * (dp - (do6 * o).sum(-1, keepdim=True)) * scale
    d_err = (do6.abs() * o_bound(o, pv, torch.bfloat16)).sum(-1, keepdim=True)
    # dP itself is an fp32 sum of d exact products: d steps of the sum of their sizes.
    dp_err = d * 2.0 ** -24 * (do6.abs() @ v6.abs().transpose(-1, -2))
    e_ds = (h + EXP_REL) * (ds.abs() + p * scale * (d_err + dp_err)) + p * scale * (d_err + dp_err)
    grads = {"dq": ds @ k6, "dk": ds.transpose(-1, -2) @ q6, "dv": dv}
    errs = {"dq": e_ds @ k6.abs(), "dk": e_ds.transpose(-1, -2) @ q6.abs(),
            "dv": (h + EXP_REL) * (p.transpose(-1, -2) @ do6.abs())}
    for x in ("dk", "dv"):
        grads[x] = grads[x].view(b, hkv, g, *grads[x].shape[2:]).sum(2)
        errs[x] = errs[x].view(b, hkv, g, *errs[x].shape[2:]).sum(2)
    # 1e-5 of the terms' size for fp32 sums over some thousand of them.
    return {x: (grads[x], errs[x] * (1 + 1e-5) + h * grads[x].abs() + 1e-6) for x in grads}


def decode_ref(q, k, v, lengths, window, sinks, scale, kp=None, vp=None):
    """Sequence by sequence; kp, vp [Hkv, P, d] are seen by every token."""
    b, hq, t, d = q.shape
    g, cap = hq // k.shape[1], k.shape[2]
    outs = []
    for i in range(b):
        n = min(max(int(lengths[i]), 0), cap)
        ks, vs = k[i, :, :n].double(), v[i, :, :n].double()
        pos = torch.arange(t, device=q.device)[:, None] + n - t
        j = torch.arange(n, device=q.device)[None, :]
        seen = (j <= pos) & ((j > pos - window) | (j < sinks))
        if kp is not None:
            ks, vs = torch.cat([kp.double(), ks], 1), torch.cat([vp.double(), vs], 1)
            seen = torch.cat([torch.ones(t, kp.shape[1], dtype=torch.bool, device=q.device), seen], 1)
        ks, vs = ks.repeat_interleave(g, 0), vs.repeat_interleave(g, 0)
        outs.append(attention64(q[i].double(), ks, vs, seen, scale))
    return tuple(torch.stack([o[x] for o in outs]) for x in (0, 1, 3))


def rotary64(x, positions, freqs, interleaved, amplitude=1.0, sign=1.0):
    r = 2 * freqs.numel()
    a = positions.double()[..., None] * freqs
    c, s = (torch.cos(a) * amplitude)[..., None, :, :], (torch.sin(a) * amplitude * sign)[..., None, :, :]
    y = x.double().clone()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, w = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = u * c - w * s, u * s + w * c
    return y
