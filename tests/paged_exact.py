"""Attention over pages in 64 bits on the device, with a bound per element: for batches too large for tests/paged_ref.py and for
errors that a bound over a whole batch would hide."""
import math

import torch

from paged_ref import DEV, seen

U = 2.0 ** -24


def out_step(ref, io):
    """Rounding of an output to its type: half a step, or half of the smallest one."""
    return ref.abs() * 2.0 ** -11 + 2.0 ** -25 if io is torch.float16 else ref.abs() * U + 2.0 ** -149


def exact(pool, q, q_len, window=0, sink=0, softcap=0.0, scale=None, lens=None, score_error=True):
    """(outputs, bound of the f32 arithmetic per element) of rows q [n, hq, d], chunks q_len, on the device in 64 bits.

    ``lens`` (default: the pool's) are the lengths the call is given: positions count from them, keys end with the table.
    The bound: a weight is off by twice its score's error relative (numerator and denominator); a score is a sum of d products in
    chains of at most d / 4 and a few joins, operands held to 22 bits (4 half steps), tanh and exp a few steps more;
    sums over the keys run in chains of at most kv / 16 + 64 steps, weights are held to 22 bits at least, 8 for the joins and the
    division: all of it times sum_j w_j |v_j| of the element.  ``score_error=False``: scores that the kernel forms without an error."""
    n, hq, d = q.shape
    g = hq // pool.hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, bound = (torch.zeros(n, hq, d, dtype=torch.float64, device=DEV) for _ in range(2))
    limit = pool.table.shape[1] * pool.page
    at = 0
    for s, m in enumerate(q_len):
        length = pool.kv[s] if lens is None else lens[s]
        kv = min(length, limit)
        if m and kv > 0:
            j = torch.arange(kv)
            p = pool.table[s].long()[j // pool.page]
            there = (p >= 0) & (p < pool.k.shape[1])
            k, v = (x[pool.layer].double()[p.clamp(0, x.shape[1] - 1).to(DEV), :, (j % pool.page).to(DEV)] for x in (pool.k, pool.v))
            ok = (seen(kv, range(length - m, length), window, sink) & there[None]).to(DEV).repeat_interleave(g, 0)     # [m g, kv]
            any_seen = ok.any(0)[:, None, None]
            k, v = (torch.where(any_seen, x, 0.0) for x in (k, v))
            for h in range(pool.hkv):
                qs = q[at:at + m, h * g:(h + 1) * g].double().reshape(m * g, d)
                x = qs @ k[:, h].t().contiguous() * scale
                big = (qs.abs() @ k[:, h].abs().t().contiguous() * scale).masked_fill(~ok, 0.0).amax(1) if score_error else torch.zeros(m * g, device=DEV)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                w = torch.softmax(x.masked_fill(~ok, -math.inf), -1).nan_to_num(0.0)
                rel = 2 * (big * (d / 4 + 8) * U + 8 * U) + (kv / 16 + 64 + 8) * U
                out[at:at + m, h * g:(h + 1) * g] = (w @ v[:, h]).view(m, g, d)
                bound[at:at + m, h * g:(h + 1) * g] = (w @ v[:, h].abs() * rel[:, None]).view(m, g, d)
        at += m
    return out, bound


def assert_near(o, ref, bound, io, what=""):
    err, tol = (o.double() - ref).abs(), bound + out_step(ref, io)
    worst = (err / tol.clamp(min=1e-300)).nan_to_num(math.inf).max().item() if o.numel() else 0.0
    print(f"{what} worst error {err.max().item() if o.numel() else 0.0:.3g}, {worst:.3g} of its bound", flush=True)
    assert worst <= 1.0, (what, worst)
