"""Reference of the paged-cache operators in 64 bits, one sequence at a time, and the inputs of their tests."""
import math

import torch

import vulkanforge_amd as vf

DEV = "cuda:0"
CACHE_TYPE = {vf.KvDtype.F32: torch.float32, vf.KvDtype.F16: torch.float16, vf.KvDtype.F8: torch.float8_e4m3fn}


class Pool:
    """A cache over torch buffers, with page tables for sequences of the given lengths in shuffled pages.

    Slots that hold no row of a sequence are NaN; table entries behind a sequence's last page are -1."""

    def __init__(self, dtype, hkv, d, page, kv, layers=1, layer=0, seed=0, spare=3, extra_entries=1):
        self.dtype, self.hkv, self.d, self.page, self.layer = dtype, hkv, d, page, layer
        self.kv = list(kv)
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in kv]
        n_pages = sum(used) + spare
        ids = torch.randperm(n_pages, generator=g)
        self.table = torch.full((len(kv), max(used + [1]) + extra_entries), -1, dtype=torch.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = ids[at:at + u]
            at += u
        shape = (layers, n_pages, hkv, page, d)
        ct = CACHE_TYPE[dtype]
        self.k = torch.full(shape, float("nan"), dtype=torch.float32)
        self.v = torch.full(shape, float("nan"), dtype=torch.float32)
        for i, n in enumerate(kv):
            j = torch.arange(n)
            p, sl = self.table[i].long()[j // page], j % page
            self.k[:, p, :, sl] = torch.randn((n, layers, hkv, d), generator=g)
            self.v[:, p, :, sl] = torch.randn((n, layers, hkv, d), generator=g)
        self.k, self.v = self.k.to(ct).to(DEV), self.v.to(ct).to(DEV)
        self.cache = vf.PagedKvCache(vf.PagedKvConfig(layers, hkv, d, page, n_pages, dtype), k_buffer=self.k.data_ptr(),
                                     v_buffer=self.v.data_ptr())
        self.table_dev = self.table.to(DEV)
        self.kv_dev = torch.tensor(self.kv, dtype=torch.int32, device=DEV)

    def rows(self, x, s, n=None):
        """Rows of sequence s in positions 0..n-1 as [n, hkv, d] in 64 bits (NaN where the table has no page)."""
        n = self.kv[s] if n is None else n
        j = torch.arange(n)
        p = self.table[s].long()[j // self.page]
        y = x[self.layer].float().cpu().double()
        out = y[p.clamp(0, y.shape[0] - 1), :, j % self.page]
        out[(p < 0) | (p >= y.shape[0])] = float("nan")
        return out

    def batch(self, q_len=None, n_tokens=None, max_kv_len=0):
        off = None
        if q_len is not None:
            off = torch.tensor([0] + list(torch.tensor(q_len).cumsum(0)), dtype=torch.int32, device=DEV)
            n_tokens = sum(q_len) if n_tokens is None else n_tokens
        return vf.SeqBatch(self.table_dev, self.kv_dev, off, n_tokens=n_tokens, max_kv_len=max_kv_len)


def seen(n_keys, pos, window, sink):
    """[len(pos), n_keys]: which keys the queries at these positions see."""
    j = torch.arange(n_keys)[None]
    p = torch.as_tensor(pos)[:, None]
    ok = j <= p
    if window:
        ok = ok & ((j > p - window) | (j < sink))
    return ok


def attention(pool, q, q_len, window=0, sink=0, softcap=0.0, scale=None):
    """(outputs, tolerance of f32 arithmetic) for rows q [n, hq, d] of chunks q_len, positions from the pool's lengths."""
    q = q.float().cpu().double()
    n, hq, d = q.shape
    g = hq // pool.hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out, at, worst = torch.zeros(n, hq, d, dtype=torch.float64), 0, 0.0
    for s, m in enumerate(q_len):
        kv = pool.kv[s]
        k, v = pool.rows(pool.k, s), pool.rows(pool.v, s)
        ok = seen(kv, range(kv - m, kv), window, sink)
        held = ~torch.isnan(k[:, 0, 0]) if kv else torch.zeros(0, dtype=torch.bool)
        ok = ok & held[None]
        k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
        for h in range(hq):
            x = q[at:at + m, h] @ k[:, h // g].t() * scale
            big = float((q[at:at + m, h].abs() @ k[:, h // g].abs().t()).max()) * scale if kv and m else 0.0
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            x = x.masked_fill(~ok, -math.inf)
            w = torch.softmax(x, -1).nan_to_num(0.0) if kv else x
            out[at:at + m, h] = w @ v[:, h // g]
            top = float(v.abs().max()) if kv else 0.0
            # A score is a sum of d products: off by at most (d / 4 + 8) half steps of sum|q k| (chains of at most d / 4
            # products and a few joins, operands held to 22 bits = 4 half steps each); tanh and exp are a few
            # steps more.  A weight is off by twice the score's error relative (numerator and denominator); sums over
            # the keys run in chains of at most kv / 16 + 64 steps; weights are held to 22 bits at least.
            u = 2.0 ** -24
            ds = big * (d / 4 + 8) * u + 8 * u
            worst = max(worst, top * (2 * ds + (kv / 16 + 64 + 8) * u))
        at += m
    return out, worst


def f16_tolerance(pool):
    """What f16 queries and outputs add: the output's rounding and, in the prefill kernel, the weights' (half a step each)."""
    top = float(pool.v.float().nan_to_num(0.0).abs().max())
    return top * 2 * 2.0 ** -11


def axis_of(p, sections, interleaved):
    if len(sections) == 1:
        return 0
    if interleaved:
        a = p % len(sections)
        return a if p // len(sections) < sections[a] else 0
    a = 0
    while p >= sum(sections[:a + 1]):
        a += 1
    return a


def turned(x, weight, pos, base, rot, sections, interleaved, mode, eps=1e-6, ff=None, freq_scale=1.0, attn=1.0):
    """Norm and rotation of rows x [n, heads, d] with positions pos [axes][n], in 64 bits."""
    x = x.float().cpu().double().clone()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.cpu().double()
    for p in range(rot // 2):
        t = torch.as_tensor(pos[axis_of(p, sections, interleaved)]).double() * base ** (-2.0 * p / rot) * freq_scale
        if ff is not None:
            t = t / float(ff[p])
        c, s = (torch.cos(t) * attn)[:, None], (torch.sin(t) * attn)[:, None]
        i0, i1 = (p, p + rot // 2) if mode == vf.ROPE_NEOX else (2 * p, 2 * p + 1)
        a, b = x[..., i0].clone(), x[..., i1].clone()
        x[..., i0], x[..., i1] = a * c - b * s, a * s + b * c
    return x
