"""What the paged-cache operators are measured on: the cases, their inputs, a plain form of each operator and its
definition in 64 bits.

Four operators work on one cache of pages, K and V as [layer][page][kv_head][slot][d] each:

  pages    copies and forks of pages (all layers, K and V)
  write    RMS norm, rotation with positions of several axes, append into the sequences' pages
  decode   attention of one new token per sequence over its pages
  prefill  causal attention of a ragged batch of chunks over their pages

Both attention forms take a sliding window with first tokens that stay visible.  ``own`` says whether ``run`` calls the
framework (True) or computes the plain form (False).
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "fp8": 1}
KIND = {"f32": 0, "f16": 1, "fp8": 2}
BASE = 1.0e6         # rotation base
EPS = 1e-6           # of the RMS norm


# ---- cases --------------------------------------------------------------------------------------
def listed():
    return [
        # a sampled request splits into four continuations: they share the full pages, each gets its own last page
        dict(name="fork_4_fp8", op="pages", kind="fork", cache="fp8", layers=32, hkv=8, d=128, page=16, pool=128, kv=1000, n=4),
        # live pages move to the front of the pool of a whole model
        dict(name="move_200_pages_f16", op="pages", kind="copy", cache="f16", layers=32, hkv=8, d=128, page=64, pool=400, n=200),
        # one token of each of 32 running requests, text positions (all axes alike are still three arrays)
        dict(name="write_decode_32", op="write", cache="fp8", io="f32", hq=32, hkv=8, d=128, rot=128, mode="neox", axes=3,
             inter=False, norm=True, seqs=32, q_min=1, q_max=1, kv_min=1, kv_max=2048, page=16, mix=1),
        # image tokens of several requests, written in one launch
        dict(name="write_image_6000", op="write", cache="f16", io="f16", hq=32, hkv=8, d=128, rot=128, mode="neox", axes=3,
             inter=True, norm=True, seqs=5, q_min=300, q_max=1700, kv_min=1700, kv_max=4096, page=64, mix=2),
        # the start of one conversation: latency
        dict(name="decode_1x200_fp8", op="decode", cache="fp8", io="f32", hq=32, hkv=8, d=128, seqs=1, kv_min=200, kv_max=200,
             page=16, window=0, sink=0, softcap=0.0, mix=3),
        # an ordinary batch of requests of very different lengths
        dict(name="decode_48_ragged_fp8", op="decode", cache="fp8", io="f16", hq=32, hkv=8, d=128, seqs=48, kv_min=17,
             kv_max=8193, page=64, window=0, sink=0, softcap=0.0, mix=4),
        # Gemma-style sliding layers with four first tokens kept, soft-capped
        dict(name="decode_12_window_f16", op="decode", cache="f16", io="f32", hq=16, hkv=8, d=256, seqs=12, kv_min=1000,
             kv_max=16384, page=32, window=4096, sink=4, softcap=50.0, mix=5),
        # one long context alone on the card: the split over the length carries it
        dict(name="decode_1x65536_fp8", op="decode", cache="fp8", io="f32", hq=32, hkv=8, d=128, seqs=1, kv_min=65536,
             kv_max=65536, page=16, window=0, sink=0, softcap=0.0, mix=6),
        # a handful of drafted tokens behind a short context
        dict(name="prefill_7x300_f16", op="prefill", cache="f16", io="f32", hq=14, hkv=2, d=64, seqs=1, q_min=7, q_max=7,
             kv_min=300, kv_max=300, page=16, window=0, sink=0, softcap=0.0, mix=7),
        # the framework's own prefill chunk, over pages, with the f32 activations its other calls take
        dict(name="prefill_512x4608_fp8", op="prefill", cache="fp8", io="f32", hq=32, hkv=8, d=128, seqs=1, q_min=512, q_max=512,
             kv_min=4608, kv_max=4608, page=64, window=0, sink=0, softcap=0.0, mix=8),
        # chunks of several requests with a window per query and first tokens kept
        dict(name="prefill_6_window_f16", op="prefill", cache="f16", io="f16", hq=32, hkv=8, d=128, seqs=6, q_min=1, q_max=1500,
             kv_min=1500, kv_max=8192, page=32, window=1024, sink=4, softcap=0.0, mix=9),
        # a long prompt from its first token
        dict(name="prefill_8192_fp8", op="prefill", cache="fp8", io="f16", hq=32, hkv=8, d=128, seqs=1, q_min=8192, q_max=8192,
             kv_min=8192, kv_max=8192, page=64, window=0, sink=0, softcap=0.0, mix=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: every type, head layout, page size and length of the ranges above."""
    while True:
        op = rng.choice(["pages", "write", "decode", "decode", "prefill", "prefill"])
        hkv = rng.choice([1, 2, 4, 8])
        c = dict(op=op, cache=rng.choice(["f32", "f16", "fp8"]), hkv=hkv, d=rng.choice([64, 80, 96, 128, 128, 192, 256]),
                 page=rng.choice([16, 32, 64, 128, 256]))
        if op == "pages":
            n = _log(rng, 1, 200)
            c.update(kind=rng.choice(["fork", "copy"]), layers=rng.randint(1, 40), n=n)
            if c["kind"] == "fork":
                c.update(n=min(n, 32), kv=_log(rng, 1, 5000))
                c["pool"] = -(-c["kv"] // c["page"]) + 2 * c["n"]
            else:
                c["pool"] = 2 * n + rng.randint(0, 40)
            if work(c)["bytes"] > work(listed()[1])["bytes"]:
                continue
            return c
        c.update(io=rng.choice(["f32", "f16"]), hq=hkv * rng.choice([1, 2, 3, 4, 7, 8, 12]), mix=rng.randrange(1 << 20))
        if op == "write":
            c.update(rot=rng.choice([c["d"], c["d"] // 2]), mode=rng.choice(["neox", "norm"]), axes=rng.choice([1, 2, 3]),
                     inter=rng.random() < 0.5, norm=rng.random() < 0.5, seqs=_log(rng, 1, 64))
            c["q_max"] = _log(rng, 1, 2048)
            c["q_min"] = rng.randint(1, c["q_max"])
            c["kv_min"] = c["q_max"]
            c["kv_max"] = c["kv_min"] + _log(rng, 1, 4096)
            if c["seqs"] * c["q_max"] > 8192 or work(c)["bytes"] > 4e8:
                continue
            return c
        c.update(window=rng.choice([0, 0, _log(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 50.0]))
        c["sink"] = rng.randint(0, 64) if c["window"] else 0
        if op == "decode":
            c.update(seqs=_log(rng, 1, 128), kv_max=_log(rng, 1, 65536))
            c["kv_min"] = rng.randint(1, c["kv_max"])
            if c["seqs"] * c["kv_max"] * hkv * c["d"] > 3e8 or work(c)["flops"] > 4e10:
                continue
            return c
        c.update(seqs=_log(rng, 1, 16), q_max=_log(rng, 1, 4096))
        c["q_min"] = rng.randint(1, c["q_max"])
        c["kv_min"] = c["q_max"]
        c["kv_max"] = c["kv_min"] + _log(rng, 1, 8192)
        if c["seqs"] * c["q_max"] * c["kv_max"] * c["hq"] > 2.2e9 or work(c)["flops"] > 5e11:
            continue
        return c


def _lengths(case):
    """(chunk lengths, lengths with the chunk) of the sequences: a fixed function of the case."""
    r = random.Random(case["mix"])
    kv = [r.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    q = [r.randint(case.get("q_min", 1), case.get("q_max", 1)) for _ in range(case["seqs"])]
    return q, kv


def _visible(case, pos):
    """Number of keys the query at position ``pos`` sees."""
    n = pos + 1
    if case["window"] and n > case["window"]:
        return case["window"] + min(case["sink"], n - case["window"])
    return n


def work(case):
    es = SIZE[case["cache"]]
    if case["op"] == "pages":
        rows = case["n"] * (case["kv"] % case["page"] if case["kind"] == "fork" else case["page"])
        return {"bytes": max(1, 4 * case["layers"] * case["hkv"] * rows * case["d"] * es), "flops": 0}
    q, kv = _lengths(case)
    io, hq, hkv, d = SIZE[case["io"]], case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        n = sum(q)
        return {"bytes": n * d * (2 * hq * io + 2 * hkv * (io + es)) + 4 * n * case["axes"], "flops": 8 * n * d * (hq + hkv)}
    rows = pairs = 0
    for m, n in zip(q, kv):
        vis = [_visible(case, p) for p in range(n - m, n)] if case["window"] else None
        pairs += sum(vis) if vis else sum(range(n - m + 1, n + 1))
        first = _visible(case, n - m)                       # keys of the chunk's first query, and one more for each later one
        rows += min(n, first + m - 1)
    return {"bytes": 2 * rows * hkv * d * es + 2 * sum(q) * hq * d * io, "flops": 4 * pairs * hq * d}


# ---- inputs -------------------------------------------------------------------------------------
def _values(gen, shape, dtype, std=1.0):
    """Seeded normal values; the 8-bit cache holds saturated E4M3 values."""
    n = math.prod(shape)
    x = torch.empty(n, dtype=torch.float16 if dtype is torch.float8_e4m3fn else dtype, device=DEV)
    x.normal_(0.0, std, generator=gen)
    return x.to(dtype).view(shape)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    s = {"case": case}
    dt, page, hkv, d = DTYPES[case["cache"]], case["page"], case["hkv"], case["d"]
    layers = case.get("layers", 1)
    if case["op"] == "pages":
        n_pages = case["pool"]
        if case["kind"] == "fork":
            used = -(-case["kv"] // page)                    # the request's pages: the lowest ids of a fresh pool
            s["pages"] = list(range(used))
            part = case["kv"] % page
            s["fresh"] = list(range(used, used + case["n"])) if part else []
            s["src"], s["dst"] = [used - 1] * len(s["fresh"]), s["fresh"]
            s["rows"] = part or page
        else:
            ids = host.sample(range(n_pages), 2 * case["n"])
            s["src"], s["dst"], s["rows"] = ids[:case["n"]], ids[case["n"]:], page
        s["src_t"], s["dst_t"] = (torch.tensor(x, dtype=torch.int64, device=DEV) for x in (s["src"], s["dst"]))
    else:
        q, kv = _lengths(case)
        used = [-(-n // page) for n in kv]
        n_pages = sum(used) + 3
        ids = host.sample(range(n_pages), sum(used))
        table = torch.full((len(kv), max(used)), -1, dtype=torch.int32)
        at = 0
        for i, u in enumerate(used):
            table[i, :u] = torch.tensor(ids[at:at + u], dtype=torch.int32)
            at += u
        s["table"], s["kv"] = table.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV)
        off = [0]
        for m in q:
            off.append(off[-1] + m)
        s["off"] = torch.tensor(off, dtype=torch.int32, device=DEV)
        s["n"], s["max_q"], s["max_kv"] = off[-1], max(q), max(kv)
        io, hq = DTYPES[case["io"]], case["hq"]
        s["q"] = _values(gen, (s["n"], hq, d), io)
    shape = (layers, n_pages, hkv, page, d)
    s["k"], s["v"] = _values(gen, shape, dt, 0.7), _values(gen, shape, dt, 0.7)
    if case["op"] == "write":
        s["k_new"], s["v_new"] = (_values(gen, (s["n"], hkv, d), io) for _ in range(2))
        half = case["rot"] // 2
        a = case["axes"]
        s["sections"] = [half - (a - 1) * (half // a)] + [half // a] * (a - 1)
        text = torch.randint(0, 200000, (1, s["n"]), generator=gen, device=DEV, dtype=torch.int32)
        grid = torch.randint(0, 512, (a, s["n"]), generator=gen, device=DEV, dtype=torch.int32)
        s["pos"] = (text + grid).contiguous()
        s["wq"], s["wk"] = ((1.0 + 0.1 * torch.randn(d, generator=gen, device=DEV)) if case["norm"] else None for _ in range(2))
        s["q_out"] = torch.zeros_like(s["q"])
    elif case["op"] != "pages":
        s["o"] = torch.zeros_like(s["q"])
    if own:
        import vulkanforge_amd as vf
        cfg = vf.PagedKvConfig(layers, hkv, d, page, n_pages, vf.KvDtype(KIND[case["cache"]]))
        s["cache"] = vf.PagedKvCache(cfg, k_buffer=s["k"].data_ptr(), v_buffer=s["v"].data_ptr())
        if case["op"] == "pages":
            if case["kind"] == "fork":
                assert s["cache"].alloc(len(s["pages"])) == s["pages"]
        else:
            one = case["op"] == "decode"
            s["batch"] = vf.SeqBatch(s["table"], s["kv"], None if one else s["off"], n_tokens=s["n"], max_kv_len=s["max_kv"])
            s["fwd"] = vf.PagedForward(s["cache"], case["hq"])
            if case["op"] == "write":
                s["rope"] = vf.MRope(rotary_dim=case["rot"], freq_base=BASE, sections=s["sections"], interleaved=case["inter"],
                                     rope_mode=vf.ROPE_NEOX if case["mode"] == "neox" else vf.ROPE_NORM, eps=EPS)
    return s


# ---- one pass -----------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"pages": _plain_pages, "write": _plain_write, "decode": _plain_attention, "prefill": _plain_attention}[s["case"]["op"]](s)


def _run_own(s):
    c = s["case"]
    if c["op"] == "pages":
        if c["kind"] == "fork":
            tables = s["cache"].fork(s["pages"], c["kv"], c["n"])
            for t in tables:
                s["cache"].release(t)
            return {"k": s["k"], "v": s["v"], "tables": torch.tensor(tables)}
        s["cache"].copy_pages(s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if c["op"] == "write":
        s["fwd"].qk_rope_kv_write(0, s["batch"], s["q"], s["k_new"], s["v_new"], s["rope"], q_out=s["q_out"],
                                  q_norm_weight=s["wq"], k_norm_weight=s["wk"], positions=s["pos"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    call = s["fwd"].decode_attention if c["op"] == "decode" else s["fwd"].prefill_attention
    call(0, s["batch"], s["q"], s["o"], window=c["window"], n_sink=c["sink"], softcap=c["softcap"])
    return s["o"]


def _bytes(x):
    """8-bit floats as bytes: what indexing works on."""
    return x.view(torch.uint8) if x.dtype is torch.float8_e4m3fn else x


def _plain_pages(s):
    rows = s["rows"]
    for x in (_bytes(s["k"]), _bytes(s["v"])):
        x[:, s["dst_t"], :, :rows] = x[:, s["src_t"], :, :rows]
    if s["case"]["kind"] == "copy":
        return {"k": s["k"], "v": s["v"]}
    n, full = s["case"]["n"], s["case"]["kv"] // s["case"]["page"]
    tables = torch.tensor(s["pages"]).repeat(n, 1)
    if s["fresh"]:
        tables[:, full] = torch.tensor(s["fresh"])
    return {"k": s["k"], "v": s["v"], "tables": tables}


def _axis_of_pair(case, sections, half):
    """Axis whose position turns pair p."""
    p = torch.arange(half, device=DEV)
    if case["inter"]:
        a = p % case["axes"]
        cap = torch.tensor(sections, device=DEV)[a]
        return torch.where(p // case["axes"] < cap, a, 0)
    edges = torch.tensor(sections, device=DEV).cumsum(0)
    return (p[:, None] >= edges[None, :]).sum(1)


def _store(x, dtype):
    return x.clamp(-448.0, 448.0).to(dtype) if dtype is torch.float8_e4m3fn else x.to(dtype)


def _plain_write(s):
    c = s["case"]
    d, rot, half = c["d"], c["rot"], c["rot"] // 2
    freq = torch.pow(torch.tensor(BASE, dtype=torch.float64, device=DEV), -2.0 * torch.arange(half, device=DEV).double() / rot)
    angle = s["pos"].double()[_axis_of_pair(c, s["sections"], half)].t() * freq      # [n, half]; far positions need 64 bits
    cs, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if c["mode"] == "neox":
            a, b = x[..., :half], x[..., half:rot]
            return torch.cat([a * cs - b * sn, a * sn + b * cs, x[..., rot:]], -1)
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat([torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2), x[..., rot:]], -1)

    q = turn(s["q"], s["wq"]).to(s["q"].dtype)
    k, v = _store(turn(s["k_new"], s["wk"]), s["k"].dtype), _store(s["v_new"].float(), s["v"].dtype)
    t = torch.arange(s["n"], device=DEV)
    seq = torch.searchsorted(s["off"][1:].long(), t, right=True)
    pos = s["kv"].long()[seq] - s["off"].long()[seq + 1] + t
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    _bytes(s["k"])[0, page, :, slot] = _bytes(k)
    _bytes(s["v"])[0, page, :, slot] = _bytes(v)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_attention(s):
    """Pages gathered into padded rows, scores of all padded (query, key) pairs, masked softmax, in 32 bits."""
    c = s["case"]
    b, hkv, d, page = c["seqs"], c["hkv"], c["d"], c["page"]
    g = c["hq"] // hkv
    n_keys = s["table"].shape[1] * page
    table = s["table"].long().clamp(min=0)
    k, v = (x[0][table] for x in (_bytes(s["k"]), _bytes(s["v"])))                  # [b, pages, hkv, page, d]
    k, v = (x.view(s["k"].dtype).float().permute(0, 2, 1, 3, 4).reshape(b, hkv, n_keys, d) for x in (k, v))
    off, kv = s["off"].long(), s["kv"].long()
    i = torch.arange(s["max_q"], device=DEV)
    row = off[:-1, None] + i                                                         # [b, max_q]
    real = row < off[1:, None]
    q = s["q"].float()[row.clamp(max=s["n"] - 1)].reshape(b, s["max_q"], hkv, g, d).permute(0, 2, 1, 3, 4)
    q = q.reshape(b, hkv, s["max_q"] * g, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.view(b, hkv, s["max_q"], g, n_keys)
    p = (kv - off[1:] + off[:-1])[:, None] + i                                       # position of each query
    j = torch.arange(n_keys, device=DEV)
    seen = j <= p[..., None]
    if c["window"]:
        seen &= (j > p[..., None] - c["window"]) | (j < c["sink"])
    x.masked_fill_(~seen[:, None, :, None], float("-inf"))
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hkv, s["max_q"] * g, n_keys), v).view(b, hkv, s["max_q"], g, d) / total
    return o.permute(0, 2, 1, 3, 4).reshape(b, s["max_q"], hkv * g, d)[real].to(s["q"].dtype)


# ---- the definition in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "pages":
        if sum(x.numel() for x in (s["k"], s["v"])) > 1e9:
            return None                                                              # a copy: nothing is computed
        out = [x.to(torch.float32) for x in (s["k"], s["v"])]
        for src, dst in zip(s["src"], s["dst"]):
            for x in out:
                x[:, dst, :, :s["rows"]] = x[:, src, :, :s["rows"]]
        res = {"k": out[0], "v": out[1]}
        return res if case["kind"] == "copy" else {**res, "tables": None}
    off, kv = s["off"].tolist(), s["kv"].tolist()
    rows = []                                                                        # flat cache row of every key, per sequence
    for i, n in enumerate(kv):
        j = torch.arange(n, device=DEV)
        rows.append(s["table"][i].long()[j // case["page"]] * case["page"] + j % case["page"])
    flat = lambda x: x[0].to(torch.float32).double().transpose(1, 2).reshape(-1, case["hkv"], case["d"])  # noqa: E731
    if case["op"] == "write":
        return _exact_write(case, s, off, kv, rows, flat)
    k, v = flat(s["k"]), flat(s["v"])
    g, out = case["hq"] // case["hkv"], []
    for i, n in enumerate(kv):
        m = off[i + 1] - off[i]
        q = s["q"][off[i]:off[i + 1]].double()
        ki, vi = k[rows[i]], v[rows[i]]
        o = torch.empty_like(q)
        for at in range(0, m, 512):
            pos = torch.arange(n - m + at, min(n, n - m + at + 512), device=DEV)
            j = torch.arange(n, device=DEV)
            hidden = j[None] > pos[:, None]
            if case["window"]:
                hidden |= (j[None] <= pos[:, None] - case["window"]) & (j[None] >= case["sink"])
            for h in range(case["hkv"]):
                w = q[at:at + 512, h * g:(h + 1) * g].transpose(0, 1) @ ki[:, h].t() / math.sqrt(case["d"])
                if case["softcap"]:
                    w = torch.tanh(w / case["softcap"]) * case["softcap"]
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                o[at:at + 512, h * g:(h + 1) * g] = (w @ vi[:, h]).transpose(0, 1)
        out.append(o)
    return torch.cat(out)


def _exact_write(case, s, off, kv, rows, flat):
    d, rot = case["d"], case["rot"]
    half = rot // 2
    axis = []
    for p in range(half):
        if case["inter"]:
            a = p % case["axes"]
            axis.append(a if p // case["axes"] < s["sections"][a] else 0)
        else:
            a = 0
            while p >= sum(s["sections"][:a + 1]):
                a += 1
            axis.append(a)
    z = torch.zeros(s["n"], half, dtype=torch.complex128, device=DEV)
    for p in range(half):
        t = s["pos"][axis[p]].double() * BASE ** (-2.0 * p / rot)
        z[:, p] = torch.complex(torch.cos(t), torch.sin(t))

    def turned(x, w):
        x = x.double().clone()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * w.double()
        i0, i1 = (slice(0, half), slice(half, rot)) if case["mode"] == "neox" else (slice(0, rot, 2), slice(1, rot, 2))
        y = torch.complex(x[..., i0], x[..., i1]) * z[:, None]
        x[..., i0], x[..., i1] = y.real, y.imag
        return x

    k, v = flat(s["k"]).clone(), flat(s["v"]).clone()
    kn, vn = turned(s["k_new"], s["wk"]), s["v_new"].double()
    for i, n in enumerate(kv):
        m = off[i + 1] - off[i]
        k[rows[i][n - m:]], v[rows[i][n - m:]] = kn[off[i]:off[i + 1]], vn[off[i]:off[i + 1]]
    shape = (1, s["k"].shape[1], case["page"], case["hkv"], d)
    return {"q": turned(s["q"], s["wq"]), "k": k.view(shape).transpose(2, 3).contiguous(), "v": v.view(shape).transpose(2, 3).contiguous()}
