"""Paged cache on the GPU against 64-bit references: page copies, norm + rotation + append, decode and prefill attention
over ragged batches, and a run of them together."""
import math

import pytest
import torch

import vulkanforge_amd as vf
from paged_ref import CACHE_TYPE, DEV, Pool, attention, f16_tolerance, seen, turned

pytestmark = pytest.mark.gpu

F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8


def rand_q(n, hq, d, io=torch.float32, seed=1, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((n, hq, d), generator=g) * scale).to(io).to(DEV)


def check_attention(pool, hq, q_len, io=torch.float32, window=0, sink=0, softcap=0.0, decode=False, seed=1, qscale=1.0, max_kv_len=0):
    fwd = vf.PagedForward(pool.cache, hq)
    n = sum(q_len)
    q = rand_q(n, hq, pool.d, io, seed, qscale)
    o = torch.full_like(q, float("nan"))
    batch = pool.batch(None if decode else q_len, max_kv_len=max_kv_len)
    call = fwd.decode_attention if decode else fwd.prefill_attention
    call(pool.layer, batch, q, o, window=window, n_sink=sink, softcap=softcap)
    torch.cuda.synchronize()
    ref, tol = attention(pool, q, q_len, window, sink, softcap)
    if io is torch.float16:
        tol += f16_tolerance(pool)
    err = (o.float().cpu().double() - ref).abs().max().item() if n else 0.0
    print(f"max error {err:.3g}, tolerance {tol:.3g}", flush=True)
    assert err <= tol, (err, tol)                       # (a NaN fails this too)
    return q, o


# ---- page copies ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, hkv, d, page", [(F8, 8, 128, 16), (F16, 2, 64, 64), (F32, 3, 80, 32), (F8, 1, 3, 16),
                                                 (F16, 5, 33, 128), (F8, 2, 256, 256)])
@pytest.mark.parametrize("rows", [None, "ragged"])
def test_copy_moves_exactly_the_given_rows(dtype, hkv, d, page, rows):
    layers, n = 3, 12
    g = torch.Generator().manual_seed(d)
    es = dtype.element_size()
    k, v = (torch.randint(0, 256, (layers, n, hkv, page, d * es), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    c = vf.PagedKvCache(vf.PagedKvConfig(layers, hkv, d, page, n, dtype), k_buffer=k.data_ptr(), v_buffer=v.data_ptr())
    src, dst = [0, 3, 3, 11], [5, 1, 2, 7]
    cnt = None if rows is None else [1, page, 0, page - 3]
    want = [x.clone() for x in (k, v)]
    for i, (s, t) in enumerate(zip(src, dst)):
        r = page if cnt is None else cnt[i]
        for x in want:
            x[:, t, :, :r] = x[:, s, :, :r]
    c.copy_pages(src, dst, cnt)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_of_more_pairs_than_one_launch_holds():
    n = 700
    k, v = (torch.randint(0, 256, (2, 2 * n, 1, 16, 64), dtype=torch.uint8, device=DEV) for _ in range(2))
    c = vf.PagedKvCache(vf.PagedKvConfig(2, 1, 64, 16, 2 * n, F8), k_buffer=k.data_ptr(), v_buffer=v.data_ptr())
    perm = torch.randperm(2 * n, generator=torch.Generator().manual_seed(3)).tolist()
    src, dst = perm[:n], perm[n:]
    want = k.clone()
    want[:, dst] = want[:, src]
    c.copy_pages(src, dst)
    torch.cuda.synchronize()
    assert torch.equal(k, want)


def test_copy_beyond_4_gib():
    # the last page of a buffer of 5 GiB: offsets that do not fit 32 bits
    n = 5 * 1024 * 4
    k = torch.zeros((1, n, 8, 256, 128), dtype=torch.uint8, device=DEV)
    c = vf.PagedKvCache(vf.PagedKvConfig(1, 8, 128, 256, n, F8), k_buffer=k.data_ptr(), v_buffer=k.data_ptr())
    k[0, n - 2] = 7
    c.copy_pages([n - 2], [n - 1])
    c.copy_pages([n - 1], [0])
    torch.cuda.synchronize()
    assert bool((k[0, n - 1] == 7).all()) and bool((k[0, 0] == 7).all()) and int(k[0, 1].max()) == 0


def test_compact_then_attention_gives_the_same_rows():
    pool = Pool(F16, 2, 64, 16, [100, 37, 64], layers=2, layer=1, spare=9)
    live = sorted(int(p) for p in pool.table.flatten() if p >= 0)
    c = pool.cache
    c.alloc(c.config.n_pages)
    c.release([p for p in range(c.config.n_pages) if p not in live])
    q, o = check_attention(pool, 4, [5, 1, 7])
    ids = c.compact()
    pool.table = torch.tensor([[ids[int(p)] if p >= 0 else -1 for p in row] for row in pool.table], dtype=torch.int32)
    assert sorted(int(p) for p in pool.table.flatten() if p >= 0) == list(range(len(live)))
    pool.table_dev.copy_(pool.table)
    q2, o2 = check_attention(pool, 4, [5, 1, 7])
    assert torch.equal(o, o2)


# ---- norm + rotation + append --------------------------------------------------------------------------
def write_case(dtype, io, hq, hkv, d, page, q_len, kv, rot, mode, sections, inter, norm=True, positions="far", ff=False, base=1e6,
               strided=False, in_place=False, n_pad=0):
    pool = Pool(dtype, hkv, d, page, kv, layers=2, layer=1, seed=d + len(kv))
    n = sum(q_len)
    g = torch.Generator().manual_seed(5)
    tot = (hq + 2 * hkv)
    if strided:
        packed = torch.randn((n + n_pad, tot, d), generator=g).to(io).to(DEV)
        q, k, v = packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]
    else:
        q, k, v = (torch.randn((n + n_pad, h, d), generator=g).to(io).to(DEV) for h in (hq, hkv, hkv))
    q0, k0, v0 = (x.clone() for x in (q, k, v))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(DEV) if norm else None for _ in range(2))
    fft = (1 + torch.rand(rot // 2, generator=g)).to(DEV) if ff else None
    own = torch.cat([torch.arange(b - m, b) for m, b in zip(q_len, kv)]) if n else torch.zeros(0)
    if positions == "far":
        pos = torch.randint(0, 2_000_000, (len(sections), n + n_pad), generator=g, dtype=torch.int32)
        posd = pos.to(DEV)
        pos = pos[:, :n]
    else:
        pos, posd = own[None].repeat(len(sections), 1), None
    out = q if in_place else torch.full_like(q0, 9.0)
    fwd = vf.PagedForward(pool.cache, hq)
    rope = vf.MRope(rot, base, sections, inter, mode)
    before_k, before_v = pool.k.clone(), pool.v.clone()
    batch = pool.batch(q_len, n_tokens=n + n_pad)
    fwd.qk_rope_kv_write(1, batch, q, k, v, rope, q_out=None if in_place else out, q_norm_weight=wq, k_norm_weight=wk,
                         positions=posd, freq_factors=fft)
    torch.cuda.synchronize()
    ct = CACHE_TYPE[dtype]
    u = 2.0 ** -24
    half_io = 2.0 ** -11 if io is torch.float16 else u
    # f32 arithmetic per element: the norm (sum of d squares in chains of d / 64 + 6, a root, two products: at most
    # d / 64 + 16 half steps), two products and a sum (4), cos and sin (4, and 2^-24 of a turn's fraction: 7 half steps)
    rel = (d / 64 + 16 + 4 + 11) * u

    def near(x, ref, half, what):
        size = ref.abs().amax(-1, keepdim=True) * math.sqrt(2)     # a turned pair is at most sqrt 2 times its larger element
        err = (x.float().cpu().double() - ref).abs()
        assert bool((err <= size * rel + ref.abs() * half + 2.0 ** -25).all()), (what, err.max())

    rq = turned(q0[:n], wq, pos, base, rot, sections, inter, mode, ff=fft)
    rk = turned(k0[:n], wk, pos, base, rot, sections, inter, mode, ff=fft)
    near(out[:n], rq, half_io, "q")
    if n_pad:
        assert torch.equal(out[n:], (q0 if in_place else torch.full_like(q0, 9.0))[n:])
    if not in_place and not strided:
        assert torch.equal(q, q0)
    at = 0
    lowest = 2.0 ** -10 if dtype == F8 else 2.0 ** -25           # half of the smallest step
    half = {F8: 2.0 ** -4, F16: 2.0 ** -11, F32: u}[dtype]
    written = torch.zeros(pool.k.shape[1], page, dtype=torch.bool)
    for s, (m, b) in enumerate(zip(q_len, kv)):
        for i in range(m):
            j = b - m + i
            page_id, slot = int(pool.table[s, j // page]), j % page
            written[page_id, slot] = True
            ref = rk[at + i].clamp(-448, 448) if dtype == F8 else rk[at + i]
            err = (pool.k[1, page_id, :, slot].float().cpu().double() - ref).abs()
            size = ref.abs().amax(-1, keepdim=True) * math.sqrt(2)
            assert bool((err <= size * rel + ref.abs() * half + lowest).all()), (s, i, err.max())
            vv = v0[at + i].float()
            vv = (vv.clamp(-448, 448) if dtype == F8 else vv).to(ct)
            assert torch.equal(pool.v[1, page_id, :, slot].view(torch.uint8), vv.view(torch.uint8))
        at += m
    # nothing else has changed: bytes of unwritten slots and of the other layer
    for x, y in ((pool.k, before_k), (pool.v, before_v)):
        a, b = (t.cpu().view(torch.uint8).reshape(*t.shape[:4], -1).transpose(2, 3) for t in (x, y))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1][~written], b[1][~written])


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("mode", [vf.ROPE_NEOX, vf.ROPE_NORM])
def test_write_three_axes(dtype, io, mode):
    write_case(dtype, io, 8, 2, 128, 16, [3, 1, 20], [30, 1, 47], 128, mode, [16, 24, 24], False)


@pytest.mark.parametrize("sections, inter", [([64], False), ([64], True), ([24, 20, 20], True), ([32, 32], False), ([32, 32], True),
                                             ([16, 16, 16, 16], True), ([0, 64], False), ([64, 0, 0], False), ([10, 50, 4], True)])
def test_write_sections(sections, inter):
    write_case(F16, torch.float32, 4, 2, 128, 32, [9, 4], [33, 64], 128, vf.ROPE_NEOX, sections, inter)


@pytest.mark.parametrize("d, rot", [(128, 64), (80, 80), (80, 32), (64, 2), (256, 256), (512, 128), (33, 32), (100, 50), (6, 6), (96, 0),
                                    (20, 12)])
@pytest.mark.parametrize("mode", [vf.ROPE_NEOX, vf.ROPE_NORM])
def test_write_widths(d, rot, mode):
    write_case(F16, torch.float32, 3, 1, d, 16, [5, 2], [5, 19], rot, mode, [rot // 2], False)
    write_case(F8, torch.float16, 3, 3, d, 16, [1], [17], rot, mode, [rot // 2], False, norm=False)


@pytest.mark.parametrize("kw", [dict(norm=False), dict(positions=None), dict(ff=True), dict(strided=True), dict(in_place=True),
                                dict(strided=True, in_place=True), dict(n_pad=5), dict(n_pad=3, in_place=True), dict(base=10000.0)])
def test_write_options(kw):
    write_case(F8, torch.float32, 4, 2, 64, 16, [6, 0, 1, 11], [10, 3, 40, 11], 64, vf.ROPE_NEOX, [12, 10, 10], True, **kw)
    write_case(F16, torch.float16, 5, 1, 96, 64, [70, 3], [200, 65], 96, vf.ROPE_NORM, [16, 16, 16], False, **kw)


def test_write_bounds_what_the_device_arrays_say():
    """Lengths beyond the table, negative lengths, pages that do not exist, tokens in front of the first position: rows are
    dropped, nothing else is touched."""
    d, page = 64, 16
    pool = Pool(F16, 2, d, page, [16, 16, 16, 16, 16], spare=2, extra_entries=0)
    pool.table_dev[0, 0] = 10_000
    pool.table_dev[1, 0] = -5
    pool.kv_dev.copy_(torch.tensor([16, 16, 900, -7, 2], dtype=torch.int32))   # 900: clamped to the table's 16
    fwd = vf.PagedForward(pool.cache, 2)
    n = 5 * 3
    off = torch.arange(0, n + 1, 3, dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(pool.table_dev, pool.kv_dev, off, n_tokens=n)
    k, v = (torch.full((n, 2, d), float(i + 1), device=DEV) for i in range(2))
    before = pool.k.clone()
    fwd.qk_rope_kv_write(0, batch, None, k, v, vf.MRope(0))
    torch.cuda.synchronize()
    want = before.clone()
    want[0, int(pool.table[2, 0]), :, 13:16] = 1.0
    want[0, int(pool.table[4, 0]), :, 0:2] = 1.0              # three tokens, two positions: the first has no row
    assert torch.equal(pool.k.view(torch.uint8), want.view(torch.uint8))
    # offsets that run backwards or leave the rows
    bad = torch.tensor([-3, 9, 4, 99, 15, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    pool.kv_dev.fill_(16)
    pool.table_dev.copy_(pool.table)
    fwd.qk_rope_kv_write(0, vf.SeqBatch(pool.table_dev, pool.kv_dev, bad, n_tokens=n), None, k, v, vf.MRope(0))
    o = torch.zeros((n, 2, d), device=DEV)
    fwd.prefill_attention(0, vf.SeqBatch(pool.table_dev, pool.kv_dev, bad, n_tokens=n), torch.ones_like(o), o)
    torch.cuda.synchronize()


# ---- attention -----------------------------------------------------------------------------------------
DTYPES = pytest.mark.parametrize("dtype", [F32, F16, F8])
IOS = pytest.mark.parametrize("io", [torch.float32, torch.float16])
CALL = pytest.mark.parametrize("decode", [True, False])


@DTYPES
@IOS
@CALL
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_ragged_batch(dtype, io, d, decode):
    kv = [1, 2, 15, 16, 17, 33, 64, 65, 200, 511]
    pool = Pool(dtype, 2, d, 16, kv, layers=2, layer=1)
    check_attention(pool, 8, [1] * 10 if decode else [1, 2, 3, 16, 1, 33, 20, 64, 100, 130], io, decode=decode)


@DTYPES
@CALL
@pytest.mark.parametrize("d", [16, 48, 80, 96, 112, 160, 192, 208, 240, 72, 33, 272, 512, 8])
def test_attention_widths(dtype, d, decode):
    pool = Pool(dtype, 2, d, 32, [70, 3, 129])
    check_attention(pool, 4, [1] * 3 if decode else [40, 3, 5], decode=decode)
    check_attention(pool, 4, [1] * 3 if decode else [40, 3, 5], torch.float16, decode=decode, window=20, sink=3)


@CALL
@pytest.mark.parametrize("hq, hkv", [(1, 1), (2, 1), (3, 1), (5, 1), (7, 1), (8, 1), (9, 1), (12, 1), (16, 1), (17, 1), (40, 1), (14, 2), (32, 8),
                                     (6, 3), (24, 24)])
def test_attention_head_groups(hq, hkv, decode):
    pool = Pool(F16, hkv, 64, 64, [150, 31])
    check_attention(pool, hq, [1, 1] if decode else [37, 31], decode=decode)
    pool = Pool(F8, hkv, 128, 16, [70, 200, 1])
    check_attention(pool, hq, [1, 1, 1] if decode else [3, 40, 1], torch.float16, decode=decode)


@DTYPES
@CALL
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_page_sizes(dtype, page, decode):
    pool = Pool(dtype, 2, 128, page, [page - 1, page, page + 1, 3 * page + 7, 1])
    check_attention(pool, 8, [1] * 5 if decode else [2, page, page // 2, 9, 1], decode=decode)


@DTYPES
@CALL
@pytest.mark.parametrize("window, sink", [(1, 0), (1, 1), (16, 4), (31, 0), (33, 33), (64, 100), (100, 7), (1000, 4), (500, 300), (7, 16)])
def test_attention_window_and_first_tokens(dtype, window, sink, decode):
    pool = Pool(dtype, 2, 128, 16, [1, 40, 131, 777, 300])
    check_attention(pool, 8, [1] * 5 if decode else [1, 40, 60, 200, 17], window=window, sink=sink, decode=decode)


@CALL
@IOS
def test_attention_softcap_and_large_scores(io, decode):
    pool = Pool(F16, 2, 128, 32, [300, 90])
    check_attention(pool, 4, [1, 1] if decode else [50, 90], io, softcap=50.0, decode=decode)
    check_attention(pool, 4, [1, 1] if decode else [50, 90], softcap=2.0, decode=decode, window=64, sink=8)
    check_attention(pool, 4, [1, 1] if decode else [50, 90], decode=decode, qscale=12.0)


@CALL
@pytest.mark.parametrize("dtype, hq, hkv, d, kv", [(F8, 32, 8, 128, [5000]), (F16, 4, 1, 64, [3333, 1]), (F32, 8, 2, 128, [2500, 9]),
                                                   (F16, 16, 8, 256, [2100]), (F8, 12, 1, 96, [4097, 64, 1000])])
def test_attention_long_sequences_are_split_and_joined(dtype, hq, hkv, d, kv, decode):
    pool = Pool(dtype, hkv, d, 64, kv)
    n = [1] * len(kv) if decode else [min(20, x) for x in kv]
    check_attention(pool, hq, n, decode=decode)
    check_attention(pool, hq, n, torch.float16, decode=decode, window=1500, sink=5)


def test_decode_many_sequences():
    kv = [(37 * i * i) % 191 for i in range(300)]            # zeros among them
    pool = Pool(F16, 2, 64, 16, kv)
    check_attention(pool, 4, [1] * 300, decode=True)
    check_attention(pool, 4, [1] * 300, decode=True, window=50, sink=2)


@CALL
def test_a_bound_on_the_lengths_changes_the_rounding_only(decode):
    pool = Pool(F8, 2, 128, 16, [700, 3])
    for bound in (0, 1, 64, 700, 100000):
        check_attention(pool, 8, [1, 1] if decode else [11, 2], decode=decode, max_kv_len=bound)


@CALL
@DTYPES
def test_rows_without_keys_are_zero_and_padding_rows_stay(dtype, decode):
    pool = Pool(dtype, 2, 64, 16, [0, 20, 0, 5, 0])
    fwd = vf.PagedForward(pool.cache, 4)
    if decode:
        q = rand_q(5, 4, 64)
        o = torch.full_like(q, 3.0)
        fwd.decode_attention(0, pool.batch(), q, o)
        torch.cuda.synchronize()
        assert bool((o[[0, 2, 4]] == 0).all()) and bool(o[[1, 3]].isfinite().all()) and bool((o[[1, 3]] != 3.0).any())
        return
    q_len, pad = [2, 4, 0, 9, 1], 6                           # chunks longer than their sequences: tokens in front of position 0
    n = sum(q_len)
    q = rand_q(n + pad, 4, 64)
    o = torch.full_like(q, 3.0)
    fwd.prefill_attention(0, pool.batch(q_len, n_tokens=n + pad), q, o)
    torch.cuda.synchronize()
    assert bool((o[n:] == 3.0).all())
    assert bool((o[0:2] == 0).all()) and bool((o[6:10] == 0).all()) and bool((o[15] == 0).all())
    real, _ = attention(Pool(dtype, 2, 64, 16, [0, 20, 0, 5, 0]), torch.cat([q[2:6], q[10:15]]), [0, 4, 0, 5, 0])
    assert (o[[2, 3, 4, 5, 10, 11, 12, 13, 14]].cpu().double() - real).abs().max() < 1e-4


@CALL
@DTYPES
@pytest.mark.parametrize("d", [128, 40])
def test_missing_pages_hide_their_keys(dtype, d, decode):
    pool = Pool(dtype, 1, d, 16, [100, 60, 40])
    pool.table[0, 2] = -1
    pool.table[0, 5] = 10 ** 6
    pool.table[1, :2] = -1                                    # pages that left the window
    pool.table[2, :] = -1                                     # nothing left: zeros
    pool.table_dev.copy_(pool.table)
    check_attention(pool, 4, [1, 1, 1] if decode else [20, 5, 3], decode=decode)
    check_attention(pool, 4, [1, 1, 1] if decode else [20, 5, 3], decode=decode, window=20, sink=3)


@CALL
@DTYPES
def test_infinities_and_nan_in_masked_places_do_not_reach_the_output(dtype, decode):
    # behind the last key, between the first tokens and the window, in unused pages (Pool leaves NaN in unused slots)
    pool = Pool(dtype, 2, 128, 32, [90, 33])
    kv, window, sink = pool.kv, 20, 3
    bad = float("inf") if dtype != F8 else float("nan")
    for s, n in enumerate(kv):
        lo = n - window if decode else n - window - 1          # chunk of two: the first query sees one key more
        for j in range(sink, lo):
            p, sl = int(pool.table[s, j // 32]), j % 32
            for x in (pool.k, pool.v):
                row = torch.full((pool.hkv, pool.d), bad).to(x.dtype).to(DEV)
                x[0, p, :, sl] = row
    q_len = [1, 1] if decode else [2, 2]
    fwd = vf.PagedForward(pool.cache, 4)
    q = rand_q(sum(q_len), 4, 128)
    o = torch.full_like(q, float("nan"))
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else q_len), q, o, window=window, n_sink=sink)
    torch.cuda.synchronize()
    clean = [x.float().cpu().nan_to_num(0.0, 0.0, 0.0) for x in (pool.k, pool.v)]
    pool.k, pool.v = clean
    ref, tol = attention(pool, q, q_len, window, sink)
    assert (o.cpu().double() - ref).abs().max() <= tol


@CALL
def test_nan_in_a_visible_place_does_reach_the_output(decode):
    pool = Pool(F16, 1, 64, 16, [50])
    p, sl = int(pool.table[0, 1]), 3
    pool.k[0, p, 0, sl, 5] = float("nan")
    fwd = vf.PagedForward(pool.cache, 2)
    q = rand_q(1, 2, 64)
    o = torch.zeros_like(q)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else [1]), q, o)
    torch.cuda.synchronize()
    assert bool(o.isnan().all())


@CALL
@IOS
def test_strided_rows(io, decode):
    pool = Pool(F8, 2, 64, 16, [40, 100, 7])
    q_len = [1, 1, 1] if decode else [10, 1, 7]
    n = sum(q_len)
    packed = rand_q(n, 4 + 4, 64, io)
    q = packed[:, :4]
    big = torch.full((n, 9, 64), 5.0, dtype=io, device=DEV)
    o = big[:, 3:7]
    fwd = vf.PagedForward(pool.cache, 4)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else q_len), q, o)
    torch.cuda.synchronize()
    ref, tol = attention(pool, q, q_len)
    tol += f16_tolerance(pool) if io is torch.float16 else 0.0
    assert (o.float().cpu().double() - ref).abs().max() <= tol
    assert bool((big[:, :3] == 5.0).all()) and bool((big[:, 7:] == 5.0).all())


@CALL
def test_rows_at_odd_addresses(decode):
    # q and o not 16-byte aligned: still served
    pool = Pool(F16, 2, 64, 16, [40, 9])
    q_len = [1, 1] if decode else [3, 9]
    n = sum(q_len)
    raw = rand_q(1, 1, n * 4 * 64 + 8).flatten()
    q = raw[1:1 + n * 256].view(n, 4, 64)
    buf = torch.zeros(n * 256 + 8, device=DEV)
    o = buf[3:3 + n * 256].view(n, 4, 64)
    fwd = vf.PagedForward(pool.cache, 4)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else q_len), q, o)
    torch.cuda.synchronize()
    ref, tol = attention(pool, q, q_len)
    assert (o.cpu().double() - ref).abs().max() <= tol
    assert float(buf[:3].abs().max()) == 0 and float(buf[3 + n * 256:].abs().max()) == 0


@CALL
def test_cache_beyond_4_gib(decode):
    # pages at both ends of a 6 GiB buffer per tensor
    n, page = 6 * 4096, 256
    k = torch.zeros((1, n, 8, page, 128), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.zeros((1, n, 8, page, 128), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    table = torch.tensor([[n - 1, 0, n // 2 + 1, n - 3]], dtype=torch.int32)
    small = Pool(F8, 8, 128, page, [1000], spare=0, extra_entries=0)
    for i in range(4):
        for x, y in ((k, small.k), (v, small.v)):
            x.view(torch.uint8)[0, int(table[0, i])] = y.view(torch.uint8)[0, int(small.table[0, i])]
    c = vf.PagedKvCache(vf.PagedKvConfig(1, 8, 128, page, n, F8), k_buffer=k.data_ptr(), v_buffer=v.data_ptr())
    fwd = vf.PagedForward(c, 16)
    q_len = [1] if decode else [30]
    off = None if decode else torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(table.to(DEV), small.kv_dev, off, n_tokens=q_len[0])
    q = rand_q(q_len[0], 16, 128)
    o = torch.empty_like(q)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, batch, q, o)
    torch.cuda.synchronize()
    ref, tol = attention(small, q, q_len)
    assert (o.cpu().double() - ref).abs().max() <= tol


def test_results_repeat_bit_for_bit():
    pool = Pool(F8, 4, 128, 16, [3000, 17, 900, 1, 0, 450])
    fwd = vf.PagedForward(pool.cache, 16)
    for q_len in (None, [200, 17, 3, 1, 0, 77]):
        n = 6 if q_len is None else sum(q_len)
        q = rand_q(n, 16, 128)
        outs = []
        for _ in range(3):
            o = torch.full_like(q, float("nan"))
            (fwd.decode_attention if q_len is None else fwd.prefill_attention)(0, pool.batch(q_len), q, o)
            outs.append(o)
        torch.cuda.synchronize()
        assert torch.equal(outs[0].nan_to_num(7), outs[1].nan_to_num(7)) and torch.equal(outs[0].nan_to_num(7), outs[2].nan_to_num(7))


def test_refusals_of_wrong_tensors():
    pool = Pool(F16, 2, 64, 16, [20, 9])
    fwd = vf.PagedForward(pool.cache, 4)
    b = pool.batch()
    q = rand_q(2, 4, 64)
    o = torch.empty_like(q)
    for bad in (q[:1], q[:, :3], q.double(), q.to(torch.bfloat16), q.cpu(), q.transpose(0, 1).contiguous().transpose(0, 1), q[..., ::2],
                q[:1].expand(2, 4, 64)):
        with pytest.raises((ValueError, vf.VfkvError)):
            fwd.decode_attention(0, b, bad, o)
    with pytest.raises(ValueError):
        fwd.decode_attention(0, b, q, o.half())
    with pytest.raises(ValueError):
        fwd.decode_attention(0, b, q, o, window=-1)
    with pytest.raises(vf.VfkvError):
        fwd.decode_attention(0, b, q, q)
    with pytest.raises(vf.VfkvError):
        fwd.decode_attention(0, pool.batch([1, 1]), q, o)
    with pytest.raises(vf.VfkvError):
        vf.PagedForward(pool.cache, 8, workspace=fwd.workspace).decode_attention(0, b, rand_q(2, 8, 64), rand_q(2, 8, 64))
    for kw in (dict(kv_lens=pool.kv_dev.long()), dict(kv_lens=pool.kv_dev.cpu()), dict(page_table=pool.table_dev[:1]),
               dict(q_offsets=pool.kv_dev), dict(q_offsets=torch.zeros(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            vf.SeqBatch(**{**dict(page_table=pool.table_dev, kv_lens=pool.kv_dev), **kw})


# ---- together --------------------------------------------------------------------------------------------
def serve(steps, capture, io=torch.float32):
    """Two requests prefill, the second forks in two, all three decode `steps` tokens with pages taken as they fill; the
    decode step is captured once and replayed when `capture`.  Returns the outputs of every step and the pool."""
    layers, hq, hkv, d, page = 2, 8, 2, 128, 16
    c = vf.PagedKvCache(vf.PagedKvConfig(layers, hkv, d, page, 40, F8))
    fwd = vf.PagedForward(c, hq)
    rope = vf.MRope(d, 1e6, [16, 24, 24])
    g = torch.Generator().manual_seed(11)
    lens = [45, 37]
    lists = [c.alloc(c.pages_for(n)) for n in lens]
    entries = 8

    def table(ls):
        return torch.tensor([x + [-1] * (entries - len(x)) for x in ls], dtype=torch.int32).to(DEV)

    n = sum(lens)
    qkv = torch.randn((layers, n, hq + 2 * hkv, d), generator=g).to(io).to(DEV)
    off = torch.tensor([0, lens[0], n], dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(table(lists), torch.tensor(lens, dtype=torch.int32, device=DEV), off, n_tokens=n)
    o = torch.zeros((layers, n, hq, d), dtype=io, device=DEV)
    for l in range(layers):
        x = qkv[l]
        q = torch.empty((n, hq, d), dtype=io, device=DEV)
        fwd.qk_rope_kv_write(l, batch, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], rope, q_out=q)
        fwd.prefill_attention(l, batch, q, o[l], window=24, n_sink=4)
    outs = [o.clone()]
    forks = c.fork(lists[1], lens[1], 2).tolist()
    c.release(lists[1])
    lists, lens = [lists[0]] + forks, [lens[0], lens[1], lens[1]]
    tab, kv = table(lists), torch.tensor(lens, dtype=torch.int32, device=DEV)
    step_batch = vf.SeqBatch(tab, kv, max_kv_len=entries * page)
    x = torch.zeros((layers, 3, hq + 2 * hkv, d), dtype=io, device=DEV)
    q = torch.empty((3, hq, d), dtype=io, device=DEV)
    o = torch.zeros((layers, 3, hq, d), dtype=io, device=DEV)

    def step():
        for l in range(layers):
            fwd.qk_rope_kv_write(l, step_batch, x[l, :, :hq], x[l, :, hq:hq + hkv], x[l, :, hq + hkv:], rope, q_out=q)
            fwd.decode_attention(l, step_batch, q, o[l], window=24, n_sink=4)

    graph = None
    for i in range(steps):
        for s in range(3):
            if lens[s] % page == 0:
                lists[s] = lists[s] + c.alloc(1)
            lens[s] += 1
        tab.copy_(table(lists))
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        x.copy_(torch.randn(x.shape, generator=g).to(io))
        if not capture:
            step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        outs.append(o.clone())
        (x * 2).sum().item()                              # eager work between the steps
    torch.cuda.synchronize()
    for s in range(3):
        c.release(lists[s])
    assert c.free_count == 40
    return outs


@IOS
def test_serving_loop_captured_and_eager_agree(io):
    eager = serve(20, False, io)
    replayed = serve(20, True, io)
    assert all(torch.equal(a, b) for a, b in zip(eager, replayed)) and all(bool(a.isfinite().all()) for a in eager)


def test_paged_and_contiguous_caches_agree():
    """The same tokens through the contiguous cache's calls and the paged ones: cache bytes alike, outputs to rounding."""
    hq, hkv, d, n, page = 8, 2, 128, 300, 32
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn((n, h, d), generator=g).to(DEV) for h in (hq, hkv, hkv))
    flat = vf.KvCache(vf.KvCacheConfig(1, hkv, d, 512, dtype=F8))
    old = vf.Forward(flat, hq)
    old.b_step_kv_write(0, 0, n, k, v)
    o_old, d_old = torch.empty_like(q), torch.empty((hq, d), device=DEV)
    old.b_step_attention(0, 0, n, q, o_old)
    old.run_scalar_attn(0, n - 1, q[-1].contiguous(), d_old)
    c = vf.PagedKvCache(vf.PagedKvConfig(1, hkv, d, page, 12, F8))
    table = torch.tensor([[7, 2, 9, 0, 1, 11, 3, 4, 10, 5]], dtype=torch.int32, device=DEV)
    kv = torch.tensor([n], dtype=torch.int32, device=DEV)
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(table, kv, off, n_tokens=n)
    new = vf.PagedForward(c, hq)
    new.qk_rope_kv_write(0, batch, None, k, v, vf.MRope(0))
    o_new, d_new = torch.empty_like(q), torch.empty((1, hq, d), device=DEV)
    new.prefill_attention(0, batch, q, o_new)
    new.decode_attention(0, vf.SeqBatch(table, kv), q[-1:].contiguous(), d_new)
    torch.cuda.synchronize()
    assert (o_old - o_new).abs().max() < 1e-4 and (d_old - d_new[0]).abs().max() < 1e-4


def test_two_streams_with_workspaces_of_their_own():
    pools = [Pool(F8, 2, 128, 16, [900, 40], seed=i) for i in range(2)]
    fwds = [vf.PagedForward(p.cache, 8) for p in pools]
    qs = [rand_q(2, 8, 128, seed=i) for i in range(2)]
    outs = [torch.empty_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                fwds[i].decode_attention(0, pools[i].batch(), qs[i], outs[i])
    torch.cuda.synchronize()
    for i in range(2):
        ref, tol = attention(pools[i], qs[i], [1, 1])
        assert (outs[i].cpu().double() - ref).abs().max() <= tol


@IOS
def test_prefill_captured_follows_its_arrays(io):
    """One captured prefill call, replayed with other lengths, offsets and page tables, against the eager call."""
    pool = Pool(F8, 2, 128, 16, [200, 90, 33], spare=0)
    fwd = vf.PagedForward(pool.cache, 8)
    n = 60
    off = torch.tensor([0, 20, 21, 55], dtype=torch.int32, device=DEV)
    kv, table = pool.kv_dev.clone(), pool.table_dev.clone()
    batch = vf.SeqBatch(table, kv, off, n_tokens=n)
    q = rand_q(n, 8, 128, io)
    o = torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fwd.prefill_attention(0, batch, q, o, window=70, n_sink=5)
    for rep, (lens, offsets) in enumerate((([200, 90, 33], [0, 20, 21, 55]), ([20, 90, 0], [0, 5, 40, 40]), ([199, 1, 33], [0, 0, 1, 34]),
                                           ([200, 64, 32], [0, 30, 59, 60]))):
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        off.copy_(torch.tensor(offsets, dtype=torch.int32))
        q.copy_(rand_q(n, 8, 128, io, seed=rep))
        o.fill_(7.0)
        graph.replay()
        eager = torch.full_like(o, 7.0)
        fwd.prefill_attention(0, batch, q, eager, window=70, n_sink=5)
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and bool((o[offsets[-1]:] == 7.0).all()) and bool(o.isfinite().all())
        (q * 2).sum().item()


def test_decode_4096_sequences():
    kv = [(13 * i) % 37 for i in range(4096)]
    pool = Pool(F16, 1, 16, 16, kv)
    fwd = vf.PagedForward(pool.cache, 2)
    q = rand_q(4096, 2, 16)
    for bound in (36, 0, 5000):                            # a workgroup per sequence; dealt
        o = torch.full_like(q, float("nan"))
        fwd.decode_attention(0, vf.SeqBatch(pool.table_dev, pool.kv_dev, max_kv_len=bound), q, o)
        torch.cuda.synchronize()
        assert bool(o.isfinite().all())
        for s in (0, 1, 5, 37, 2047, 4094, 4095):
            one = Pool.__new__(Pool)
            one.__dict__.update(pool.__dict__)
            one.kv, one.table = [kv[s]], pool.table[s:s + 1]
            ref, tol = attention(one, q[s:s + 1], [1])
            assert (o[s:s + 1].cpu().double() - ref).abs().max() <= tol, s
    wide = torch.zeros((4097, 1), dtype=torch.int32, device=DEV)
    with pytest.raises(vf.VfkvError) as e:
        fwd.decode_attention(0, vf.SeqBatch(wide, torch.zeros(4097, dtype=torch.int32, device=DEV)), rand_q(4097, 2, 16), rand_q(4097, 2, 16, seed=2))
    assert e.value.status == -4


@pytest.mark.parametrize("dtype, d, unit", [(F8, 128, 32), (F8, 64, 64), (F16, 64, 32), (F16, 256, 16), (F32, 128, 16), (F8, 256, 32)])
def test_decode_lengths_around_the_ways_of_dealing(dtype, d, unit):
    for kv in ([32 * unit - 1], [32 * unit], [32 * unit + 1], [33 * unit, 1, 40 * unit + 3, 0, unit], [unit, unit + 1, unit - 1, 1]):
        pool = Pool(dtype, 2, d, 64, kv)
        check_attention(pool, 4, [1] * len(kv), decode=True)
        check_attention(pool, 4, [1] * len(kv), decode=True, max_kv_len=1)      # a bound that does not hold: slower, not wrong


def test_write_many_sequences_and_offsets():
    n = 150                                                   # more sequences than lanes
    q_len = [(7 * i) % 4 for i in range(n)]
    kv = [m + (11 * i) % 29 for i, m in enumerate(q_len)]
    write_case(F8, torch.float32, 4, 2, 64, 16, q_len, kv, 64, vf.ROPE_NEOX, [32], False)
    write_case(F16, torch.float16, 2, 1, 33, 16, q_len, kv, 32, vf.ROPE_NORM, [8, 8], True)


def test_sequences_may_share_pages():
    pool = Pool(F16, 2, 64, 16, [64, 80])
    pool.table[1, :4] = pool.table[0, :4]
    pool.table_dev.copy_(pool.table)
    check_attention(pool, 4, [1, 1], decode=True)
    check_attention(pool, 4, [30, 40])


@DTYPES
@IOS
def test_values_of_later_tokens_do_not_reach_earlier_ones(dtype, io):
    """Infinities and NaN in V rows of the chunk itself: the rows that see them get them, the earlier ones are untouched."""
    bad = float("nan") if dtype == F8 else float("inf")
    for hq, m, window in ((2, 70, 0), (8, 40, 0), (2, 70, 20), (1, 300, 33)):
        pool = Pool(dtype, 1, 128, 16, [m + 30])
        at = m + 10                                           # a key in the middle of the chunk
        p, sl = int(pool.table[0, at // 16]), at % 16
        clean = Pool(dtype, 1, 128, 16, [m + 30])
        row = pool.v[0, p, 0, sl].float().clone()
        row[5] = bad
        pool.v[0, p, 0, sl] = row.to(pool.v.dtype)
        fwd = [vf.PagedForward(x.cache, hq) for x in (pool, clean)]
        q = rand_q(m, hq, 128, io)
        o = [torch.zeros_like(q) for _ in range(2)]
        for f, x, y in zip(fwd, (pool, clean), o):
            f.prefill_attention(0, x.batch([m]), q, y, window=window)
        torch.cuda.synchronize()
        pos = torch.arange(30, m + 30, device=DEV)
        sees = (pos >= at) & ((pos - window < at) if window else True)
        assert bool(sees.any()) and not bool(sees.all())
        hit = ~o[0].isfinite()
        assert bool(hit[sees][:, :, 5].all()) and not bool(hit[~sees].any()) and not bool(hit[..., :5].any()) and not bool(hit[..., 6:].any())
        same = o[0].clone()
        same[..., 5] = o[1][..., 5] = 0
        assert torch.equal(same, o[1])


def test_batch_on_another_device_is_refused():
    pool = Pool(F16, 1, 64, 16, [5])
    fwd = vf.PagedForward(pool.cache, 2)
    pool.cache.device = 1                                     # as if the cache were there
    with pytest.raises(ValueError):
        fwd.decode_attention(0, pool.batch(), rand_q(1, 2, 64), rand_q(1, 2, 64, seed=2))
    with pytest.raises(ValueError):
        fwd.qk_rope_kv_write(0, pool.batch(), None, rand_q(1, 1, 64), rand_q(1, 1, 64), vf.MRope(0))


def test_prefill_without_a_workspace():
    import ctypes as C
    from vulkanforge_amd import _ffi
    pool = Pool(F8, 2, 128, 16, [3000])
    q = rand_q(5, 8, 128)
    o = torch.empty_like(q)
    b = pool.batch([5])
    p = _ffi.PagedAttnParams(8, 0, 0, 0, 0, 0, 1.0 / math.sqrt(128), 0.0)
    _ffi.check(_ffi.lib().vfkv_paged_prefill_attention(pool.cache.handle, 0, b.args, C.byref(p), q.data_ptr(), o.data_ptr(), None,
                                                       torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    ref, tol = attention(pool, q, [5])
    assert (o.cpu().double() - ref).abs().max() <= tol


def test_a_small_workspace_only_limits_the_split():
    pool = Pool(F8, 2, 128, 16, [5000, 40])
    for max_seq in (1, 64, 256, 100000):
        ws = vf.Workspace(8, 128, max_seq)
        ws.handle = ws._h
        fwd = vf.PagedForward(pool.cache, 8, workspace=ws)
        for q_len in (None, [9, 3]):
            n = 2 if q_len is None else 12
            q = rand_q(n, 8, 128)
            o = torch.full_like(q, float("nan"))
            (fwd.decode_attention if q_len is None else fwd.prefill_attention)(0, pool.batch(q_len), q, o)
            torch.cuda.synchronize()
            ref, tol = attention(pool, q, q_len or [1, 1])
            assert (o.cpu().double() - ref).abs().max() <= tol


def test_generic_kernel_leaves_a_note():
    from vulkanforge_amd import _ffi
    note = lambda: _ffi.lib().vfkv_last_note()  # noqa: E731
    for d, text in ((64, b""), (72, b"generic")):
        pool = Pool(F16, 1, d, 16, [20])
        fwd = vf.PagedForward(pool.cache, 2)
        q = rand_q(1, 2, d)
        for call in (fwd.decode_attention, ):
            call(0, pool.batch(), q, torch.empty_like(q))
            assert (text in note()) if text else note() == b""
    torch.cuda.synchronize()


@CALL
@IOS
@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("d, hq, hkv, page", [(512, 8, 1, 64), (512, 4, 4, 16), (272, 6, 2, 32), (320, 33, 1, 128), (448, 16, 2, 256)])
def test_rows_wider_than_256(d, hq, hkv, page, dtype, io, decode):
    from vulkanforge_amd import _ffi
    kv = [130, 1, 0, 700, 33]
    q_len = [1] * 5 if decode else [130, 1, 0, 65, 20]
    check_attention(Pool(dtype, hkv, d, page, kv), hq, q_len, io, decode=decode)
    assert _ffi.lib().vfkv_last_note() == b""                  # (the matrix-core kernels, not the generic one)
    check_attention(Pool(dtype, hkv, d, page, kv), hq, q_len, io, window=37, sink=5, softcap=20.0, decode=decode)


@IOS
@pytest.mark.parametrize("dtype", [F16, F8])
def test_rows_wider_than_256_over_long_contexts(dtype, io):
    # few rows: the keys go to many workgroups and are joined
    for d in (512, 336):
        pool = Pool(dtype, 2, d, 64, [5000, 40])
        check_attention(pool, 8, [1, 1], io, decode=True)
        check_attention(pool, 8, [7, 3], io)
        check_attention(pool, 8, [7, 3], io, window=2000, sink=70)


@IOS
@pytest.mark.parametrize("dtype", [F16, F8])
def test_wide_rows_hide_what_is_not_seen(dtype, io):
    """Pages that are not there, and V elements that are not finite, in every quarter of a row of 512 elements."""
    bad = float("nan") if dtype == F8 else float("inf")
    pool = Pool(dtype, 1, 512, 16, [100, 50])
    pool.table[0, 2] = -1
    pool.table[1, 0] = 10 ** 6
    pool.table_dev.copy_(pool.table)
    check_attention(pool, 4, [40, 50], io)
    check_attention(pool, 4, [1, 1], io, decode=True)
    for hq, m, window in ((2, 70, 0), (8, 40, 20)):
        pool, clean = (Pool(dtype, 1, 512, 16, [m + 30]) for _ in range(2))
        at = m + 10
        p, sl = int(pool.table[0, at // 16]), at % 16
        row = pool.v[0, p, 0, sl].float().clone()
        odd = [5, 200, 300, 511]
        row[odd] = bad
        pool.v[0, p, 0, sl] = row.to(pool.v.dtype)
        q = rand_q(m, hq, 512, io)
        o = [torch.zeros_like(q) for _ in range(2)]
        for x, y in zip((pool, clean), o):
            vf.PagedForward(x.cache, hq).prefill_attention(0, x.batch([m]), q, y, window=window)
        torch.cuda.synchronize()
        pos = torch.arange(30, m + 30, device=DEV)
        sees = (pos >= at) & ((pos - window < at) if window else True)
        hit = ~o[0].isfinite()
        want = torch.zeros_like(hit)
        want[:, :, odd] = sees[:, None, None]
        assert torch.equal(hit, want)
        assert torch.equal(o[0][~hit], o[1][~hit])


def test_f32_pages_wider_than_256_take_the_generic_kernel():
    from vulkanforge_amd import _ffi
    pool = Pool(F32, 1, 512, 16, [70, 3])
    for decode, q_len in ((True, [1, 1]), (False, [30, 3])):
        check_attention(pool, 2, q_len, decode=decode)
        assert b"generic" in _ffi.lib().vfkv_last_note()


@CALL
@DTYPES
@pytest.mark.parametrize("d", [64, 80, 128, 256, 512])
def test_tiny_and_huge_queries_keep_their_accuracy(d, dtype, decode):
    """Queries of any size, with a scale that brings the scores to ordinary sizes: an element counts to 2^-22 of its row's largest."""
    pool = Pool(dtype, 2, d, 32, [70, 3, 129])
    q_len = [1] * 3 if decode else [40, 3, 5]
    for size, softcap in ((2.0 ** -24, 0.0), (2.0 ** -24, 3.0), (2.0 ** 40, 0.0), (2.0 ** -70, 0.0)):
        q = rand_q(sum(q_len), 4, d, scale=size)
        q[:, 1] *= 2.0 ** -10                                 # heads of one token far apart
        scale = 1.0 / (size * math.sqrt(d))
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, 4)
        call = fwd.decode_attention if decode else fwd.prefill_attention
        call(0, pool.batch(None if decode else q_len), q, o, scale=scale, softcap=softcap)
        torch.cuda.synchronize()
        ref, tol = attention(pool, q, q_len, softcap=softcap, scale=scale)
        err = (o.cpu().double() - ref).abs().max().item()
        print(f"{size:.3g} {softcap}: {err:.3g} of {tol:.3g}", flush=True)
        assert err <= tol


@CALL
def test_windows_of_any_size_do_not_wrap(decode):
    pool = Pool(F16, 2, 64, 16, [200, 33])
    q_len = [1, 1] if decode else [90, 33]
    top = 2 ** 32 - 1
    full = check_attention(pool, 4, q_len, decode=decode)[1]
    for window, sink in ((top, 0), (top, top), (1, top), (0, top), (top - 1, 5)):
        o = check_attention(pool, 4, q_len, decode=decode, window=window, sink=sink)[1]
        assert (o - full).abs().max() < 1e-5


@pytest.mark.parametrize("dtype, io", [(F8, torch.float16), (F16, torch.float16), (F8, torch.float32)])
@pytest.mark.parametrize("window", [100, 384, 700, 1536, 1600])
def test_windows_around_the_choice_of_wavefronts(dtype, io, window):
    # chunks that fill blocks of 256 rows: four or eight wavefronts by the window
    pool = Pool(dtype, 1, 128, 64, [2300, 700])
    check_attention(pool, 4, [2300, 600], io, window=window, sink=0 if window in (384, 1536) else 3)


@IOS
@pytest.mark.parametrize("dtype", [F16, F8])
def test_wide_rows_captured(dtype, io):
    """Captured decode and prefill over rows of 512, replayed with other lengths, against the eager calls."""
    pool = Pool(dtype, 2, 512, 16, [700, 90, 33], spare=0)
    fwd = vf.PagedForward(pool.cache, 8)
    off = torch.tensor([0, 20, 21, 50], dtype=torch.int32, device=DEV)
    kv, table = pool.kv_dev.clone(), pool.table_dev.clone()
    chunk, step = vf.SeqBatch(table, kv, off, n_tokens=50), vf.SeqBatch(table, kv)
    q, q1 = rand_q(50, 8, 512, io), rand_q(3, 8, 512, io)
    o, o1 = torch.zeros_like(q), torch.zeros_like(q1)

    def calls(a, b):
        fwd.prefill_attention(0, chunk, q, a)
        fwd.decode_attention(0, step, q1, b)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(o, o1)
    for rep, lens in enumerate(([700, 90, 33], [20, 90, 0], [699, 1, 33], [512, 64, 32])):
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(rand_q(50, 8, 512, io, seed=rep))
        graph.replay()
        eager, eager1 = torch.zeros_like(o), torch.zeros_like(o1)
        calls(eager, eager1)
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and torch.equal(o1, eager1) and bool(o.isfinite().all())


@pytest.mark.parametrize("dtype", [F16, F8])
def test_wide_rows_around_the_ways_of_dealing(dtype):
    # a workgroup per sequence up to 256 keys, from 128 workgroups on up to 1 024; dealt beyond
    for n in (255, 256, 257):
        check_attention(Pool(dtype, 1, 512, 16, [n, 1, 17]), 2, [1] * 3, decode=True, max_kv_len=n)
    for n in (1024, 1040):
        kv = [n] + [5 + 3 * i % 70 for i in range(127)]
        check_attention(Pool(dtype, 1, 512, 16, kv), 2, [1] * 128, decode=True, max_kv_len=n)
