"""Paged cache: what device arrays may say that the kernels must not follow -- positions that the page table cannot hold, pages and
offsets that do not exist.  Position j has its row in page table[j / page_size]; one without a page has no row."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import DEV, Pool, turned

pytestmark = pytest.mark.gpu
F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8


def as_bytes(x):
    return x.view(torch.uint8)


@pytest.mark.parametrize("d", [64, 33])
def test_write_drops_rows_that_have_no_place(d):
    """A length beyond the table, a negative one, pages that do not exist, tokens in front of the first position."""
    page = 16
    pool = Pool(F16, 2, d, page, [16, 16, 16, 16, 16], spare=2, extra_entries=0)
    pool.table_dev[0, 0] = 10_000
    pool.table_dev[1, 0] = -5
    pool.kv_dev.copy_(torch.tensor([16, 16, 900, -7, 2], dtype=torch.int32))
    fwd = vf.PagedForward(pool.cache, 2)
    n = 5 * 3
    off = torch.arange(0, n + 1, 3, dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(pool.table_dev, pool.kv_dev, off, n_tokens=n)
    k, v = (torch.full((n, 2, d), float(i + 1), device=DEV) for i in range(2))
    want_k, want_v = pool.k.clone(), pool.v.clone()
    fwd.qk_rope_kv_write(0, batch, None, k, v, vf.MRope(0))
    torch.cuda.synchronize()
    want_k[0, int(pool.table[4, 0]), :, 0:2] = 1.0            # three tokens, two positions: the first has no row
    want_v[0, int(pool.table[4, 0]), :, 0:2] = 2.0
    assert torch.equal(as_bytes(pool.k), as_bytes(want_k)) and torch.equal(as_bytes(pool.v), as_bytes(want_v))
    # offsets that run backwards or leave the rows
    bad = torch.tensor([-3, 9, 4, 99, 15, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    pool.kv_dev.fill_(16)
    pool.table_dev.copy_(pool.table)
    fwd.qk_rope_kv_write(0, vf.SeqBatch(pool.table_dev, pool.kv_dev, bad, n_tokens=n), None, k, v, vf.MRope(0))
    o = torch.zeros((n, 2, d), device=DEV)
    fwd.prefill_attention(0, vf.SeqBatch(pool.table_dev, pool.kv_dev, bad, n_tokens=n), torch.ones_like(o), o)
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [64, 36])
@pytest.mark.parametrize("kv", [17, 18, 20, 21, 2 ** 31 - 1])
def test_write_across_the_end_of_the_table(d, kv):
    """A chunk of five whose last tokens are beyond the table of 16 positions: the others get their rows, all queries their angles."""
    pool = Pool(F32, 1, d, 16, [16], spare=2, extra_entries=0)
    pool.kv_dev.fill_(kv)
    g = torch.Generator().manual_seed(kv % 97)
    q, k, v = (torch.randn((5, h, d), generator=g).to(DEV) for h in (2, 1, 1))
    out = torch.zeros_like(q)
    want_k, want_v = pool.k.clone(), pool.v.clone()
    batch = vf.SeqBatch(pool.table_dev, pool.kv_dev, torch.tensor([0, 5], dtype=torch.int32, device=DEV), n_tokens=5)
    vf.PagedForward(pool.cache, 2).qk_rope_kv_write(0, batch, q, k, v, vf.MRope(d, 1e4), q_out=out)
    torch.cuda.synchronize()
    pos = [kv - 5 + i for i in range(5)]
    rq, rk = (turned(x, None, [pos], 1e4, d, [d // 2], False, vf.ROPE_NEOX) for x in (q, k))
    # two products and a sum (4 half steps), cos and sin (11), of elements below 5
    assert (out.cpu().double() - rq).abs().max() <= 2 * 5 * 15 * 2.0 ** -24
    p = int(pool.table[0, 0])
    for i, j in enumerate(pos):
        if j < 16:
            assert (pool.k[0, p, 0, j].cpu().double() - rk[i, 0]).abs().max() <= 2 * 5 * 15 * 2.0 ** -24
            want_k[0, p, 0, j] = pool.k[0, p, 0, j]
            want_v[0, p, 0, j] = v[i, 0]
    assert torch.equal(as_bytes(pool.k), as_bytes(want_k)) and torch.equal(as_bytes(pool.v), as_bytes(want_v))


def test_write_up_to_the_longest_length():
    """A table for more than 2^23 positions: rows from there on are dropped."""
    top = 2 ** 23
    pool = Pool(F16, 1, 64, 16, [16, 16], spare=1, extra_entries=0)
    a, b = int(pool.table[0, 0]), int(pool.table[1, 0])
    table = torch.full((1, top // 16 + 2), -1, dtype=torch.int32)
    table[0, top // 16 - 1], table[0, top // 16] = a, b
    k = torch.arange(1, 7, device=DEV).float()[:, None, None].expand(6, 1, 64).contiguous()
    want = pool.k.clone()
    want[0, a, 0, 13:16] = k[:3, 0].half()
    kv = torch.tensor([top + 3], dtype=torch.int32, device=DEV)
    batch = vf.SeqBatch(table.to(DEV), kv, torch.tensor([0, 6], dtype=torch.int32, device=DEV), n_tokens=6)
    vf.PagedForward(pool.cache, 1).qk_rope_kv_write(0, batch, None, k, k.clone(), vf.MRope(0))
    torch.cuda.synchronize()
    assert torch.equal(as_bytes(pool.k), as_bytes(want))


def test_captured_step_replayed_past_its_table_leaves_shared_pages_alone():
    """Two forks of 32 positions share two full pages; a captured step that runs on after their table of three pages is full
    writes nothing more."""
    c = vf.PagedKvCache(vf.PagedKvConfig(1, 1, 64, 16, 8, F16), k_buffer=(kb := torch.zeros((1, 8, 1, 16, 64), dtype=torch.float16, device=DEV)).data_ptr(),
                        v_buffer=(vb := torch.zeros_like(kb)).data_ptr())
    first = c.alloc(2)
    lists = [first + c.alloc(1), c.fork(first, 32, 1)[0].tolist() + c.alloc(1)]
    table = torch.tensor(lists, dtype=torch.int32, device=DEV)
    kv = torch.full((2,), 32, dtype=torch.int32, device=DEV)
    fwd, batch = vf.PagedForward(c, 1), vf.SeqBatch(table, kv)
    k = torch.zeros((2, 1, 64), device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fwd.qk_rope_kv_write(0, batch, None, k, k, vf.MRope(0))
    for step in range(1, 24):
        kv.fill_(32 + step)
        k.fill_(float(step))
        graph.replay()
        if step == 16:
            torch.cuda.synchronize()
            full = kb.clone(), vb.clone()
    torch.cuda.synchronize()
    assert torch.equal(kb, full[0]) and torch.equal(vb, full[1])
    assert float(kb[0, first].abs().max()) == 0.0 and [float(kb[0, x[2], 0, j, 0]) for x in lists for j in (0, 15)] == [1.0, 16.0] * 2


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype, d", [(F16, 64), (F8, 128), (F32, 128), (F8, 40), (F32, 256), (F16, 512), (F16, 256)])
@pytest.mark.parametrize("window, sink", [(0, 0), (20, 0), (40, 5), (100, 64), (7, 130), (1, 0)])
def test_queries_beyond_the_table_see_what_is_in_front_of_its_end(decode, dtype, d, window, sink):
    """Positions count from the length as given, so a window moves on when the keys do not."""
    page = 16
    pool = Pool(dtype, 2, d, page, [176, 64, 16, 176, 176, 176, 176], spare=1, extra_entries=0)    # (176: not a multiple of any tile)
    lens = [177, 70, 16, 190, 176 + 45, 5000, 2 ** 31 - 1]
    pool.kv_dev.copy_(torch.tensor(lens, dtype=torch.int32))
    q_len = [1] * 7 if decode else [9, 70, 3, 60, 100, 2, 1]
    n = sum(q_len)
    for io in (torch.float32, torch.float16):
        q = torch.randn((n, 8, d), generator=torch.Generator().manual_seed(d)).to(io).to(DEV)
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, 8)
        (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else q_len), q, o, window=window, n_sink=sink)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, q_len, window, sink, lens=lens)
        assert_near(o, ref, bound, io)


@pytest.mark.parametrize("dtype, d, io", [(F16, 64, torch.float32), (F8, 64, torch.float16), (F8, 128, torch.float16), (F16, 256, torch.float16)])
@pytest.mark.parametrize("window", [0, 50])
def test_blocks_of_256_rows_across_the_end_of_the_table(dtype, d, io, window):
    pool = Pool(dtype, 1, d, 16, [1040], spare=1, extra_entries=0)
    q = torch.randn((400, 4, d), generator=torch.Generator().manual_seed(d)).to(io).to(DEV)
    for length in (1041, 1100, 1240, 1439, 1440, 1600):
        pool.kv_dev.fill_(length)
        o = torch.full_like(q, float("nan"))
        vf.PagedForward(pool.cache, 4).prefill_attention(0, pool.batch([400]), q, o, window=window, n_sink=window // 10)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, [400], window, window // 10, lens=[length])
        assert_near(o, ref, bound, io, length)


@pytest.mark.parametrize("decode", [True, False])
def test_long_tables_and_lengths_beyond_them_in_parts(decode):
    pool = Pool(F8, 1, 128, 64, [5120, 64], spare=1, extra_entries=0)
    lens = [5300, 5120 + 3]
    pool.kv_dev.copy_(torch.tensor(lens, dtype=torch.int32))
    q_len = [1, 1] if decode else [7, 3]
    for window, sink in ((0, 0), (2000, 70), (150, 1)):
        q = torch.randn((sum(q_len), 4, 128), generator=torch.Generator().manual_seed(window)).to(DEV)
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, 4)
        (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else q_len), q, o, window=window, n_sink=sink)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, q_len, window, sink, lens=lens)
        assert_near(o, ref, bound, torch.float32)


@pytest.mark.parametrize("dtype, d", [(F16, 64), (F8, 128), (F32, 64)])
def test_rows_behind_the_end_of_the_table_do_not_reach_the_output(dtype, d):
    """The tile that the table's end cuts: what lies in the last page behind it is not there, whatever it holds."""
    pool = Pool(dtype, 1, d, 16, [48], spare=1, extra_entries=0)
    bad = float("nan")
    last = int(pool.table[0, 2])
    q = torch.randn((90, 2, d), generator=torch.Generator().manual_seed(1)).to(DEV)
    other = [p for p in range(pool.k.shape[1]) if p not in pool.table[0].tolist()]
    for x in (pool.k, pool.v):
        x[0, other] = torch.full_like(x[0, other].float(), bad).to(x.dtype)
    for length in (49, 64, 90, 120):
        pool.kv_dev.fill_(length)
        o = torch.full_like(q, float("nan"))
        vf.PagedForward(pool.cache, 2).prefill_attention(0, pool.batch([90]), q, o)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, [90], lens=[length])
        assert last < pool.k.shape[1]
        assert_near(o, ref, bound, torch.float32, length)
