"""Paged cache: what device arrays may say that the kernels must not follow -- positions that the page table cannot hold, pages and
offsets that do not exist.  Position j has its row in page table[j / page_size]; one without a page has no row."""
import pytest
import torch

import vulkanforge_amd as vf
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
