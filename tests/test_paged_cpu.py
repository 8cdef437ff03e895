"""Paged cache without a device: layout, page counting, and the refusals of every entry point."""
import ctypes as C

import pytest

import vulkanforge_amd as vf
from vulkanforge_amd import _ffi

FAKE = 0x10000


def pool(n_pages=10, page=16, dtype=vf.KvDtype.F16, layers=2, hkv=2, d=64, **kw):
    return vf.PagedKvCache(vf.PagedKvConfig(layers, hkv, d, page, n_pages, dtype), layout_only=True, **kw)


@pytest.mark.parametrize("dtype", list(vf.KvDtype))
def test_layout(dtype):
    c = pool(7, 32, dtype, layers=3, hkv=5, d=80)
    page = 5 * 32 * 80 * dtype.element_size()
    assert c.bytes_per_buffer() == 3 * 7 * page
    assert c.offset_bytes(2, 3) == (2 * 7 + 3) * page
    assert c.offset_bytes(3, 0) == 0 and c.offset_bytes(0, 7) == 0
    assert c.k_ptr == 0 and c.v_ptr == 0
    assert c.pages_for(0) == 0 and c.pages_for(1) == 1 and c.pages_for(32) == 1 and c.pages_for(33) == 2


@pytest.mark.parametrize("kw, status", [
    (dict(page=8), -1), (dict(page=48), -1), (dict(page=512), -1), (dict(n_pages=0), -1), (dict(hkv=0), -1),
    (dict(d=0), -1), (dict(d=513), -4), (dict(layers=0), -1), (dict(n_pages=1 << 27, page=16), -2), (dict(hkv=20000), -4)])
def test_bad_configurations_are_refused(kw, status):
    with pytest.raises(vf.VfkvError) as e:
        pool(**kw)
    assert e.value.status == status


def test_buffers_must_be_aligned_and_both_given():
    cfg = _ffi.PagesConfig(1, 1, 64, 16, 4, 1)
    h = C.c_void_p()
    L = _ffi.lib()
    assert L.vfkv_pages_create_external(C.byref(cfg), FAKE + 8, FAKE, C.byref(h)) == -3
    assert L.vfkv_pages_create_external(C.byref(cfg), FAKE, None, C.byref(h)) == -1
    assert L.vfkv_pages_create_external(None, None, None, C.byref(h)) == -1
    assert L.vfkv_pages_create_external(C.byref(cfg), None, None, None) == -1
    assert L.vfkv_pages_create(C.byref(cfg), None) == -1
    cfg.dtype = 3
    assert L.vfkv_pages_create_external(C.byref(cfg), None, None, C.byref(h)) == -1


def test_alloc_gives_the_lowest_free_pages_or_nothing():
    c = pool(6)
    assert c.alloc(0) == [] and c.alloc(4) == [0, 1, 2, 3] and c.free_count == 2
    with pytest.raises(vf.VfkvError) as e:
        c.alloc(3)
    assert e.value.status == -7 and c.free_count == 2
    c.release([2, 0])
    assert c.free_count == 4 and c.alloc(3) == [0, 2, 4] and c.refcount(4) == 1 and c.refcount(5) == 0
    assert c.refcount(-1) == 0 and c.refcount(6) == 0


def test_retain_and_release_count_repetitions_and_undo_on_errors():
    c = pool(6)
    c.alloc(3)
    c.retain([0, 0, 2, vf.paged.NO_PAGE])
    assert [c.refcount(p) for p in range(3)] == [3, 1, 2]
    for bad in ([0, 5], [0, 6], [0, 1, 1]):
        with pytest.raises(vf.VfkvError):
            c.release(bad)
        assert [c.refcount(p) for p in range(3)] == [3, 1, 2] and c.free_count == 3
    with pytest.raises(vf.VfkvError):
        c.retain([0, 4])
    assert c.refcount(0) == 3
    for bad in ([-2], [1 << 32], [0.5]):
        with pytest.raises(ValueError):
            c.release(bad)
    c.release([0, 0, 0, -1, 2, 2])                       # to zero in one call: one free page each
    assert c.free_count == 5 and c.alloc(5) == [0, 2, 3, 4, 5]


@pytest.mark.parametrize("kv, fresh", [(0, 0), (1, 1), (16, 0), (17, 1), (40, 1), (48, 0)])
def test_fork_shares_full_pages_and_owns_the_last(kv, fresh):
    c = pool(12)
    used = c.pages_for(kv)
    mine = c.alloc(used)
    a, b = c.fork(mine, kv, 2).tolist()
    full = kv // 16
    assert a[:full] == b[:full] == mine[:full] and len(a) == used
    assert [c.refcount(p) for p in mine[:full]] == [3] * full
    if fresh:
        assert {a[-1], b[-1]}.isdisjoint(mine) and a[-1] != b[-1] and c.refcount(a[-1]) == 1
    assert c.free_count == 12 - used - 2 * fresh
    for t in (mine, a, b):
        c.release(t)
    assert c.free_count == 12


def test_fork_refusals_change_nothing():
    c = pool(5)
    mine = c.alloc(3)
    with pytest.raises(vf.VfkvError) as e:
        c.fork(mine, 40, 3)                              # three last pages wanted, two free
    assert e.value.status == -7
    with pytest.raises(vf.VfkvError):
        c.fork([0, 4, 2], 40, 1)                         # page 4 is free
    with pytest.raises(ValueError):
        c.fork(mine[:2], 40, 1)
    assert c.fork(mine, 40, 0).shape == (0, 3)
    assert c.free_count == 2 and [c.refcount(p) for p in mine] == [1, 1, 1]
    t = c.fork([-1, 1, 2], 40, 1)[0].tolist()                     # the first page has left the window
    assert t[0] == -1 and t[1] == 1 and t[2] == 3
    t = c.fork([0, 1, -1], 40, 1)[0].tolist()
    assert t == [0, 1, -1]


def test_compact_moves_live_pages_to_the_front():
    c = pool(10)
    c.alloc(10)
    c.retain([8])
    c.release([0, 3, 4, 9, 2])
    ids = c.compact()                                    # live: 1 5 6 7 8 -> 0..4
    assert ids == [-1, 1, -1, -1, -1, 0, 2, 3, 4, -1]
    assert [c.refcount(p) for p in range(6)] == [1, 1, 1, 1, 2, 0]
    assert c.alloc(5) == [5, 6, 7, 8, 9]
    assert c.compact() == list(range(10))


def test_copy_refusals():
    c = vf.PagedKvCache(vf.PagedKvConfig(1, 1, 64, 16, 8, vf.KvDtype.F16), k_buffer=FAKE, v_buffer=FAKE)
    for src, dst, rows in (([0], [8], None), ([8], [0], None), ([0, 1], [2, 2], None), ([0, 1], [1, 3], None), ([3], [3], None),
                           ([0], [1], [17]), ([-1], [2], None)):
        with pytest.raises(vf.VfkvError) as e:
            c.copy_pages(src, dst, rows, stream=0)
        assert e.value.status == -1
    with pytest.raises(ValueError):
        c.copy_pages([0, 1], [2], stream=0)
    c.copy_pages([], [], stream=0)
    with pytest.raises(vf.VfkvError):
        pool().copy_pages([0], [1], stream=0)            # no buffers


def batch(**kw):
    a = dict(page_table=FAKE, kv_lens=FAKE, q_offsets=None, n_seqs=4, table_stride=2, n_tokens=4, max_kv_len=0)
    a.update(kw)
    return _ffi.SeqBatchArgs(*a.values())


def attn(**kw):
    a = dict(n_heads=4, window=0, n_sink=0, io_dtype=0, q_stride=0, o_stride=0, scale=0.125, softcap=0.0)
    a.update(kw)
    return _ffi.PagedAttnParams(*a.values())


@pytest.fixture
def ext():
    c = vf.PagedKvCache(vf.PagedKvConfig(2, 2, 64, 16, 8, vf.KvDtype.F16), k_buffer=FAKE, v_buffer=FAKE)
    yield c
    c.destroy()


@pytest.mark.parametrize("call", ["decode", "prefill"])
def test_attention_refusals_before_any_device_work(ext, call):
    L = _ffi.lib()
    fn = L.vfkv_paged_decode_attention if call == "decode" else L.vfkv_paged_prefill_attention

    def go(b=None, p=None, layer=0, q=FAKE, o=2 * FAKE, cache=ext.handle):
        return fn(cache, layer, C.byref(b or batch()), C.byref(p or attn()), q, o, None, None)

    for b in (batch(page_table=None), batch(kv_lens=None), batch(table_stride=0), batch(n_tokens=5)):
        assert go(b) == -1
    assert go(batch(n_seqs=4097, n_tokens=4097)) == -4
    assert go(batch(kv_lens=FAKE + 2)) == -3
    for p in (attn(n_heads=3), attn(n_heads=0), attn(scale=0.0), attn(scale=float("nan")), attn(scale=float("inf")),
              attn(softcap=-1.0), attn(softcap=float("nan")), attn(io_dtype=2), attn(q_stride=255), attn(o_stride=1)):
        assert go(p=p) == -1
    assert go(layer=2) == -1 and go(q=None) == -1 and go(o=None) == -1 and go(q=FAKE, o=FAKE) == -1 and go(cache=None) == -1
    assert go(q=FAKE + 2) == -3 and go(p=attn(io_dtype=1), q=FAKE + 1) == -3
    assert fn(ext.handle, 0, None, C.byref(attn()), FAKE, FAKE, None, None) == -1
    assert fn(ext.handle, 0, C.byref(batch()), None, FAKE, FAKE, None, None) == -1
    assert go(batch(n_seqs=0)) == 0 and go(batch(n_tokens=0)) == 0           # nothing to do
    layout = pool()
    assert go(cache=layout.handle) == -1
    if call == "decode":
        assert go(batch(q_offsets=FAKE)) == -1
        assert b"one token" in L.vfkv_last_error()
        assert go() == -1 and b"workspace" in L.vfkv_last_error()


def test_write_refusals_before_any_device_work(ext):
    L = _ffi.lib()

    def rows(**kw):
        a = dict(q=FAKE, q_norm_weight=None, q_out=FAKE, k=FAKE, v=FAKE, k_norm_weight=None, positions=None, freq_factors=None,
                 n_heads=4, io_dtype=0, q_stride=0, q_out_stride=0, k_stride=0, v_stride=0)
        a.update(kw)
        return _ffi.PagedRows(*a.values())

    def rope(**kw):
        a = dict(rope_mode=2, rotary_dim=64, n_axes=3, interleaved=0, section=(C.c_uint32 * 4)(16, 8, 8, 0), freq_base=1e4,
                 freq_scale=1.0, attn_factor=1.0, eps=1e-6)
        a.update(kw)
        return _ffi.MRopeParams(*a.values())

    def go(r=None, p=None, b=None, layer=0):
        return L.vfkv_paged_qk_rope_kv_write(ext.handle, layer, C.byref(b or batch()), C.byref(r or rows()), C.byref(p or rope()), None)

    assert go(p=rope(rope_mode=8)) == -4
    for p in (rope(rotary_dim=63), rope(rotary_dim=66), rope(n_axes=0), rope(n_axes=5), rope(interleaved=2), rope(n_axes=2),
              rope(section=(C.c_uint32 * 4)(16, 16, 8, 0)), rope(freq_base=0.0), rope(freq_base=float("inf")),
              rope(freq_scale=float("nan"))):
        assert go(p=p) == -1
    for r in (rows(k=None), rows(v=None), rows(q_out=None), rows(n_heads=0), rows(io_dtype=2), rows(q_stride=100),
              rows(k_stride=127), rows(v_stride=1), rows(q_stride=512)):
        assert go(r) == -1
    for r in (rows(k=FAKE + 2), rows(positions=FAKE + 1), rows(q_norm_weight=FAKE + 2), rows(io_dtype=1, v=FAKE + 1)):
        assert go(r) == -3
    assert go(layer=2) == -1
    assert go(b=batch(n_seqs=0)) == 0
    assert L.vfkv_paged_qk_rope_kv_write(ext.handle, 0, C.byref(batch()), None, C.byref(rope()), None) == -1
    assert L.vfkv_paged_qk_rope_kv_write(ext.handle, 0, C.byref(batch()), C.byref(rows()), None, None) == -1


def test_workspace_refusals():
    c = pool()
    L = _ffi.lib()
    h = C.c_void_p()
    assert L.vfkv_paged_workspace_create(c.handle, 3, C.byref(h)) == -1
    assert L.vfkv_paged_workspace_create(c.handle, 0, C.byref(h)) == -1
    assert L.vfkv_paged_workspace_create(None, 2, C.byref(h)) == -1
    assert L.vfkv_paged_workspace_create(c.handle, 2, None) == -1


@pytest.mark.parametrize("call", ["decode", "prefill"])
@pytest.mark.parametrize("kw", [dict(scale=1e-38), dict(scale=1e31), dict(softcap=1e-39), dict(softcap=3e38), dict(softcap=float("inf"))])
def test_scale_and_softcap_that_leave_the_normal_numbers_are_refused(ext, call, kw):
    # (their reciprocals and products with log2 e would be infinite or zero: 0 * inf is NaN)
    L = _ffi.lib()
    fn = L.vfkv_paged_decode_attention if call == "decode" else L.vfkv_paged_prefill_attention
    assert fn(ext.handle, 0, C.byref(batch()), C.byref(attn(**kw)), FAKE, 2 * FAKE, None, None) == -1
    assert list(kw)[0].encode() in L.vfkv_last_error()
