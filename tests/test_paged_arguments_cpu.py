"""Paged cache, Python layer: numbers that do not fit the 32 bits of the C ABI, without a device."""
import pytest

import vulkanforge_amd as vf


def pool(n_pages=10, page=16, dtype=vf.KvDtype.F16, layers=2, hkv=2, d=64):
    return vf.PagedKvCache(vf.PagedKvConfig(layers, hkv, d, page, n_pages, dtype), layout_only=True)


@pytest.mark.parametrize("kv_len, n_forks", [(-1, 1), (-5, 1), (-15, 2), (-16, 1), (-(2 ** 32) + 20, 1), (2 ** 32, 1), (2 ** 32 + 40, 1),
                                             (20, -1), (20, 2 ** 32 + 1), (0, -1)])
def test_fork_of_impossible_numbers_is_refused(kv_len, n_forks):
    """(A length below zero passed for no pages here and for 2^28 pages behind the call, which read past the list.)"""
    c = pool()
    mine = c.alloc(2)
    with pytest.raises(ValueError):
        c.fork(mine, kv_len, n_forks)
    assert c.free_count == 8 and [c.refcount(p) for p in mine] == [1, 1]


def test_alloc_of_impossible_counts_is_refused():
    c = pool()
    for n in (-1, 11, 2 ** 32, 2 ** 32 + 1, 2 ** 40, 2 ** 63):
        with pytest.raises(vf.VfkvError) as e:
            c.alloc(n)
        assert e.value.status == -7 and c.free_count == 10
    assert c.alloc(10) == list(range(10)) and c.alloc(0) == []


def test_pages_and_layers_do_not_wrap():
    c = pool()
    c.alloc(4)
    for page in (2 ** 32, 2 ** 32 + 1, -(2 ** 32), 2 ** 64):
        assert c.refcount(page) == 0 and c.offset_bytes(0, page) == 0
    assert c.offset_bytes(0, 1) > 0 and c.offset_bytes(2 ** 32, 1) == 0 and c.offset_bytes(1, 2 ** 32 + 1) == 0


@pytest.mark.parametrize("kw", [dict(n_pages=2 ** 32 + 4), dict(page=2 ** 32 + 16), dict(d=2 ** 32 + 64), dict(layers=2 ** 32 + 1),
                                dict(hkv=2 ** 32 + 2), dict(n_pages=-1), dict(d=-1), dict(layers=-1), dict(hkv=-1), dict(page=-16)])
def test_configurations_do_not_wrap(kw):
    with pytest.raises(vf.VfkvError):
        pool(**kw)


class _Rows:
    """Stands in for a batch and rows: what the attention call passes on is what is looked at."""
    index, args = 0, None


@pytest.mark.parametrize("given, passed", [((0, 0), (0, 0)), ((2 ** 32 - 1, 7), (2 ** 32 - 1, 7)), ((2 ** 32 + 5, 0), (2 ** 32 - 1, 0)),
                                           ((5, 2 ** 32), (5, 2 ** 32 - 1)), ((2 ** 70, 2 ** 70), (2 ** 32 - 1, 2 ** 32 - 1))])
def test_windows_and_layers_of_calls_do_not_wrap(given, passed, monkeypatch):
    c = pool()
    fwd = vf.PagedForward(c, 4, workspace=type("W", (), {"handle": None})())
    monkeypatch.setattr(fwd, "_rows", lambda t, heads, batch, name: (0, heads * 64, 0))
    seen = {}

    def fn(handle, layer, batch, p, q, o, ws, stream):
        seen.update(layer=layer, window=p._obj.window, n_sink=p._obj.n_sink)
        return 0

    for layer, there in ((1, 1), (2 ** 32, 2 ** 32 - 1), (2 ** 32 + 1, 2 ** 32 - 1), (-1, 2 ** 32 - 1), (-(2 ** 32), 2 ** 32 - 1)):
        fwd._attention(fn, layer, _Rows, None, None, *given, None, 0.0, 0)
        assert seen == dict(layer=there, window=passed[0], n_sink=passed[1])
    for bad in ((-1, 0), (0, -1), (-(2 ** 32) + 5, 0)):
        with pytest.raises(ValueError):
            fwd._attention(fn, 0, _Rows, None, None, *bad, None, 0.0, 0)


def test_rotations_do_not_wrap():
    # (2^32 - 1 is odd and no number of pairs: the call refuses it)
    assert vf.MRope(2 ** 32 + 64, sections=[32])._args.rotary_dim == 2 ** 32 - 1
    assert list(vf.MRope(64, sections=[2 ** 32 + 16, 16])._args.section[:2]) == [2 ** 32 - 1, 16]
    assert vf.MRope(64, sections=[-1, 33])._args.section[0] == 2 ** 32 - 1
    assert vf.MRope(64, rope_mode=2 ** 32 + 2)._args.rope_mode == 2 ** 32 - 1
