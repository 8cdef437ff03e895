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
