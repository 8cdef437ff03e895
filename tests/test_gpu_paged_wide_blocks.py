"""Paged prefill in blocks of 256 rows (eight wavefronts): chunks that fill them, over a context at least twice as long."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import DEV, Pool

pytestmark = pytest.mark.gpu
F16, F8 = vf.KvDtype.F16, vf.KvDtype.F8
KV, CHUNKS, HEADS = [2500, 700], [200, 131], 4       # 1 324 rows of one KV head: at least 256 per sequence, contexts longer than 2 * 166


def run(pool, io, q_len, seed, window=0, sink=0, softcap=0.0):
    q = torch.randn((sum(q_len), HEADS * pool.hkv, pool.d), generator=torch.Generator().manual_seed(seed)).to(io).to(DEV)
    o = torch.full_like(q, float("nan"))
    fwd = vf.PagedForward(pool.cache, HEADS * pool.hkv)
    fwd.prefill_attention(pool.layer, pool.batch(q_len), q, o, window=window, n_sink=sink, softcap=softcap)
    torch.cuda.synchronize()
    return q, o


@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [16, 48, 64, 96, 128, 144, 192, 256])
@pytest.mark.parametrize("softcap", [0.0, 50.0])
@pytest.mark.parametrize("window, sink", [(0, 0), (1600, 5), (50, 3)])      # (50: four wavefronts up to 128 elements, eight above)
def test_widths_types_and_windows(dtype, io, d, softcap, window, sink):
    pool = Pool(dtype, 2 if d == 64 else 1, d, 16 if d == 128 else 64, KV, layers=2, layer=1, seed=d)
    q, o = run(pool, io, CHUNKS, d, window, sink, softcap)
    ref, bound = exact(pool, q, CHUNKS, window, sink, softcap)
    assert_near(o, ref, bound, io)


@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [48, 64, 128, 256])
def test_missing_pages_and_stale_rows(dtype, io, d):
    pool = Pool(dtype, 1, d, 32, KV, seed=d)
    pool.table[0, 3] = -1
    pool.table[0, 77] = 10 ** 6                              # one of the chunk's own pages
    pool.table[1, :5] = -1
    pool.table_dev.copy_(pool.table)
    for window, sink in ((0, 0), (300, 100)):
        q, o = run(pool, io, CHUNKS, d, window, sink)
        ref, bound = exact(pool, q, CHUNKS, window, sink)
        assert_near(o, ref, bound, io)


@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("d", [48, 64, 128, 256])
def test_values_that_are_not_finite_reach_only_the_rows_that_see_them(dtype, io, d):
    bad = float("nan") if dtype == F8 else float("inf")
    for window in (0, 150):
        pool, clean = (Pool(dtype, 1, d, 16, [900], seed=d) for _ in range(2))
        odd, keys = [1, d // 2 + 3, d - 1], [640, 701, 702, 899]        # in the chunk of positions 600..899
        for at in keys:
            p, sl = int(pool.table[0, at // 16]), at % 16
            row = pool.v[0, p, 0, sl].float().clone()
            row[odd] = bad
            pool.v[0, p, 0, sl] = row.to(pool.v.dtype)
        o = [run(x, io, [300], d, window)[1] for x in (pool, clean)]
        pos = torch.arange(600, 900, device=DEV)
        sees = torch.zeros(300, dtype=torch.bool, device=DEV)
        for at in keys:
            sees |= (pos >= at) & ((pos - window < at) if window else True)
        want = torch.zeros_like(o[0], dtype=torch.bool)
        want[:, :, odd] = sees[:, None, None]
        assert torch.equal(~o[0].isfinite(), want) and torch.equal(o[0][~want], o[1][~want])
