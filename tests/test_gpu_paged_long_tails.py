"""One key that outweighs each of very many others: their sum counts, though each alone is below the last bit of the first."""
import math

import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import CACHE_TYPE, DEV, Pool

pytestmark = pytest.mark.gpu
F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8


def tail_pool(dtype, n, d, seed):
    """n keys, the first of them along e_0, the others zero; V -1 in the first row and about 1 in the others."""
    pool, page = Pool.__new__(Pool), 256
    g = torch.Generator().manual_seed(seed)
    pool.dtype, pool.hkv, pool.d, pool.page, pool.layer, pool.kv = dtype, 1, d, page, 0, [n]
    pool.table = torch.arange(-(-n // page), dtype=torch.int32)[None]
    pages = pool.table.shape[1]
    k, v = torch.zeros((1, pages, 1, page, d)), 1 + 0.25 * torch.randn((1, pages, 1, page, d), generator=g)
    k[0, 0, 0, 0, 0], v[0, 0, 0, 0] = 1.0, -1.0
    pool.k, pool.v = (x.to(CACHE_TYPE[dtype]).to(DEV) for x in (k, v))
    pool.cache = vf.PagedKvCache(vf.PagedKvConfig(1, 1, d, page, pages, dtype), k_buffer=pool.k.data_ptr(), v_buffer=pool.v.data_ptr())
    pool.table_dev, pool.kv_dev = pool.table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    return pool


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("n, tokens", [(65536, 512), (65536, 1), (2 ** 20, 3), (2 ** 20, 400)])
def test_a_long_tail_counts(dtype, io, n, tokens):
    """Weights 2^-20 to 2^-32 of the first one's; a chunk of many tokens is not split over the keys, so one wavefront sums them all."""
    pool = tail_pool(dtype, n, 64, n % 97)
    for drop in (20, 24, 28, 32):
        q = torch.zeros((tokens, 4, 64), device=DEV)
        q[..., 0] = drop * math.log(2.0)
        q = q.to(io)
        fwd = vf.PagedForward(pool.cache, 4)
        for decode in ((True, False) if tokens == 1 else (False,)):
            o = torch.full_like(q, float("nan"))
            batch = vf.SeqBatch(pool.table_dev, pool.kv_dev, None if decode else torch.tensor([0, tokens], dtype=torch.int32, device=DEV),
                                n_tokens=tokens, max_kv_len=0 if tokens < 4 else 1)
            (fwd.decode_attention if decode else fwd.prefill_attention)(0, batch, q, o, scale=1.0)
            torch.cuda.synchronize()
            some = sorted({0, tokens // 2, tokens - 1})
            for t in some:
                lens = [n - tokens + 1 + t]
                ref, bound = exact(pool, q[t:t + 1], [1], scale=1.0, lens=lens)
                assert_near(o[t:t + 1], ref, bound, io, (drop, t))
