"""Attention over F32 pages with elements of V up to the bound that the header names, 2^110, under any number of keys."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import DEV, Pool

pytestmark = pytest.mark.gpu
F32 = vf.KvDtype.F32


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256, 40])
@pytest.mark.parametrize("kv", [[17, 300], [5000, 40], [200000]])
def test_v_up_to_2_to_the_110(d, kv, decode):
    """The first key scores 7.9 (log2 units) below the others, so that these come close to the largest weight that the running
    maximum is not raised for; all of V has one sign."""
    pool = Pool(F32, 1, d, 64, kv)
    k = torch.zeros_like(pool.k)
    k[..., 0] = 1.0
    for s in range(len(kv)):
        k[0, int(pool.table[s, 0]), 0, 0, 0] = 0.0
    pool.k.copy_(torch.where(pool.k.isnan(), pool.k, k))
    pool.v.copy_(torch.where(pool.v.isnan(), pool.v, (1.0 - pool.v.abs() / 8).clamp(0.1, 0.999) * 2.0 ** 110))
    lens = [1] * len(kv) if decode else [min(x, 3) for x in kv]
    n = sum(lens)
    q = torch.zeros((n, 2, d), device=DEV)
    q[..., 0] = 7.9 / 1.44269504
    o = torch.full_like(q, float("nan"))
    fwd = vf.PagedForward(pool.cache, 2)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q, o, scale=1.0)
    torch.cuda.synchronize()
    ref, bound = exact(pool, q, lens, scale=1.0)
    assert_near(o, ref, bound, torch.float32)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256, 40])
def test_small_values_keep_their_accuracy(d, decode):
    pool = Pool(F32, 1, d, 16, [90, 3])
    pool.v.mul_(2.0 ** -95)
    lens = [1, 1] if decode else [50, 3]
    q = torch.randn((sum(lens), 2, d), generator=torch.Generator().manual_seed(d)).to(DEV)
    o = torch.full_like(q, float("nan"))
    fwd = vf.PagedForward(pool.cache, 2)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q, o)
    torch.cuda.synchronize()
    ref, bound = exact(pool, q, lens)
    assert_near(o * 2.0 ** 95, ref * 2.0 ** 95, bound * 2.0 ** 95, torch.float32)
