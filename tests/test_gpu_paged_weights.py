"""Attention weights over the paged cache: f16 rows give what the formula gives, rounded once at the output."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import DEV, Pool

pytestmark = pytest.mark.gpu
F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8


def outliers(pool, seed):
    """A tenth of V at -40 or 40: sums in which large terms cancel."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = pool.v.float()
    r = torch.rand(x.shape, generator=g, device=DEV)
    x = torch.where(r < 0.05, torch.full_like(x, -40.0), torch.where(r < 0.1, torch.full_like(x, 40.0), x))
    pool.v.copy_(torch.where(pool.v.float().isnan(), pool.v.float(), x).to(pool.v.dtype))


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("d, hq, hkv", [(64, 4, 2), (80, 2, 1), (128, 8, 2), (256, 4, 2), (512, 4, 2)])
@pytest.mark.parametrize("peaked", [False, True])
@pytest.mark.parametrize("window, sink, softcap", [(0, 0, 0.0), (50, 4, 0.0), (0, 0, 30.0)])
def test_f16_rows_round_only_at_the_output(dtype, d, hq, hkv, peaked, window, sink, softcap):
    kv, q_len = [300, 37, 700], [300, 5, 64]
    pool = Pool(dtype, hkv, d, 32, kv, seed=d)
    outliers(pool, d + 1)
    g = torch.Generator().manual_seed(d)
    for decode in (False, True):
        lens = [1] * 3 if decode else q_len
        n = sum(lens)
        q = (torch.randn((n, hq, d), generator=g) * (4.0 if peaked else 1.0)).half().to(DEV)
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, hq)
        (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q, o, window=window,
                                                                    n_sink=sink, softcap=softcap)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, lens, window, sink, softcap)
        assert_near(o, ref, bound, torch.float16, "decode" if decode else "prefill")


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("d, hq, hkv", [(64, 4, 1), (128, 8, 2), (256, 4, 2), (512, 4, 2), (40, 2, 1)])
@pytest.mark.parametrize("window, sink", [(0, 0), (3000, 70)])
def test_f16_rows_over_long_contexts(dtype, d, hq, hkv, window, sink):
    """Outputs of a few hundredths, where a key lost or counted twice is more than the bound of an element."""
    kv, q_len = [5000, 2049, 1], [7, 40, 1]
    pool = Pool(dtype, hkv, d, 64, kv, seed=d)
    g = torch.Generator().manual_seed(d)
    for decode in (False, True):
        lens = [1] * 3 if decode else q_len
        q = torch.randn((sum(lens), hq, d), generator=g).half().to(DEV)
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, hq)
        (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q, o, window=window, n_sink=sink)
        torch.cuda.synchronize()
        ref, bound = exact(pool, q, lens, window, sink)
        assert_near(o, ref, bound, torch.float16, "decode" if decode else "prefill")
