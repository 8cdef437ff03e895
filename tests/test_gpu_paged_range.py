"""Attention over pages at scores of any size that an f32 holds: far below, far above, and both among ordinary rows."""
import math

import pytest
import torch

import vulkanforge_amd as vf
from paged_exact import assert_near, exact
from paged_ref import DEV, Pool

pytestmark = pytest.mark.gpu
F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8
SIZES = [0.0, 1.0, -3.0, 1e4, -1e4, 3e6, -3e6, 1e8, -1e8, 2e8, 7e8, -7e8, 1e9, -1e9, 3e12, -3e12, 1e20, -1e20, 5e29, -5e29, 2e30, -2e30,
         4e33, -4e33, 1e36, -1e36]


def one_axis(pool, seed):
    """K rows c e_0 with c of -1, 1 or 2: the score of a key is c q_0 scale without an error, and equal keys have equal ones."""
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(pool.k.shape)
    k[..., 0] = torch.tensor([-1.0, 1.0, 2.0])[torch.randint(0, 3, pool.k.shape[:-1], generator=g)]
    pool.k.copy_(torch.where(pool.k.float().cpu().isnan(), torch.tensor(float("nan")), k).to(pool.k.dtype))


def check(pool, hq, lens, decode, io, window=0, sink=0, softcap=0.0, first=0):
    n = sum(lens)
    scale = 1.0 if io is torch.float32 else (1.0, 1e4, 1e30)[first % 3]
    s = torch.tensor(SIZES, dtype=torch.float64)[(torch.arange(n * hq) * 7 + first) % len(SIZES)].view(n, hq)
    if io is torch.float16:
        s = s.clamp(-6e4 * scale, 6e4 * scale)
    q = torch.zeros(n, hq, pool.d, dtype=torch.float64)
    q[..., 0] = s / scale
    q[..., 1:] = torch.randn(q[..., 1:].shape, generator=torch.Generator().manual_seed(3)) * (0.2 * s.abs() / scale)[..., None]   # (meets zeros)
    q = q.to(io).to(DEV)
    o = torch.full_like(q, float("nan"))
    fwd = vf.PagedForward(pool.cache, hq)
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q, o, window=window, n_sink=sink,
                                                                scale=scale, softcap=softcap)
    torch.cuda.synchronize()
    # a score of an ordinary row (at most 6) is off by 6 (2^-23 + 3 * 2^-24), a weight by twice that, 60 half steps: less than what the
    # sums may be off, at least 88
    q2 = q.clone()
    q2[..., 1:] = 0
    ref, bound = exact(pool, q2, lens, window, sink, softcap, scale=scale, score_error=False)
    assert_near(o, ref, bound * 2, io, f"{'decode' if decode else 'prefill'} {window}")


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("d", [64, 96, 128, 256, 512, 40])
def test_scores_of_any_size(dtype, io, decode, d):
    pool = Pool(dtype, 2, d, 16, [1, 2, 33, 200, 70], seed=d)
    one_axis(pool, d)
    lens = [1] * 5 if decode else [1, 2, 20, 130, 3]
    for first in range(0, len(SIZES), 5):
        check(pool, 8, lens, decode, io, first=first)
    check(pool, 8, lens, decode, io, window=20, sink=3)


@pytest.mark.parametrize("dtype", [F32, F16, F8])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_scores_of_any_size_in_parts_that_are_joined(dtype, decode, d):
    pool = Pool(dtype, 1, d, 64, [5000, 40])
    one_axis(pool, d)
    for first in range(0, len(SIZES), 2 if decode else 9):
        check(pool, 4, [1, 1] if decode else [7, 3], decode, torch.float32, first=first)


@pytest.mark.parametrize("dtype", [F16, F8])
def test_scores_of_any_size_in_blocks_of_256_rows(dtype):
    for d, io in ((64, torch.float32), (128, torch.float16), (256, torch.float16)):
        pool = Pool(dtype, 1, d, 64, [1400])
        one_axis(pool, d)
        check(pool, 4, [600], False, io)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("d", [128, 40, 512])
def test_only_keys_far_below_zero(decode, d):
    """One visible key gives its V row and equal keys their mean, however low the score."""
    for dtype in (F32, F16, F8):
        pool = Pool(dtype, 1, d, 16, [1, 48])
        pool.k.copy_(torch.where(pool.k.float().isnan(), float("nan"), 1.0).to(pool.k.dtype))
        n = [1, 1]
        for size in (1e28, 2e30, 1e33, 1e35):
            q = torch.full((2, 2, d), -size / d, device=DEV)
            o = torch.zeros_like(q)
            fwd = vf.PagedForward(pool.cache, 2)
            (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else n), q, o, scale=1.0)
            torch.cuda.synchronize()
            for s, kv in enumerate(pool.kv):
                mean = pool.rows(pool.v, s).mean(0).expand(2, d)
                assert (o[s].cpu().double() - mean).abs().max() <= 4.0 * (kv / 16 + 72) * 2.0 ** -24 * (1 + math.log2(kv)), (dtype, size)


@pytest.mark.parametrize("dtype", [F16, F8])
@pytest.mark.parametrize("decode", [True, False])
def test_rows_far_out_leave_the_ordinary_ones_alone(dtype, decode):
    """Every other head with scores beyond 2^30: the heads between them give what they give without, to the steps of their weights (the
    running maximum is raised for all rows of a wavefront at once): two weights of 22 bits times elements below 5 that sum to 1."""
    pool = Pool(dtype, 1, 128, 32, [500, 90])
    lens = [1, 1] if decode else [60, 9]
    q = torch.randn((sum(lens), 4, 128), generator=torch.Generator().manual_seed(2)).to(DEV)
    outs = []
    for by in (1.0, 2.0 ** 31):
        q2 = q.clone()
        q2[:, 1::2] *= by
        o = torch.full_like(q, float("nan"))
        fwd = vf.PagedForward(pool.cache, 4)
        (fwd.decode_attention if decode else fwd.prefill_attention)(0, pool.batch(None if decode else lens), q2, o)
        torch.cuda.synchronize()
        assert bool(o.isfinite().all())
        outs.append(o[:, ::2])
    assert (outs[0] - outs[1]).abs().max() <= 2 * 5 * 2.0 ** -22
