"""Norm + rotation + append of so many tokens that a wavefront takes several steps of rows: the steps requested ahead, those that
cross from query to key to value rows, the ones past the last, and queries rotated in place while later rows are on their way."""
import math

import pytest
import torch

import vulkanforge_amd as vf
from paged_ref import CACHE_TYPE, DEV, Pool, turned

pytestmark = pytest.mark.gpu
F32, F16, F8 = vf.KvDtype.F32, vf.KvDtype.F16, vf.KvDtype.F8
U = 2.0 ** -24


def steps_per_wavefront(n, hq, hkv, d):
    rows = 64 // (8 if d <= 64 else 16 if d <= 128 else 32 if d <= 256 else 64)       # rows per step
    steps = -(-hq // rows) + 2 * -(-hkv // rows)
    return -(-steps // min(-(-4096 // n), steps))


def check(dtype, io, hq, hkv, d, n, rot, mode=vf.ROPE_NEOX, in_place=False, strided=False, no_q=False, n_pad=0, norm=True, page=64):
    q_len = [n // 2 - 3, 0, n - n // 2, 3]
    kv = [q_len[0] + 11, 5, q_len[2], 40]
    pool = Pool(dtype, hkv, d, page, kv, layers=2, layer=1, seed=d)
    g = torch.Generator().manual_seed(n)
    total = n + n_pad
    if strided:
        packed = torch.randn((total, hq + 2 * hkv, d), generator=g).to(io).to(DEV)
        q, k, v = packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]
    else:
        q, k, v = (torch.randn((total, h, d), generator=g).to(io).to(DEV) for h in (hq, hkv, hkv))
    q0, k0, v0 = (x.clone() for x in (q, k, v))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(DEV) if norm else None for _ in range(2))
    sections = [rot // 2 - 2 * (rot // 6), rot // 6, rot // 6]
    pos = torch.randint(0, 200_000, (3, total), generator=g, dtype=torch.int32)
    out = q if in_place else torch.full_like(q0, 9.0)
    before = [x.clone() for x in (pool.k, pool.v)]
    fwd = vf.PagedForward(pool.cache, hq)
    fwd.qk_rope_kv_write(1, pool.batch(q_len, n_tokens=total), None if no_q else q, k, v, vf.MRope(rot, 1e6, sections, True, mode),
                         q_out=None if in_place or no_q else out, q_norm_weight=wq, k_norm_weight=wk, positions=pos.to(DEV))
    torch.cuda.synchronize()
    # per element, as in test_gpu_paged.py: norm (d / 64 + 16 half steps), two products and a sum (4), cos and sin (4 + 7)
    rel = (d / 64 + 16 + 4 + 11) * U

    def near(x, ref, half, lowest, what):
        size = ref.abs().amax(-1, keepdim=True) * math.sqrt(2)
        err = (x.float().cpu().double() - ref).abs()
        assert bool((err <= size * rel + ref.abs() * half + lowest).all()), (what, err.max())

    if no_q:
        assert bool((out == 9.0).all()) and torch.equal(q, q0)
    else:
        near(out[:n], turned(q0[:n], wq, pos[:, :n], 1e6, rot, sections, True, mode), 2.0 ** -11 if io is torch.float16 else U, 2.0 ** -25, "q")
        assert torch.equal(out[n:], (q0 if in_place else torch.full_like(q0, 9.0))[n:])
    if not in_place:
        assert torch.equal(q, q0)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    rk = turned(k0[:n], wk, pos[:, :n], 1e6, rot, sections, True, mode)
    vv = v0[:n].float()
    if dtype == F8:
        rk, vv = rk.clamp(-448, 448), vv.clamp(-448, 448)
    half = {F8: 2.0 ** -4, F16: 2.0 ** -11, F32: U}[dtype]
    written = torch.zeros(pool.k.shape[1], page, dtype=torch.bool)
    at = 0
    for s, (m, b) in enumerate(zip(q_len, kv)):
        j = torch.arange(b - m, b)
        p, sl = pool.table[s].long()[j // page], j % page
        near(pool.k[1].cpu()[p, :, sl], rk[at:at + m], half, 2.0 ** -10 if dtype == F8 else 2.0 ** -25, ("k", s))
        assert torch.equal(pool.v[1].cpu()[p, :, sl].view(torch.uint8), vv[at:at + m].to(CACHE_TYPE[dtype]).cpu().view(torch.uint8))
        written[p, sl] = True
        at += m
    for x, y in ((pool.k, before[0]), (pool.v, before[1])):
        a, b = (t.cpu().view(torch.uint8).reshape(*t.shape[:4], -1).transpose(2, 3) for t in (x, y))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1][~written], b[1][~written])


@pytest.mark.parametrize("n, steps", [(700, 2), (1500, 4), (2100, 6), (4200, 12)])
@pytest.mark.parametrize("io", [torch.float32, torch.float16])
@pytest.mark.parametrize("dtype", [F16, F8])
def test_several_steps(n, steps, io, dtype):
    assert steps_per_wavefront(n, 32, 8, 128) == steps
    check(dtype, io, 32, 8, 128, n, 128)


@pytest.mark.parametrize("d, hq, hkv, rot, n, steps", [(64, 32, 8, 64, 1500, 2), (64, 28, 4, 32, 4200, 6), (256, 16, 4, 256, 1500, 4), (256, 7, 1, 128, 4200, 6),
                                                       (512, 8, 2, 128, 1500, 4), (512, 5, 1, 512, 4200, 7), (128, 6, 3, 128, 4200, 4), (80, 10, 5, 80, 2100, 4),
                                                       (96, 13, 1, 48, 4200, 6), (8, 9, 3, 8, 4200, 4), (200, 6, 2, 96, 4200, 5)])
@pytest.mark.parametrize("mode", [vf.ROPE_NEOX, vf.ROPE_NORM])
def test_several_steps_of_other_widths(d, hq, hkv, rot, n, steps, mode):
    assert steps_per_wavefront(n, hq, hkv, d) == steps
    check(F16, torch.float32, hq, hkv, d, n, rot, mode)
    check(F8, torch.float16, hq, hkv, d, n, rot, mode, norm=False)


@pytest.mark.parametrize("kw", [dict(in_place=True), dict(strided=True), dict(in_place=True, strided=True), dict(no_q=True), dict(n_pad=9),
                                dict(in_place=True, n_pad=70), dict(page=16)])
@pytest.mark.parametrize("n", [700, 4200])
def test_several_steps_options(kw, n):
    check(F16, torch.float16, 32, 8, 128, n, 128, **kw)
    check(F32, torch.float32, 14, 2, 64, n, 64, vf.ROPE_NORM, **kw)
