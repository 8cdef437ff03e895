"""What the paged attention calls leave as their advisory."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_ref import DEV, Pool
from vulkanforge_amd import _ffi

pytestmark = pytest.mark.gpu
F32, F16 = vf.KvDtype.F32, vf.KvDtype.F16


def note(pool, decode=True, skew=0, n=1):
    d = pool.d
    buf = torch.zeros(n * 2 * d + 8, device=DEV)
    q, o = buf[skew:skew + n * 2 * d].view(n, 2, d), torch.zeros((n, 2, d), device=DEV)
    fwd = vf.PagedForward(pool.cache, 2)
    batch = vf.SeqBatch(pool.table_dev[:n], pool.kv_dev[:n]) if decode else pool.batch([n])
    (fwd.decode_attention if decode else fwd.prefill_attention)(0, batch, q, o)
    torch.cuda.synchronize()
    return _ffi.lib().vfkv_last_note()


@pytest.mark.parametrize("decode", [True, False])
def test_the_reason_is_named(decode):
    call = b"paged_decode_attention" if decode else b"paged_prefill_attention"
    for pool, skew, why in ((Pool(F16, 1, 72, 16, [20]), 0, b"multiple of 16"), (Pool(F32, 1, 512, 16, [20]), 0, b"wider than 256"),
                            (Pool(F16, 1, 64, 16, [20]), 1, b"16-byte aligned")):
        text = note(pool, decode, skew)
        assert text.startswith(call) and why in text and b"generic" in text and b"slab" not in text
    assert note(Pool(F16, 1, 64, 16, [20]), decode) == b""


def test_a_call_without_rows_leaves_none():
    pool = Pool(F16, 1, 72, 16, [20])
    assert note(pool) != b""
    assert note(pool, n=0) == b""
