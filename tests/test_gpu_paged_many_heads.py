"""Paged prefill with more workgroups than one dimension of a launch holds."""
import pytest
import torch

import vulkanforge_amd as vf
from paged_ref import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads, n", [(8192, 4096), (16384, 1500), (8192, 2047)])
def test_as_many_workgroups_as_tokens_and_heads_allow(heads, n):
    # n requests of one token behind one shared page: every output is the V row of its head
    d, page = 16, 16
    k, v = (torch.randn((1, 1, heads, page, d), generator=torch.Generator().manual_seed(i)).to(torch.float8_e4m3fn).to(DEV) for i in range(2))
    c = vf.PagedKvCache(vf.PagedKvConfig(1, heads, d, page, 1, vf.KvDtype.F8), k_buffer=k.data_ptr(), v_buffer=v.data_ptr())
    batch = vf.SeqBatch(torch.zeros((n, 1), dtype=torch.int32, device=DEV), torch.ones(n, dtype=torch.int32, device=DEV),
                        torch.arange(n + 1, dtype=torch.int32, device=DEV), n_tokens=n, max_kv_len=1)
    q = torch.ones((n, heads, d), dtype=torch.float16, device=DEV)
    o = torch.full_like(q, float("nan"))
    vf.PagedForward(c, heads).prefill_attention(0, batch, q, o)
    torch.cuda.synchronize()
    want = v[0, 0, :, 0].half()
    for at in range(0, n, 512):                          # (one weight: a power of two, and its own sum)
        assert torch.equal(o[at:at + 512], want.expand_as(o[at:at + 512]))
