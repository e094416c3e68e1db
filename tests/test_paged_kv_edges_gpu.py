"""The paged key/value cache at the edges of its contract."""
import pytest
import torch

import cutilegpt_b200 as cg
from cutilegpt_b200 import _lib as L
from test_paged_kv_gpu import BF, F32, make

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append past a table
@pytest.mark.parametrize("dtype,D,rot", [(BF, 64, 0), (BF, 64, 64), (F32, 64, 32), (BF, 7, 4), (F32, 7, 0)])
@pytest.mark.parametrize("T,past", [(1, 1), (5, 2), (5, 5), (5, 100), (3, 2 ** 31 - 1 - 48)])
def test_append_past_the_table(dtype, D, rot, T, past):
    """Tokens that fit go to their own positions, the others nowhere; no earlier position changes."""
    page, cap = 16, 48
    kv, _ = make(dtype, 2, 1, T, 4, 2, D, page, [20], [cap - 17, cap - 17], garbage=False)
    assert kv.page_table.shape[1] * page == cap
    kv.seq_lens.copy_(torch.tensor([cap + past, 30]))
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, h, T, D, generator=g).to(dtype).cuda() for h in (4, 2, 2))
    table = torch.randn(20 + cap + 8, rot, generator=g).cuda() if rot else None
    before = kv.k_pages.clone(), kv.v_pages.clone()
    L.device_error()
    got = cg.cutile_paged_kv_append(q, k, v, kv, table)
    with pytest.raises(L.GptError):
        L.device_error()
    after = kv.k_pages.clone(), kv.v_pages.clone()
    # the same with one call for each token that has a place
    kv.k_pages.copy_(before[0])
    kv.v_pages.copy_(before[1])
    want = torch.zeros_like(q) if rot else q
    for b, n in enumerate((cap + past, 30)):
        for t in range(T):
            i = n - T + t
            if i >= cap:
                continue
            one = cg.PagedKV(kv.k_pages, kv.v_pages, kv.page_table[b:b + 1], torch.tensor([i + 1], dtype=torch.int32).cuda(),
                             kv.prefix_table, kv.prefix_lens)
            x = cg.cutile_paged_kv_append(q[b:b + 1, :, t:t + 1], k[b:b + 1, :, t:t + 1], v[b:b + 1, :, t:t + 1], one, table)
            if rot:
                want[b, :, t] = x[0, :, 0]
    assert L.device_error() == 0
    assert torch.equal(after[0], kv.k_pages) and torch.equal(after[1], kv.v_pages)
    assert torch.equal(got, want)
