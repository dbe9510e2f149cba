"""Calls of the paged-cache operators next to their limits: values, sinks and sizes that
ordinary batches do not have. Tolerances as in test_paged_gpu.py."""
import pytest
import torch

from oracle import paged as OP
from test_paged_gpu import E4M3, check_attention, make_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# a NaN code of e4m3 under a finite scale
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,widen", [(1, False), (12, False), (40, False), (300, True)])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_nan_code_of_e4m3_is_nan_in_every_form(cuda_device, D, n, widen, code):
    """A pool may hold e4m3's NaN in a row with an ordinary scale byte (torch's cast
    makes it). Position 0, which every row sees: a NaN in the value row is a NaN in that
    column of every row, one in the key row makes the rows of its head NaN."""
    import d2sd_b200 as d
    Hq, Hk, kl = 8, 2, 400
    g = torch.Generator().manual_seed(90 + n)
    c = make_cache(g, [kl], Hk, D, E4M3, "paged_umma", cuda_device)
    q = torch.randn(n, Hq, D, generator=g).to(torch.bfloat16).to(cuda_device)
    plan = d.PagedAttentionPlan([n], [kl], Hq, Hk, D, cuda_device, cache_dtype=E4M3)
    assert plan.widen == widen
    col = D - 3
    run = lambda c: d.paged_attention(q, c["k"], c["v"], "paged_umma", c["table"], plan,  # noqa: E731
                                      k_scale=c["ks"], v_scale=c["vs"])[0]

    def planted(pool):  # position 0 of kv head 1
        x = pool.clone()
        page = int(c["table"][0])
        x.view(torch.uint8)[page, 1].flatten()[OP.page_index("paged_umma", D, 1)[0, col]] = code
        return x
    base = run(c)
    out = run(dict(c, v=planted(c["v"])))
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[:, Hq // 2:, col] = True
    assert torch.equal(out.isnan(), nan)
    assert torch.equal(out[~nan], base[~nan])
    out = run(dict(c, k=planted(c["k"])))
    assert out[:, Hq // 2:].isnan().all() and torch.equal(out[:, :Hq // 2], base[:, :Hq // 2])
