"""GPU: what paged attention promises beyond its results — broken tables, padded batches, the bound of its error — against
64-bit restatements."""
import math

import pytest
import torch

from oracle import serving as oracle
from test_gpu_paged import _i32, _ops, make_cache, o_tolerance, to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new, ctx, Hq, Hkv", [(300, 300, 8, 2), (300, 900, 8, 2), (520, 520, 4, 2), (9, 300, 8, 2), (1, 300, 4, 4)])
@pytest.mark.parametrize("where", ["last", "middle"])
def test_rows_that_see_a_missing_page_are_nan(new, ctx, Hq, Hkv, where):
    """Of a sequence whose rows make several units of 256 those that see the page are NaN; the others are NaN or right, as
    is said of them; the other sequences are right."""
    D, page, dt, lens = 64, 16, torch.bfloat16, [ctx, 40]
    ops = _ops()
    k, v, table = make_cache(lens, Hkv, D, page, dt, "hnd", 5)
    q = torch.randn(new + 1, Hq, D, generator=torch.Generator().manual_seed(2)).to(dt)
    cu = [0, new, new + 1]
    o64, lse64 = oracle.paged_attention(q, k, v, table, lens, cu)
    bad_page = -(-ctx // page) - 1 if where == "last" else -(-ctx // page) // 2
    broken = table.clone()
    broken[0, bad_page] = k.shape[0] + 7
    o, lse = ops.paged_gqa_fwd(q.cuda(), to_gpu(k), to_gpu(v), broken.cuda(), _i32(lens).cuda(), cu_q=_i32(cu).cuda())
    assert ops.kernel_status() == 8 and ops.kernel_status() == 0
    o, lse = o.cpu(), lse.cpu()
    sees = torch.arange(ctx - new, ctx) >= bad_page * page
    assert torch.isnan(o[:new][sees]).all() and torch.isnan(lse[:new][sees]).all()
    big = v.double()[torch.isfinite(v)].abs().max()
    right = (o.double() - o64).abs() <= o_tolerance(o64, v, dt) + torch.finfo(dt).eps / 2 * big
    gone = torch.isnan(o)
    assert (gone[:new][~sees] | right[:new][~sees]).all() and right[new:].all() and torch.isfinite(lse[new:]).all()
    assert torch.equal(gone.all(2), gone.any(2)) and torch.equal(torch.isnan(lse), gone.all(2))      # a row is NaN as a whole
