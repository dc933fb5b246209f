"""ops.kv_append_paged at places outside the angles' tables: clamped into them, as
ops.qk_norm_rope does, for queries and keys alike."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("rows", [1, 30, 64])
def test_the_last_angles_are_taken(rows):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    cache = Cache([(9, 70), (3, 31), (5, 5)], 2, 64, 16, BF16)
    g = torch.Generator().manual_seed(rows)
    q, k = (torch.randn(17, h, 64, generator=g).to(BF16).cuda() for h in (4, 2))
    a = torch.rand(rows, 32, generator=g) * 6.28
    cos, sin = torch.cos(a).cuda(), torch.sin(a).cuda()
    (kp, vp, table, lens, cu), _ = cache.to_gpu()
    qo = ops.kv_append_paged(k, k, kp, vp, table, lens, cu, q=q, cos=cos, sin=sin)
    places = torch.cat([torch.arange(length - n, length) for n, length in cache.batch])
    pos = places.clamp(max=rows - 1).to(torch.int32)[None].cuda()
    qw, kw = ops.qk_norm_rope(q.transpose(0, 1)[None], k.transpose(0, 1)[None], cos, sin, pos)
    assert torch.equal(qo, qw[0].transpose(0, 1))
    page = cache.table[torch.tensor([0] * 9 + [1] * 3 + [2] * 5), places // 16].long()
    assert torch.equal(kp.cpu()[page, :, places % 16], kw[0].transpose(0, 1).cpu())
