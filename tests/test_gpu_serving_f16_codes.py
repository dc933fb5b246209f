"""A float16 model over an E4M3 cache: its keys and values appended as codes, its
rotated queries cast to bfloat16 for attention_paged, its outputs back."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, check_attention

pytestmark = pytest.mark.gpu

F16, BF16, FP8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
def test_codes_of_float16_values_are_read(D, page):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    cache = Cache([(40, 40), (300, 300), (1, 1)], 2, D, page, FP8, seed=D)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(341, h, D, generator=g).to(F16).cuda() for h in (8, 2, 2))
    a = torch.rand(300, D // 2, generator=g) * 6.28
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    qr = ops.kv_append_paged(k, v, kp, vp, table, lens, cu, q=q, cos=torch.cos(a).cuda(),
                             sin=torch.sin(a).cuda(), **scales)
    cache.k, cache.v = kp.cpu(), vp.cpu()
    for b, (n, _) in enumerate(cache.batch):
        rows = slice(int(cache.cu[b]), int(cache.cu[b + 1]))
        scale = cache.v_scales[cache.table[b, torch.arange(n) // page].long()].double()[..., None]
        # a code holds at most 448 times its scale, the nearest value below that: half a
        # step, 2^-4 of it, or 2^-10 of the scale below the normal codes; 2^-22 for fp32
        want = torch.maximum(torch.minimum(v[rows].cpu().double(), 448 * scale), -448 * scale)
        got = cache.values(b, "v").permute(1, 0, 2)
        bound = torch.maximum(2.0**-4 * want.abs(), 2.0**-10 * scale) * (1 + 2.0**-22)
        assert ((got - want).abs() <= bound).all()
    qb = qr.to(BF16)
    o, lse = ops.attention_paged(qb, kp, vp, table, lens, cu, return_lse=True, max_seq_len=300,
                                 **scales)
    check_attention(cache, qb.cpu(), o.cpu(), lse.cpu())
    assert torch.isfinite(o.to(F16)).all()
