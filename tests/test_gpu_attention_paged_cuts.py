"""ops.attention_paged: that keys are cut where the cases mean it, and their states
combined, by eight groups of lanes and by one.

A launch that cuts keys leaves its states in the workspace and only the combine
writes those tiles' outputs; one that cuts none does not touch it. (The plan's side,
on the CPU: test_attn_plan.py.)"""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, check_attention

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn

CUTS = [
    # (batch, Hq, Hk, D, page, q's type, pools' type, whether keys are cut, combine's groups)
    ([(1, 5000)], 8, 2, 128, 64, BF16, BF16, True, 8),
    ([(1, 20000)], 32, 8, 128, 64, BF16, BF16, True, 8),  # more splits than groups
    ([(3, 2900)], 8, 1, 64, 16, F16, F16, True, 8),
    ([(1, 9000), (1, 4000)], 8, 2, 128, 16, BF16, FP8, True, 8),
    ([(2, 3001), (1, 70)], 6, 2, 64, 64, BF16, FP8, True, 8),
    ([(40, 3333)], 12, 4, 128, 64, BF16, BF16, True, 8),  # two wide tiles of few heads
    ([(40, 3333), (150, 1500)], 8, 2, 128, 64, BF16, BF16, True, 1),
    ([(40, 3333), (150, 1500)], 8, 2, 128, 48, BF16, FP8, True, 1),
    ([(130, 1500), (1, 1), (0, 300), (77, 900)], 16, 4, 64, 48, F16, F16, True, 1),
    ([(90, 2000), (33, 700)], 8, 2, 64, 16, BF16, FP8, True, 1),
    ([(5, 4000)] * 16, 8, 2, 128, 64, BF16, BF16, True, 1),
    # room for states, but work-groups enough without
    ([(1, 500)] * 600, 8, 1, 64, 16, BF16, BF16, False, 1),
    ([(1400, 1400)] * 2, 24, 6, 64, 64, F16, F16, False, 1),
]


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _q(cache, Hq, dtype, seed=7):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(cache.tokens, Hq, cache.D, generator=g).to(dtype)


@pytest.mark.parametrize("batch,Hq,Hk,D,page,qt,kt,cut,groups", CUTS, ids=lambda x: str(x)[:24])
def test_cut_keys_leave_states(batch, Hq, Hk, D, page, qt, kt, cut, groups):
    cache = Cache(batch, Hk, D, page, kt, seed=D + page)
    q = _q(cache, Hq, qt)
    args, scales = cache.to_gpu()
    need = ops.attention_paged_workspace_bytes(cache.tokens, len(batch), Hq, Hk, D, cache.max_len,
                                               dtype=qt, fp8=kt == FP8)
    assert need > 0
    ws = torch.full((need,), 0x5a, dtype=torch.uint8, device="cuda")
    o, lse = ops.attention_paged(q.cuda(), *args, max_seq_len=cache.max_len, return_lse=True,
                                 workspace=ws, **scales)
    torch.cuda.synchronize()
    assert bool((ws != 0x5a).any()) == cut
    check_attention(cache, q, o.cpu(), lse.cpu())
