"""ops.attention_paged over pages that several sequences share."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, check_attention

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _q(cache, Hq, dtype, seed=7):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(cache.tokens, Hq, cache.D, generator=g).to(dtype)


@pytest.mark.parametrize("D,qt,kt", [(128, BF16, BF16), (64, F16, F16), (128, BF16, FP8),
                                     (64, BF16, FP8)], ids=str)
@pytest.mark.parametrize("batch,shared", [
    ([(1, 700), (1, 900), (1, 650)], 640), ([(2, 2500), (40, 2222), (1, 2100)], 2048),
    ([(1, 3000)] * 20, 2944)], ids=["single", "mixed", "twenty"])
def test_pages_that_sequences_share(batch, shared, D, qt, kt):
    """A common prefix of `shared` tokens, its pages in every sequence's table."""
    cache = Cache(batch, 2, D, 32, kt, seed=D)
    cache.table[1:, :shared // 32] = cache.table[0, :shared // 32]
    q = _q(cache, 8, qt)
    args, scales = cache.to_gpu()
    o, lse = ops.attention_paged(q.cuda(), *args, max_seq_len=cache.max_len, return_lse=True,
                                 **scales)
    torch.cuda.synchronize()
    check_attention(cache, q, o.cpu(), lse.cpu())
