"""CPU tests of the torch front's refusals that its operators share: one row expanded
to a tensor, and pairs of outputs that are not both given."""

import pytest
import torch

from neptune_hip import ops

bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32


def meta(*shape, dtype=bf16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _row(*shape):
    return meta(shape[-1]).expand(*shape)


@pytest.mark.parametrize("out", [(meta(2, 8, 5, 128), None), (None, meta(2, 2, 5, 128)),
                                 (None, None), (meta(2, 8, 5, 128),), meta(2, 8, 5, 128),
                                 (meta(2, 8, 5, 128), meta(2, 2, 5, 128), None)],
                         ids=["no_k", "no_q", "neither", "one", "a_tensor", "three"])
def test_rope_takes_both_outputs_or_none(out):
    with pytest.raises(ValueError, match="q_out, k_out"):
        ops.qk_norm_rope(meta(2, 8, 5, 128), meta(2, 2, 5, 128), meta(100, 64, dtype=f32),
                         meta(100, 64, dtype=f32), meta(2, 5, dtype=i32), out=out)
