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


def _device_meta(t):
    """What a plan knows of such a tensor on a GPU."""
    return t.shape, t.stride(), t.dtype, torch.device("cuda", 0)


@pytest.mark.parametrize("at", ["q", "k", "v", "out"])
def test_expanded_rows_are_refused_by_attention(at):
    """All strides zero would read as contiguous, far past the row."""
    shapes = dict(q=(2, 8, 5, 128), k=(2, 2, 9, 128), v=(2, 2, 9, 128), out=(2, 8, 5, 128))
    tensors = {n: _device_meta(_row(*s) if n == at else meta(*s)) for n, s in shapes.items()}
    with pytest.raises(ValueError, match="one row expanded"):
        ops._attn_plan(*tensors.values(), None, False, None, None, 0, 0)


def test_a_single_row_may_have_any_strides():
    """Where no step is taken, strides of zero mean nothing."""
    row = _device_meta(_row(1, 1, 1, 128))
    desc, _, shape = ops._attn_plan(row, row, row, None, None, False, None, None, 0, 0)
    assert shape == (1, 1, 1)


def test_a_workspace_is_for_its_own_sizes():
    """Cutting keys needs room where tiles are few; one sequence of many is not cut."""
    few, many = (ops.attention_paged_workspace_bytes(n, 1, 32, 8, 128, 100000)
                 for n in (4000, 40000))
    assert few > 0 and many == 0
