"""CPU tests of attention_paged's caps and windows that the library's own types do not
hold: refused, or what they stand for."""

import pytest
import torch

from neptune_hip import ops
from test_mx_validation import _attend, _pools, meta


@pytest.mark.parametrize("softcap", [1e-50, 1e-46, 5e-324])
def test_a_cap_that_is_no_float(softcap):
    """A positive cap that fp32 has as 0, which means none to the library, is refused as
    other caps below 2^-60 are."""
    with pytest.raises(ValueError, match="softcap"):
        _attend(softcap=softcap)


def _score(monkeypatch, **kw):
    """The scores' descriptor that a call hands to the library."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *a: None)
    p = {k: ops._meta(v) for k, v in _pools().items()}
    args = dict(softcap=None, slopes=None, window=None, max_seq_len=512, scale=None, out=None)
    args.update(kw)
    ext = ops._attn_paged_plan(
        ops._meta(meta(10, 8, 128)), p["k_pages"], p["v_pages"], p["block_table"], p["seq_lens"],
        p["cu_seqlens"], p["k_scales"], p["v_scales"], args["out"], args["max_seq_len"],
        args["scale"], args["softcap"], args["slopes"], args["window"])[3]
    return ext[1]._obj


def test_ordinary_scores(monkeypatch):
    s = _score(monkeypatch, softcap=30.0, window=7)
    assert s.softcap == 30.0 and s.window == 7
    assert _score(monkeypatch, softcap=1e-30).softcap == torch.tensor(1e-30).item()
    assert _score(monkeypatch, softcap=30.0).window == 0


@pytest.mark.parametrize("window", [2**63 - 1, 2**63, 2**64, 2**64 + 5, 10**30])
def test_a_window_past_64_bits_hides_nothing(monkeypatch, window):
    assert _score(monkeypatch, window=window).window >= 512
