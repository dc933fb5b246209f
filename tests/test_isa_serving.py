"""Register budgets and wait order of the paged attention's and the rotation's
compiled code."""

import re
import subprocess

import pytest

from test_isa_hazards import CSRC, HIPCC, _build_flags, kernel_resources


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("isa")
    out = {}
    for name in ("attn_paged", "rope"):
        s = tmp / f"{name}.s"
        subprocess.run([HIPCC, *_build_flags(), "--cuda-device-only", "-S", "-o", str(s),
                        str(CSRC / f"{name}.hip")], check=True, stderr=subprocess.DEVNULL)
        out[name] = s.read_text()
    return out


@pytest.mark.parametrize("name,pattern,limit,why", [
    ("attn_paged", r"10attn_paged", 256, "two waves per SIMD"),
    ("attn_paged", r"attn_paged_combine", 64, "eight waves per SIMD"),
    ("rope", r"norm_rope.*Li1EEEv", 64, "eight waves per SIMD"),
    ("rope", r"norm_rope.*Li4EEEv", 96, "five waves per SIMD"),
])
def test_budgets(asm, name, pattern, limit, why):
    hits = {k: v for k, v in kernel_resources(asm[name]).items() if re.search(pattern, k)}
    assert hits, "the check is looking at the wrong code"
    for kernel, (vgpr, scratch) in hits.items():
        assert vgpr <= limit and not scratch, (kernel, vgpr, scratch, why)


def test_no_packed_fp32(asm):
    for text in asm.values():
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
