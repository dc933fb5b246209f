"""Register budgets of the kernels over MXFP4 pools, of shaped scores and of the cache's
reading."""

import re
import subprocess

import pytest

from test_isa_hazards import CSRC, HIPCC, _build_flags, kernel_resources


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("isa")
    out = {}
    for name in ("attn_paged_mx", "attn_paged_shaped", "rope", "kv_read"):
        s = tmp / f"{name}.s"
        subprocess.run([HIPCC, *_build_flags(), "--cuda-device-only", "-S", "-o", str(s),
                        str(CSRC / f"{name}.hip")], check=True, stderr=subprocess.DEVNULL)
        out[name] = s.read_text()
    return out


@pytest.mark.parametrize("name,pattern,limit,why", [
    ("attn_paged_mx", r"10attn_paged", 256, "two waves per SIMD"),
    ("attn_paged_shaped", r"10attn_paged", 256, "two waves per SIMD"),
    ("rope", r"append_mx", 128, "four waves per SIMD"),
    ("kv_read", r"kv_read", 64, "eight waves per SIMD"),
])
def test_budgets(asm, name, pattern, limit, why):
    hits = {k: v for k, v in kernel_resources(asm[name]).items() if re.search(pattern, k)}
    assert hits, "the check is looking at the wrong code"
    for kernel, (vgpr, scratch) in hits.items():
        assert vgpr <= limit and not scratch, (kernel, vgpr, scratch, why)


def test_no_packed_fp32(asm):
    for text in asm.values():
        assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
