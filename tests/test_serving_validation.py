"""CPU tests of qk_norm_rope, kv_append_paged and attention_paged: argument
checks of the torch front (meta tensors, no GPU) and of the C-ABI, whose
refusals come before any HIP call, and the layout of their descriptors."""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from neptune_hip import _abi, ops

ROOT = Path(__file__).resolve().parents[1]
bf16, f16, f32, u8, i32 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int32
INVALID, UNSUPPORTED, SMALL, NO_DEVICE = (_abi.ERR_INVALID_ARGUMENT, _abi.ERR_UNSUPPORTED,
                                          _abi.ERR_WORKSPACE_TOO_SMALL, _abi.ERR_NO_DEVICE)


def meta(*shape, dtype=bf16):
    return torch.empty(shape, dtype=dtype, device="meta")


# ---- torch front ---------------------------------------------------------

def _rope(**kw):
    a = dict(q=meta(2, 8, 5, 128), k=meta(2, 2, 5, 128), cos=meta(100, 64, dtype=f32),
             sin=meta(100, 64, dtype=f32), positions=meta(2, 5, dtype=i32))
    a.update(kw)
    return ops.qk_norm_rope(**a)


@pytest.mark.parametrize("kw,match", [
    ({}, "device tensors"),
    (dict(q=meta(2, 5, 8, 128).transpose(1, 2), q_weight=meta(128, dtype=f32)), "device tensors"),
    (dict(out=(meta(2, 8, 5, 128), meta(2, 2, 5, 128))), "device tensors"),
    (dict(q=meta(8, 5, 128)), "batch, heads, seq"),
    (dict(q=meta(2, 8, 128, 5).transpose(2, 3)), "unit head_dim"),
    (dict(k=meta(2, 2, 6, 128)), "shape mismatch"),
    (dict(k=meta(2, 2, 5, 128, dtype=f16)), "share one"),
    (dict(q=meta(2, 8, 5, 128, dtype=u8), k=meta(2, 2, 5, 128, dtype=u8)), "share one"),
    (dict(cos=None, sin=None), "cos and sin"),
    (dict(sin=None), "together"),
    (dict(cos=meta(100, 64)), "float32"),
    (dict(cos=meta(64, 100, dtype=f32).t()), "contiguous"),
    (dict(sin=meta(99, 64, dtype=f32)), "match"),
    (dict(q_weight=meta(64, dtype=f32)), "q_weight"),
    (dict(k_weight=meta(128)), "k_weight"),
    (dict(positions=meta(2, 5, dtype=torch.int64)), "positions"),
    (dict(positions=meta(5, dtype=i32)), "positions"),
    (dict(out=(meta(2, 8, 5, 128), meta(2, 2, 5, 128, dtype=f16))), "match k's"),
])
def test_rope_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _rope(**kw)


def _cache(kv=bf16, layout="head", D=128, page=64):
    shape = (20, 2, page, D) if layout == "head" else (20, page, 2, D)
    pools = [meta(*shape, dtype=kv) for _ in range(2)]
    if layout == "token":
        pools = [p.permute(0, 2, 1, 3) for p in pools]
    scales = {} if kv in (bf16, f16) else {
        "k_scales": meta(20, 2, dtype=f32), "v_scales": meta(20, 2, dtype=f32)}
    return dict(k_pages=pools[0], v_pages=pools[1], block_table=meta(3, 8, dtype=i32),
                seq_lens=meta(3, dtype=i32), cu_seqlens=meta(4, dtype=i32), **scales)


def _append(**kw):
    a = dict(k=meta(10, 2, 128), v=meta(10, 2, 128), q=meta(10, 8, 128), **_cache())
    a.update(kw)
    return ops.kv_append_paged(**a)


def _attend(**kw):
    a = dict(q=meta(10, 8, 128), **_cache())
    a.update(kw)
    return ops.attention_paged(**a)


POOL_CASES = [
    (_cache(layout="token"), "device tensors"),
    (_cache(kv=u8), "device tensors"),
    (_cache(kv=torch.float8_e4m3fn), "device tensors"),
    (dict(k_pages=meta(20, 2, 64, 128, dtype=f16), v_pages=meta(20, 2, 64, 128, dtype=f16)),
     "pools must be"),
    (dict(v_pages=meta(20, 2, 64, 128, dtype=f16)), "pools must be"),
    (dict(v_pages=meta(20, 2, 32, 128)), "matching"),
    (dict(k_pages=meta(20, 2, 128, 64).transpose(2, 3)), "D contiguous"),
    (dict(block_table=meta(3, 8, dtype=torch.int64)), "block_table"),
    (dict(block_table=meta(24, dtype=i32)), "block_table"),
    (dict(block_table=meta(8, 3, dtype=i32).t()), "block_table"),
    (dict(seq_lens=meta(4, dtype=i32)), "seq_lens"),
    (dict(cu_seqlens=meta(3, dtype=i32)), "cu_seqlens"),
    (dict(cu_seqlens=None), "one new token"),
    (dict(k_scales=meta(20, 2, dtype=f32)), "E4M3 pools only"),
    (dict(_cache(kv=u8), k_scales=None), "k_scales"),
    (dict(_cache(kv=u8), v_scales=meta(2, 20, dtype=f32)), "v_scales"),
]


@pytest.mark.parametrize("kw,match", POOL_CASES)
def test_pools_front(kw, match):
    for call in (_append, _attend):
        with pytest.raises(ValueError, match=match):
            call(**kw)


@pytest.mark.parametrize("kw,match", [
    ({}, "device tensors"),
    (dict(q=None), "device tensors"),
    (dict(cos=meta(9, 32, dtype=f32), sin=meta(9, 32, dtype=f32)), "device tensors"),
    (dict(k=meta(10, 3, 128)), "k is"),
    (dict(v=meta(9, 2, 128)), "v is"),
    (dict(v=meta(10, 2, 128, dtype=f16)), "v is"),
    (dict(q=meta(10, 8, 64)), "q is"),
    (dict(k=meta(10, 2, 128, dtype=f32), v=meta(10, 2, 128, dtype=f32)), "float16 or bfloat16"),
    (dict(out=meta(10, 4, 128)), "out is"),
    (dict(q=None, out=meta(10, 8, 128)), "go with q"),
    (dict(q=None, q_weight=meta(128, dtype=f32)), "go with q"),
    (dict(cos=meta(9, 32, dtype=f32)), "together"),
    (dict(k_weight=meta(64, dtype=f32)), "k_weight"),
])
def test_append_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(q=meta(8, 128)), "tokens, Hq, D"),
    (dict(q=meta(10, 8, 64)), "q is"),
    (dict(q=meta(10, 8, 128, dtype=f32)), "float16 or bfloat16"),
    (dict(out=meta(10, 8, 128, dtype=f16)), "out is"),
])
def test_attend_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


def test_workspace_bytes():
    """None where the keys cannot be cut, bounded by the launch's split states."""
    w = ops.attention_paged_workspace_bytes
    assert w(8, 8, 32, 8, 128, 448) == 0
    assert w(8192, 1, 32, 8, 128, 8192) == 0
    assert 0 < w(1, 1, 32, 8, 128, 32768) <= 2 * 1024 * 4 * 130 * 4
    assert 0 < w(4096, 16, 32, 8, 128, 32768) <= 2 * 1024 * 128 * 130 * 4
    with pytest.raises(_abi.NeptuneUnsupported, match="head_dim"):
        w(8, 8, 32, 8, 96, 448)
    with pytest.raises(_abi.NeptuneUnsupported, match="BF16 queries"):
        w(8, 8, 32, 8, 128, 448, dtype=f16, fp8=True)


# ---- C-ABI -----------------------------------------------------------------

FAR = 1 << 44  # placeholder addresses, far apart: no call here gets past validation


def _ptr(i):
    return (i + 1) * FAR


@pytest.fixture(scope="module")
def lib():
    return _abi.load_library()


def _set(desc, kw):
    for k, v in kw.items():
        if k.endswith("stride"):
            getattr(desc, k)[:] = v
        else:
            setattr(desc, k, v)
    return desc


def _rope_call(lib, ptrs=None, **kw):
    d = _abi.RopeDesc()
    d.batch, d.heads_q, d.heads_kv, d.seq, d.head_dim = 2, 8, 2, 5, 128
    d.rot_dim, d.table_len, d.dtype, d.eps = 128, 100, _abi.DTYPE_BF16, 1e-6
    p = [_ptr(i) for i in range(9)]  # q k qw kw cos sin positions qo ko
    for i, v in (ptrs or {}).items():
        p[i] = v
    return lib.neptune_qk_norm_rope(ctypes.byref(_set(d, kw)), *p, None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=0), INVALID), (dict(seq=-1), INVALID), (dict(heads_kv=0), INVALID),
    (dict(rot_dim=0), INVALID), (dict(rot_dim=136), INVALID), (dict(table_len=0), INVALID),
    (dict(rot_dim=12), UNSUPPORTED), (dict(head_dim=96, rot_dim=96), UNSUPPORTED),
    (dict(dtype=_abi.DTYPE_FP8_E4M3), UNSUPPORTED), (dict(interleaved=2), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(q_stride=(0, 640, 128)), INVALID), (dict(k_stride=(1280, 640, 132)), UNSUPPORTED),
    (dict(qo_stride=(1 << 62, 640, 128), batch=9), UNSUPPORTED),
    (dict(batch=1 << 20, seq=1 << 10), UNSUPPORTED),
    (dict(batch=1 << 50, seq=1 << 10), UNSUPPORTED),
    (dict(ptrs={0: None}), INVALID), (dict(ptrs={6: None}), INVALID),
    (dict(ptrs={4: None}), INVALID), (dict(ptrs={8: None}), INVALID),
    (dict(ptrs={0: FAR + 8}), UNSUPPORTED), (dict(ptrs={2: FAR + 4}), UNSUPPORTED),
    (dict(ptrs={7: _ptr(0) + 256}), INVALID),     # qo over q, moved
    (dict(ptrs={7: _ptr(1)}), INVALID),           # qo over k
    (dict(ptrs={8: _ptr(7) + 16}), INVALID),      # ko over qo
    (dict(ptrs={7: _ptr(0), 8: _ptr(0)}), INVALID),
    (dict(ptrs={7: _ptr(0)}, qo_stride=(1 << 20, 1 << 10, 256)), INVALID),  # other strides
    ({}, NO_DEVICE), (dict(ptrs={7: _ptr(0), 8: _ptr(1)}), NO_DEVICE),
    (dict(ptrs={2: None, 3: None}), NO_DEVICE),
    (dict(batch=1, q_stride=(4, 640, 128)), NO_DEVICE),  # no step along a size of 1
])
def test_rope_abi(lib, kw, status):
    if status == NO_DEVICE and lib.neptune_device_count() > 0:
        pytest.skip("a HIP device is visible; the no-device path is not reachable")
    assert _rope_call(lib, **kw) == status
    assert lib.neptune_last_error()


def _pages(**kw):
    p = _abi.PagedKvDesc()
    p.num_pages, p.page_size, p.max_pages = 64, 64, 32
    p.k_stride[:] = p.v_stride[:] = (2 * 64 * 128, 64 * 128, 128)
    return _set(p, kw)


def _append_call(lib, pages=None, ptrs=None, **kw):
    d = _abi.AppendDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim = 10, 3, 8, 2, 128
    d.rot_dim, d.table_len = 32, 100
    d.dtype = d.kv_dtype = _abi.DTYPE_BF16
    p = [_ptr(i) for i in range(15)]
    # 0 k, 1 v, 2 q, 3 qw, 4 kw, 5 cos, 6 sin, 7 table, 8 cu, 9 lens, 10 kp, 11 vp, 12 ks, 13 vs, 14 qo
    for i, v in (ptrs or {}).items():
        p[i] = v
    pg = _pages(**(pages or {})) if pages != "none" else None
    return lib.neptune_kv_append_paged(ctypes.byref(_set(d, kw)),
                                       ctypes.byref(pg) if pg is not None else None, *p, None)


def _attend_call(lib, pages=None, ptrs=None, ws=1 << 30, **kw):
    d = _abi.AttnPagedDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim, d.seq_kv = 10, 3, 8, 2, 128, 2000
    d.dtype = d.kv_dtype = _abi.DTYPE_BF16
    p = [_ptr(i) for i in range(11)]
    # 0 q, 1 kp, 2 vp, 3 ks, 4 vs, 5 table, 6 cu, 7 lens, 8 o, 9 lse, 10 workspace
    for i, v in (ptrs or {}).items():
        p[i] = v
    pg = _pages(**(pages or {})) if pages != "none" else None
    return lib.neptune_attn_paged(ctypes.byref(_set(d, kw)),
                                  ctypes.byref(pg) if pg is not None else None, *p, ws, None)


FP8 = _abi.DTYPE_FP8_E4M3
SHARED = [
    (dict(tokens=0), INVALID), (dict(batch=-1), INVALID), (dict(heads_kv=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=32), UNSUPPORTED),
    (dict(dtype=_abi.DTYPE_F32), UNSUPPORTED), (dict(kv_dtype=_abi.DTYPE_F16), UNSUPPORTED),
    (dict(pages="none"), INVALID), (dict(pages=dict(num_pages=0)), INVALID),
    (dict(pages=dict(page_size=0)), INVALID), (dict(pages=dict(max_pages=-1)), INVALID),
    (dict(pages=dict(k_stride=(0, 0, 0))), INVALID),
    (dict(pages=dict(v_stride=(2 * 64 * 128, 64 * 128, 132))), UNSUPPORTED),
    (dict(pages=dict(k_stride=(1 << 62, 64 * 128, 128))), UNSUPPORTED),
    (dict(kv_dtype=FP8, pages=dict(k_stride=(2 * 64 * 128, 64 * 128, 136))), UNSUPPORTED),
    (dict(pages=dict(num_pages=1 << 31, k_stride=(16, 8192, 128), v_stride=(16, 8192, 128))),
     UNSUPPORTED),
    (dict(q_stride=(1024, 0)), INVALID), (dict(q_stride=(1028, 128)), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,status", SHARED + [
    (dict(heads_q=-1), INVALID), (dict(rot_dim=130), INVALID), (dict(rot_dim=4), UNSUPPORTED),
    (dict(table_len=0), INVALID), (dict(interleaved=-1), INVALID),
    (dict(eps=float("inf")), INVALID),
    (dict(ptrs={8: None}), INVALID),                    # 10 tokens, 3 sequences
    (dict(kv_dtype=FP8, ptrs={12: None}), INVALID), (dict(ptrs={0: None}), INVALID),
    (dict(ptrs={2: None}), INVALID), (dict(ptrs={14: None}), INVALID),
    (dict(ptrs={5: None}), INVALID), (dict(ptrs={7: None}), INVALID),
    (dict(ptrs={9: None}), INVALID), (dict(ptrs={11: None}), INVALID),
    (dict(ptrs={1: FAR + 2}), UNSUPPORTED), (dict(ptrs={10: _ptr(10) + 8}), UNSUPPORTED),
    (dict(ptrs={14: _ptr(0)}), INVALID),                # qo over k
    (dict(ptrs={14: _ptr(2) + 16}), INVALID),           # qo over q, moved
    (dict(ptrs={14: _ptr(11) + 4096}), INVALID),        # qo over a pool
    (dict(ptrs={10: _ptr(1)}), INVALID),                # a pool over v
    (dict(tokens=1 << 31), UNSUPPORTED),
    ({}, NO_DEVICE), (dict(ptrs={14: _ptr(2)}), NO_DEVICE),
    (dict(heads_q=0, ptrs={2: None, 3: None, 14: None}), NO_DEVICE),
    (dict(rot_dim=0, table_len=0, ptrs={5: None, 6: None}), NO_DEVICE),
    (dict(tokens=3, ptrs={8: None}), NO_DEVICE),
    (dict(pages=dict(page_size=1)), NO_DEVICE), (dict(kv_dtype=FP8), NO_DEVICE),
    (dict(dtype=_abi.DTYPE_F16, kv_dtype=FP8), NO_DEVICE),
])
def test_append_abi(lib, kw, status):
    if status == NO_DEVICE and lib.neptune_device_count() > 0:
        pytest.skip("a HIP device is visible; the no-device path is not reachable")
    assert _append_call(lib, **kw) == status
    assert lib.neptune_last_error()


@pytest.mark.parametrize("kw,status", SHARED + [
    (dict(heads_q=0), INVALID), (dict(heads_q=9), INVALID), (dict(seq_kv=0), INVALID),
    (dict(scale_log2=-1.0), INVALID), (dict(scale_log2=float("nan")), INVALID),
    (dict(dtype=_abi.DTYPE_F16, kv_dtype=FP8), UNSUPPORTED),
    (dict(pages=dict(page_size=24, max_pages=100)), UNSUPPORTED), (dict(pages=dict(max_pages=31)), INVALID),
    (dict(seq_kv=(1 << 30) + 1, pages=dict(max_pages=1 << 25)), UNSUPPORTED),
    (dict(pages=dict(k_stride=(1 << 36, 128, 1 << 28))), UNSUPPORTED),
    (dict(tokens=1 << 30), UNSUPPORTED), (dict(batch=1 << 25), UNSUPPORTED),
    (dict(ptrs={6: None}), INVALID), (dict(kv_dtype=FP8, ptrs={4: None}), INVALID),
    (dict(ptrs={0: None}), INVALID), (dict(ptrs={5: None}), INVALID),
    (dict(ptrs={7: None}), INVALID), (dict(ptrs={8: None}), INVALID),
    (dict(ptrs={8: _ptr(0)}), INVALID), (dict(ptrs={8: _ptr(1) + 4096}), INVALID),
    (dict(ptrs={8: _ptr(8) + 8}), UNSUPPORTED), (dict(ptrs={10: _ptr(10) + 8}), UNSUPPORTED),
    (dict(ptrs={10: None}), SMALL), (dict(ws=16), SMALL),
    ({}, NO_DEVICE), (dict(ptrs={9: None}), NO_DEVICE), (dict(kv_dtype=FP8), NO_DEVICE),
    (dict(seq_kv=400, ptrs={10: None}, ws=0), NO_DEVICE),
    (dict(tokens=3, ptrs={6: None}), NO_DEVICE),
])
def test_attend_abi(lib, kw, status):
    if status == NO_DEVICE and lib.neptune_device_count() > 0:
        pytest.skip("a HIP device is visible; the no-device path is not reachable")
    assert _attend_call(lib, **kw) == status
    assert lib.neptune_last_error()


def test_null_descriptors(lib):
    p = ctypes.c_size_t()
    assert lib.neptune_qk_norm_rope(None, *[FAR] * 9, None) == INVALID
    assert lib.neptune_kv_append_paged(None, None, *[FAR] * 15, None) == INVALID
    assert lib.neptune_attn_paged(None, None, *[FAR] * 11, 0, None) == INVALID
    assert lib.neptune_attn_paged_workspace_bytes(None, ctypes.byref(p)) == INVALID
    d = _abi.AttnPagedDesc()
    assert lib.neptune_attn_paged_workspace_bytes(ctypes.byref(d), None) == INVALID


def test_descriptors_match_the_c_header(tmp_path):
    pairs = [("neptune_rope_desc", _abi.RopeDesc), ("neptune_append_desc", _abi.AppendDesc),
             ("neptune_attn_paged_desc", _abi.AttnPagedDesc)]
    lines = [f'printf("%zu\\n", offsetof({c}, {f}));' for c, cls in pairs for f, _ in cls._fields_]
    lines += [f'printf("%zu\\n", sizeof({c}));' for c, _ in pairs]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"neptune_hip.h\"\n"
                   "int main(void) {" + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True,
                                          text=True).stdout.split()]
    want = [getattr(cls, f).offset for _, cls in pairs for f, _ in cls._fields_]
    assert got == want + [ctypes.sizeof(cls) for _, cls in pairs]
