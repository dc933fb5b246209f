"""torch-tensor front of the C-ABI (device memory and streams only).

Every function hands raw device pointers, sizes and the current HIP stream
to libneptune_hip.so; no computation happens in Python and there is no
fallback path: if the library is missing, ``load_library`` raises.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _abi
from ._abi import check, load_library

LOG2E = 1.4426950408889634

_TORCH_TO_DTYPE = {
    torch.float32: _abi.DTYPE_F32,
    torch.float16: _abi.DTYPE_F16,
    torch.bfloat16: _abi.DTYPE_BF16,
}


# The checks of a call and its descriptor depend on the tensors' shapes,
# strides, dtypes and devices and on the options alone, so each entry point
# keeps them by those values (bounded; a call that fails its checks is not
# kept) and by the options' types: 4.0 is no split count, equal to 4 or not.
# Working them out took 3-8 us of every call, as long as the smallest
# kernels run: now a lookup.
_PLANS = 1024


def _meta(t: torch.Tensor | None):
    """What a plan may know of a tensor."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(lib, device: torch.device, fn, *args) -> None:
    """fn(*args, stream) on the device's current stream, that device current."""
    index = device.index
    if torch.cuda.current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _raw_stream(index))
    if st:
        check(st, lib)


def _contiguous(meta) -> bool:
    """Tensor.is_contiguous() of such a tensor."""
    shape, stride = meta[0], meta[1]
    want = 1
    for n, s in zip(reversed(shape), reversed(stride)):
        if n == 0:
            return True
        if n != 1:
            if s != want:
                return 0 in shape
            want *= n
    return True


def _check_workspace(workspace: torch.Tensor | None, device: torch.device) -> None:
    if workspace is None:
        return
    if not workspace.is_cuda:
        raise ValueError("neptune_hip ops take device tensors")
    if workspace.device != device:
        raise ValueError("all tensors must be on the same device")
    # the library writes numel * element_size bytes from data_ptr
    if not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor")


def _require_cuda(*metas) -> None:
    dev = None
    for m in metas:
        if m is None:
            continue
        if m[3].type != "cuda":
            raise ValueError("neptune_hip ops take device tensors")
        if dev is None:
            dev = m[3]
        elif m[3] != dev:
            raise ValueError("all tensors must be on the same device")


def _check_not_repeated(shape, stride) -> None:
    # all zero strides mean contiguous rows to the library, not one row repeated
    if not any(stride[:-1]) and any(n > 1 for n in shape[:-1]):
        raise ValueError("expected a tensor, not one row expanded to its shape")


def _strides_bhs(meta) -> tuple[int, int, int]:
    shape, stride = meta[0], meta[1]
    if len(shape) != 4 or stride[-1] != 1:
        raise ValueError("expected a [batch, heads, seq, head_dim] tensor with unit head_dim stride")
    _check_not_repeated(shape, stride)
    return stride[:3]


def scale_to_log2(scale: float | None, head_dim: int) -> float:
    """Softmax scale (default 1/sqrt(D)) expressed in the exp2 domain."""
    if scale is None:
        return 0.0  # library default: log2(e)/sqrt(head_dim), HTile:24
    return float(scale) * LOG2E


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _attn_plan(q, k, v, out, lse, causal, scale, scale_log2, stages, k_dim_order):
    """(descriptor, bytes of the split states' workspace, LSE shape)."""
    _require_cuda(q, k, v, out, lse)
    if q[2] not in _TORCH_TO_DTYPE or k[2] != q[2] or v[2] != q[2]:
        raise ValueError(f"q, k, v must share one of {list(_TORCH_TO_DTYPE)}")
    B, Hq, Sq, D = q[0]
    if k_dim_order not in (0, 1):
        raise ValueError("k_dim_order must be 0 or 1")
    if k_dim_order:
        Bk, Hk, Dk, Sk = k[0]
    else:
        Bk, Hk, Sk, Dk = k[0]
    if (Bk, Dk) != (B, D) or tuple(v[0]) != (Bk, Hk, Sk, Dk):
        raise ValueError(f"shape mismatch: q {tuple(q[0])} k {tuple(k[0])} v {tuple(v[0])}")
    if out is not None and (out[0] != q[0] or out[2] != q[2]):
        raise ValueError("out must match q's shape and dtype")
    if lse is not None and (tuple(lse[0]) != (B, Hq, Sq) or lse[2] != torch.float32 or
                            not _contiguous(lse)):
        raise ValueError("lse must be a contiguous float32 [B, Hq, Sq] tensor")
    desc = _abi.AttnDesc()
    desc.batch, desc.heads_q, desc.heads_kv = B, Hq, Hk
    desc.seq_q, desc.seq_kv, desc.head_dim = Sq, Sk, D
    desc.q_stride[:] = _strides_bhs(q)
    desc.k_stride[:] = _strides_bhs(k)
    desc.v_stride[:] = _strides_bhs(v)
    desc.o_stride[:] = _strides_bhs(out) if out is not None else (Hq * Sq * D, Sq * D, D)
    desc.dtype = _TORCH_TO_DTYPE[q[2]]
    desc.causal = 1 if causal else 0
    desc.scale_log2 = scale_log2 if scale_log2 is not None else scale_to_log2(scale, D)
    desc.pipeline_stages = stages
    desc.k_dim_order = int(k_dim_order)
    lib = load_library()
    n = ctypes.c_size_t()
    # what the library refuses, the launch itself reports
    st = lib.neptune_attn_workspace_bytes(ctypes.byref(desc), ctypes.byref(n))
    return ctypes.byref(desc), n.value if st == _abi.OK else 0, (B, Hq, Sq)


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = False,
    scale: float | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    scale_log2: float | None = None,
    pipeline_stages: int = 0,
    k_dim_order: int = 0,
):
    """softmax(q k^T * scale) v with the HTile numeric policy.

    q [B, Hq, Sq, D], k/v [B, Hkv, Skv, D] in float32, float16 or bfloat16
    (any strides with D contiguous, but not one row expanded to all of them);
    returns out [B, Hq, Sq, D] (and lse [B, Hq, Sq] fp32 if asked).
    ``scale_log2`` gives the score scale already in the exp2 domain (the
    HTile program's own constant, HTile:24), in place of ``scale``.
    ``pipeline_stages`` (0 = default 2, or 1..3) sets how many K/V tiles the
    kernel stages in LDS ahead of use; with ``k_dim_order=1`` k is given as
    [B, Hkv, D, Skv] (seq contiguous), the order of a dimension_order =
    [1, 0] tile load. The stage count does not change the result, and short
    launches may keep two tiles whatever it says. Short launches with
    ``k_dim_order=0`` may be cut along the keys and those with 1 are not, so
    their results may differ by the 16-bit rounding of the probabilities.
    """
    if scale is not None and scale_log2 is not None:
        raise ValueError("give scale or scale_log2, not both")
    desc, ws_bytes, lse_shape = _attn_plan(
        _meta(q), _meta(k), _meta(v), _meta(out), _meta(lse), bool(causal),
        None if scale is None else float(scale),
        None if scale_log2 is None else float(scale_log2), int(pipeline_stages), k_dim_order)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if lse is not None:
        return_lse = True
    elif return_lse:
        lse = torch.empty(lse_shape, dtype=torch.float32, device=q.device)
    # states of split keys (short launches only): held by the caching allocator
    # until the current stream is past this call
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
    lib = load_library()
    _launch(lib, q.device, lib.neptune_attn_fwd_ws, desc, q.data_ptr(), k.data_ptr(),
            v.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None,
            ws.data_ptr() if ws is not None else None, ws_bytes)
    return (out, lse) if return_lse else out


def _decode_desc(q_shape, k_shape, num_splits, scale_block, scale, kv_dtype) -> _abi.DecodeDesc:
    B, Hq, D = q_shape
    Bk, Hk, L, Dk = k_shape
    desc = _abi.DecodeDesc()
    desc.batch, desc.heads_q, desc.heads_kv = B, Hq, Hk
    desc.seq_kv, desc.head_dim = L, D
    desc.num_splits = num_splits
    desc.scale_block = scale_block
    desc.q_dtype = _abi.DTYPE_BF16
    desc.kv_dtype = kv_dtype
    desc.scale_log2 = scale_to_log2(scale, D)
    return desc


def _decode_bytes(desc: _abi.DecodeDesc) -> int:
    n = ctypes.c_size_t()
    lib = load_library()
    check(lib.neptune_decode_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)), lib)
    return n.value


def decode_workspace_bytes(q, k, *, num_splits: int = 0, fp8: bool = False) -> int:
    return _decode_bytes(_decode_desc(_as_q3(q).shape, k.shape, num_splits, 64, None,
                                      _abi.DTYPE_FP8_E4M3 if fp8 else _abi.DTYPE_BF16))


def _as_q3(q: torch.Tensor) -> torch.Tensor:
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("decode takes one query token per sequence")
        q = q[:, :, 0, :]
    return q


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _decode_plan(q, k, v, k_scale, v_scale, num_splits, scale_block, scale):
    """(descriptor, workspace bytes)."""
    fp8 = k[2] in (torch.uint8, torch.float8_e4m3fn)
    if q[2] != torch.bfloat16:
        raise ValueError("decode query must be bfloat16")
    if not fp8 and k[2] != torch.bfloat16:
        raise ValueError("decode KV must be bfloat16 or E4M3 codes")
    if len(q[0]) != 3 or len(k[0]) != 4:
        raise ValueError("decode takes q [B, Hq, D] and k, v [B, Hkv, L, D]")
    if v[2] != k[2] or v[0] != k[0]:
        raise ValueError("k and v must match")
    B, _, D = q[0]
    Bk, Hk, L, Dk = k[0]
    if (Bk, Dk) != (B, D):
        raise ValueError(f"k {tuple(k[0])} does not match q {tuple(q[0])} in batch or "
                         "head_dim")
    for m in (q, k, v):
        if not _contiguous(m):
            raise ValueError("decode tensors must be contiguous")
    if fp8:
        if scale_block <= 0:
            raise ValueError("scale_block must be positive")
        want = (B, Hk, -(-L // scale_block))
        for name, m in (("k_scale", k_scale), ("v_scale", v_scale)):
            if m is None or m[2] != torch.float32 or not _contiguous(m) or tuple(m[0]) != want:
                raise ValueError(f"fp8 KV needs {name}: contiguous float32 {list(want)} "
                                 f"(scale_block {scale_block})")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("k_scale / v_scale apply to E4M3 KV only")
    _require_cuda(q, k, v, k_scale, v_scale)
    desc = _decode_desc(q[0], k[0], num_splits, scale_block, scale,
                        _abi.DTYPE_FP8_E4M3 if fp8 else _abi.DTYPE_BF16)
    return ctypes.byref(desc), _decode_bytes(desc)


def decode_splitk(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    num_splits: int = 0,
    scale_block: int = 64,
    scale: float | None = None,
    return_lse: bool = False,
    workspace: torch.Tensor | None = None,
):
    """Split-K flash-decoding over grouped KV heads.

    q [B, Hq, D] (or [B, Hq, 1, D]) bf16; k/v [B, Hkv, L, D] bf16, or E4M3
    codes (uint8 / torch.float8_e4m3fn) with k_scale/v_scale
    [B, Hkv, ceil(L/scale_block)] fp32. Returns o [B, Hq, D] bf16.
    """
    q3 = _as_q3(q)
    desc, need = _decode_plan(_meta(q3), _meta(k), _meta(v), _meta(k_scale), _meta(v_scale),
                              num_splits, scale_block, None if scale is None else float(scale))
    _check_workspace(workspace, q3.device)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q3.device)
    out = torch.empty_like(q3)
    lse = torch.empty(q3.shape[:2], dtype=torch.float32, device=q3.device) if return_lse else None
    lib = load_library()
    _launch(lib, q3.device, lib.neptune_decode_splitk, desc, q3.data_ptr(), k.data_ptr(),
            v.data_ptr(), k_scale.data_ptr() if k_scale is not None else None,
            v_scale.data_ptr() if v_scale is not None else None, out.data_ptr(),
            lse.data_ptr() if lse is not None else None, workspace.data_ptr(),
            workspace.numel() * workspace.element_size())
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _paged_plan(q, k_pages, v_pages, block_table, seq_lens, k_scales, v_scales, max_seq_len,
                num_splits, scale):
    """(descriptor, page descriptor, workspace bytes, whether the pools are E4M3)."""
    fp8 = k_pages[2] in (torch.uint8, torch.float8_e4m3fn)
    if q[2] != torch.bfloat16 or k_pages[2] != v_pages[2] or \
            not (fp8 or k_pages[2] == torch.bfloat16):
        raise ValueError("paged decode takes bfloat16 q and bfloat16 or E4M3 KV pages")
    if len(k_pages[0]) != 4 or k_pages[0] != v_pages[0] or k_pages[1][-1] != 1 or \
            v_pages[1][-1] != 1:
        raise ValueError("k_pages / v_pages: matching [pages, Hkv, page_size, D] views, D contiguous")
    for name, m in (("block_table", block_table), ("seq_lens", seq_lens)):
        if m[2] != torch.int32 or not _contiguous(m):
            raise ValueError(f"{name} must be a contiguous int32 tensor")
    npages, Hk, psize, D = k_pages[0]
    if len(q[0]) != 3 or q[0][2] != D:
        raise ValueError(f"q {tuple(q[0])} does not match the pools' head_dim {D}")
    if fp8:
        for name, m in (("k_scales", k_scales), ("v_scales", v_scales)):
            if m is None or m[2] != torch.float32 or not _contiguous(m) or \
                    tuple(m[0]) != (npages, Hk):
                raise ValueError(f"fp8 pages need {name}: contiguous float32 [num_pages, Hkv]")
    elif k_scales is not None or v_scales is not None:
        raise ValueError("k_scales / v_scales apply to E4M3 pools only")
    B = q[0][0]
    if len(block_table[0]) != 2 or block_table[0][0] != B or tuple(seq_lens[0]) != (B,):
        raise ValueError("block_table [B, max_pages] and seq_lens [B] must match q's batch")
    _require_cuda(q, k_pages, v_pages, block_table, seq_lens, k_scales, v_scales)
    max_pages = block_table[0][1]
    L = max_seq_len if max_seq_len is not None else max_pages * psize
    desc = _decode_desc(q[0], (B, Hk, L, D), num_splits, psize if fp8 else 64, scale,
                        _abi.DTYPE_FP8_E4M3 if fp8 else _abi.DTYPE_BF16)
    pk = _abi.PagedKvDesc()
    pk.num_pages, pk.page_size, pk.max_pages = npages, psize, max_pages
    pk.k_stride[:] = k_pages[1][:3]
    pk.v_stride[:] = v_pages[1][:3]
    return ctypes.byref(desc), ctypes.byref(pk), _decode_bytes(desc), fp8


def decode_paged(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    max_seq_len: int | None = None,
    num_splits: int = 0,
    scale: float | None = None,
    return_lse: bool = False,
    workspace: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
):
    """Split-K decode over a paged KV cache.

    q [B, Hq, D] bf16; k_pages / v_pages [num_pages, Hkv, page_size, D]
    views (any page/head/position strides with D contiguous, e.g. a permuted
    [num_pages, page_size, Hkv, D] pool) of bf16, or of E4M3 codes (uint8 /
    torch.float8_e4m3fn) with k_scales / v_scales fp32 [num_pages, Hkv]
    (one scale per page and kv head); block_table [B, max_pages] and
    seq_lens [B] int32 on the device. ``max_seq_len`` (default
    max_pages * page_size) is the longest sequence and sets the split
    layout. Returns o [B, Hq, D] bf16.
    """
    q3 = _as_q3(q)
    desc, pk, need, fp8 = _paged_plan(
        _meta(q3), _meta(k_pages), _meta(v_pages), _meta(block_table), _meta(seq_lens),
        _meta(k_scales), _meta(v_scales), None if max_seq_len is None else int(max_seq_len),
        num_splits, None if scale is None else float(scale))
    _check_workspace(workspace, q3.device)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q3.device)
    out = torch.empty_like(q3)
    lse = torch.empty(q3.shape[:2], dtype=torch.float32, device=q3.device) if return_lse else None
    tail = (block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
            lse.data_ptr() if lse is not None else None, workspace.data_ptr(),
            workspace.numel() * workspace.element_size())
    lib = load_library()
    if fp8:
        _launch(lib, q3.device, lib.neptune_decode_paged_fp8, desc, pk, q3.data_ptr(),
                k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                *tail)
    else:
        _launch(lib, q3.device, lib.neptune_decode_paged, desc, pk, q3.data_ptr(),
                k_pages.data_ptr(), v_pages.data_ptr(), *tail)
    return (out, lse) if return_lse else out


def kv_quantize_fp8(kv: torch.Tensor, *, scale_block: int = 64):
    """bf16 [B, Hkv, L, D] -> (E4M3 codes uint8, scales fp32 [B, Hkv, nblocks])."""
    if not kv.is_cuda:
        raise ValueError("neptune_hip ops take device tensors")
    if kv.dtype != torch.bfloat16 or kv.dim() != 4 or not kv.is_contiguous():
        raise ValueError("kv_quantize_fp8 takes a contiguous bf16 [B, Hkv, L, D] tensor")
    B, Hk, L, D = kv.shape
    device = kv.device
    codes = torch.empty(kv.shape, dtype=torch.uint8, device=device)
    scales = torch.empty((B, Hk, -(-L // scale_block)), dtype=torch.float32, device=device)
    lib = load_library()
    _launch(lib, device, lib.neptune_kv_quantize_fp8, B, Hk, L, D, scale_block, kv.data_ptr(),
            codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _check_rotation(name, cos, sin, weights, head_dim) -> tuple[int, int]:
    """(rot_dim, table_len) of the tables, checked with the norm weights."""
    if (cos is None) != (sin is None):
        raise ValueError(f"{name}: give cos and sin together")
    if cos is not None:
        for what, m in (("cos", cos), ("sin", sin)):
            if m[2] != torch.float32 or len(m[0]) != 2 or not _contiguous(m):
                raise ValueError(f"{name}: {what} must be a contiguous float32 "
                                 "[positions, rot_dim / 2] tensor")
        if cos[0] != sin[0]:
            raise ValueError(f"{name}: cos {tuple(cos[0])} and sin {tuple(sin[0])} must match")
    for what, m in weights:
        if m is not None and (m[2] != torch.float32 or tuple(m[0]) != (head_dim,) or
                              not _contiguous(m)):
            raise ValueError(f"{name}: {what} must be a contiguous float32 [{head_dim}] tensor")
    return (0, 0) if cos is None else (2 * cos[0][1], cos[0][0])


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _rope_plan(q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out, eps, interleaved):
    """The descriptor."""
    if q[2] not in _TORCH_TO_DTYPE or k[2] != q[2]:
        raise ValueError(f"q and k must share one of {list(_TORCH_TO_DTYPE)}")
    strides = [_strides_bhs(m) for m in (q, k)]
    B, Hq, S, D = q[0]
    Hk = k[0][1]
    if tuple(k[0]) != (B, Hk, S, D):
        raise ValueError(f"shape mismatch: q {tuple(q[0])} k {tuple(k[0])}")
    for what, m, src in (("q", q_out, q), ("k", k_out, k)):
        if m is None:
            strides.append((0, 0, 0))
            continue
        if m[0] != src[0] or m[2] != src[2]:
            raise ValueError(f"out must match {what}'s shape and dtype")
        strides.append(_strides_bhs(m))
    if cos is None:
        raise ValueError("qk_norm_rope takes cos and sin tables")
    rot, rows = _check_rotation("qk_norm_rope", cos, sin,
                                (("q_weight", q_weight), ("k_weight", k_weight)), D)
    if positions[2] != torch.int32 or tuple(positions[0]) != (B, S) or not _contiguous(positions):
        raise ValueError("positions must be a contiguous int32 [B, S] tensor")
    _require_cuda(q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out)
    desc = _abi.RopeDesc()
    desc.batch, desc.heads_q, desc.heads_kv, desc.seq, desc.head_dim = B, Hq, Hk, S, D
    desc.rot_dim, desc.table_len = rot, rows
    desc.q_stride[:], desc.k_stride[:], desc.qo_stride[:], desc.ko_stride[:] = strides
    desc.dtype = _TORCH_TO_DTYPE[q[2]]
    desc.interleaved = interleaved
    desc.eps = eps
    return ctypes.byref(desc)


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each query and key head and its position rotation, one pass.

    q [B, Hq, S, D], k [B, Hkv, S, D] in float32, float16 or bfloat16 (any
    strides of whole 16-byte units with D contiguous, such as transposed
    [B, S, H, D] projections); cos, sin float32 [positions, rot_dim / 2] (the
    first rot_dim of D elements turn: pairs (i, i + rot_dim / 2), or
    (2i, 2i + 1) when ``interleaved``); positions int32 [B, S]. With
    ``q_weight`` / ``k_weight`` float32 [D] the heads are normalised first:
    x * w / sqrt(mean(x^2) + eps). ``out`` = (q_out, k_out) may be (q, k).
    Returns (q_out, k_out), by default new contiguous tensors.
    """
    if out is not None and not (isinstance(out, (tuple, list)) and len(out) == 2 and
                                all(isinstance(t, torch.Tensor) for t in out)):
        raise ValueError("out must be a pair of tensors (q_out, k_out)")
    q_out, k_out = (None, None) if out is None else out
    desc = _rope_plan(_meta(q), _meta(k), _meta(cos), _meta(sin), _meta(positions),
                      _meta(q_weight), _meta(k_weight), _meta(q_out), _meta(k_out), float(eps),
                      1 if interleaved else 0)
    if out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    lib = load_library()
    _launch(lib, q.device, lib.neptune_qk_norm_rope, desc, q.data_ptr(), k.data_ptr(),
            _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
            q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def _strides_th(name, meta, heads, head_dim, tokens, dtype) -> tuple[int, int]:
    shape, stride = meta[0], meta[1]
    if len(shape) != 3 or stride[-1] != 1:
        raise ValueError(f"{name}: expected [tokens, heads, head_dim] with unit head_dim stride")
    if tuple(shape) != (tokens, heads, head_dim) or meta[2] != dtype:
        raise ValueError(f"{name} is {tuple(shape)} {meta[2]}, expected "
                         f"{(tokens, heads, head_dim)} {dtype}")
    _check_not_repeated(shape, stride)
    return stride[:2]


_E2M1 = getattr(torch, "float4_e2m1fn_x2", None)
_E8M0 = getattr(torch, "float8_e8m0fnu", None)


def _is_mx(k_pages, k_scales) -> bool:
    """MXFP4 pools: bytes of codes whose scales are bytes too, or torch's types."""
    if _E2M1 is not None and k_pages[2] == _E2M1:
        return True
    return k_pages[2] == torch.uint8 and k_scales is not None and \
        k_scales[2] in (torch.uint8, _E8M0)


def _mx_plan(name, k_pages, v_pages, k_scales, v_scales) -> _abi.MxDesc:
    """The scales' descriptor, checked with the pools'."""
    npages, Hk, psize, half = k_pages[0]
    want = (npages, Hk, psize, half // 16)
    for what, m in (("k_scales", k_scales), ("v_scales", v_scales)):
        if m is None or m[2] not in (torch.uint8, _E8M0) or tuple(m[0]) != want or m[1][-1] != 1:
            raise ValueError(f"{name}: MXFP4 pools need {what}: a uint8 view {list(want)}, the last "
                             "axis contiguous")
    mx = _abi.MxDesc()
    mx.k_stride[:] = k_scales[1][:3]
    mx.v_stride[:] = v_scales[1][:3]
    return mx


def _pool_plan(name, dtype, tokens, k_pages, v_pages, block_table, seq_lens, cu_seqlens,
               k_scales, v_scales):
    """(page descriptor, neptune dtype of the pools, batch, head_dim, MXFP4 descriptor or
    None) of a ragged batch."""
    mx = _is_mx(k_pages, k_scales)
    fp8 = not mx and k_pages[2] in (torch.uint8, torch.float8_e4m3fn)
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name} takes float16 or bfloat16 tensors")
    if k_pages[2] != v_pages[2] or not (fp8 or mx or k_pages[2] == dtype):
        raise ValueError(f"{name}: the pools must be {dtype}, E4M3 or MXFP4, both alike")
    if len(k_pages[0]) != 4 or k_pages[0] != v_pages[0] or k_pages[1][-1] != 1 or \
            v_pages[1][-1] != 1:
        raise ValueError("k_pages / v_pages: matching [pages, Hkv, page_size, D] views, D contiguous")
    npages, Hk, psize, width = k_pages[0]
    if len(block_table[0]) != 2:
        raise ValueError("block_table must be [B, max_pages]")
    B, max_pages = block_table[0]
    want = {"block_table": (B, max_pages), "seq_lens": (B,), "cu_seqlens": (B + 1,)}
    for what, m in (("block_table", block_table), ("seq_lens", seq_lens),
                    ("cu_seqlens", cu_seqlens)):
        if m is None:
            continue
        if m[2] != torch.int32 or not _contiguous(m):
            raise ValueError(f"{what} must be a contiguous int32 tensor")
        if tuple(m[0]) != want[what]:
            raise ValueError(f"{what} is {tuple(m[0])}, expected {want[what]}")
    if cu_seqlens is None and tokens != B:
        raise ValueError(f"without cu_seqlens every sequence has one new token: {tokens} tokens, "
                         f"{B} sequences")
    if fp8:
        for what, m in (("k_scales", k_scales), ("v_scales", v_scales)):
            if m is None or m[2] != torch.float32 or not _contiguous(m) or \
                    tuple(m[0]) != (npages, Hk):
                raise ValueError(f"fp8 pages need {what}: contiguous float32 [num_pages, Hkv]")
    elif not mx and (k_scales is not None or v_scales is not None):
        raise ValueError("k_scales / v_scales apply to MXFP4 and E4M3 pools only")
    pk = _abi.PagedKvDesc()
    pk.num_pages, pk.page_size, pk.max_pages = npages, psize, max_pages
    pk.k_stride[:] = k_pages[1][:3]
    pk.v_stride[:] = v_pages[1][:3]
    if mx:
        return (pk, _abi.DTYPE_MXFP4, B, 2 * width,
                _mx_plan(name, k_pages, v_pages, k_scales, v_scales))
    return pk, _abi.DTYPE_FP8_E4M3 if fp8 else _TORCH_TO_DTYPE[dtype], B, width, None


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _append_plan(k, v, k_pages, v_pages, block_table, seq_lens, cu_seqlens, q, cos, sin, q_weight,
                 k_weight, k_scales, v_scales, out, eps, interleaved):
    """(descriptor, page descriptor, MXFP4 descriptor or None)."""
    T = k[0][0] if len(k[0]) == 3 else 0
    pk, kv_dtype, B, D, mx = _pool_plan("kv_append_paged", k[2], T, k_pages, v_pages, block_table,
                                        seq_lens, cu_seqlens, k_scales, v_scales)
    Hk = k_pages[0][1]
    desc = _abi.AppendDesc()
    desc.k_stride[:] = _strides_th("k", k, Hk, D, T, k[2])
    desc.v_stride[:] = _strides_th("v", v, Hk, D, T, k[2])
    Hq = 0
    if q is not None:
        Hq = q[0][1] if len(q[0]) == 3 else 0
        desc.q_stride[:] = _strides_th("q", q, Hq, D, T, k[2])
        if out is not None:
            desc.qo_stride[:] = _strides_th("out", out, Hq, D, T, k[2])
    elif out is not None or q_weight is not None:
        raise ValueError("out and q_weight go with q")
    rot, rows = _check_rotation("kv_append_paged", cos, sin,
                                (("q_weight", q_weight), ("k_weight", k_weight)), D)
    _require_cuda(k, v, k_pages, v_pages, block_table, seq_lens, cu_seqlens, q, cos, sin, q_weight,
                  k_weight, k_scales, v_scales, out)
    desc.tokens, desc.batch, desc.heads_q, desc.heads_kv, desc.head_dim = T, B, Hq, Hk, D
    desc.rot_dim, desc.table_len = rot, rows
    desc.dtype, desc.kv_dtype = _TORCH_TO_DTYPE[k[2]], kv_dtype
    desc.interleaved, desc.eps = interleaved, eps
    return ctypes.byref(desc), ctypes.byref(pk), None if mx is None else ctypes.byref(mx)


def kv_append_paged(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    interleaved: bool = False,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Write new tokens' keys and values into a paged cache, in place.

    k, v [T, Hkv, D] float16 or bfloat16, the new tokens of all sequences one
    after the other: sequence b has rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1
    (without ``cu_seqlens`` one row each), and seq_lens[b] counts its tokens
    with them, so that its last row lands at seq_lens[b] - 1. k_pages / v_pages
    [num_pages, Hkv, page_size, D] views as in ``decode_paged``, of k's dtype or
    E4M3 codes under the given k_scales / v_scales [num_pages, Hkv] (of either
    dtype's values: ``attention_paged`` and ``decode_paged`` read codes with
    bfloat16 queries, a float16 model casts its own), or MXFP4; block_table
    [B, max_pages], seq_lens [B], cu_seqlens [B + 1] int32 on the device.

    MXFP4 pools hold four bits an element: k_pages / v_pages [num_pages, Hkv,
    page_size, D / 2] of bytes (uint8, or torch.float4_e2m1fn_x2), two E2M1 codes each,
    the even element's in the low half, and k_scales / v_scales [num_pages, Hkv,
    page_size, D / 32] of bytes (uint8, or torch.float8_e8m0fnu), the scale 2^(e - 127)
    of 32 elements each (255: NaN), views of any page/head/position strides alike. The
    scales are outputs here: each block of 32 is quantised as it is written, by its
    largest magnitude, to the nearest codes. (Two rows sent to one slot may leave codes of
    one under scales of the other.)

    Keys are normalised (``k_weight``) and rotated (``cos``, ``sin``,
    ``interleaved``) at their positions on the way, as in ``qk_norm_rope``; with
    ``q`` [T, Hq, D] the queries too, and [T, Hq, D] is returned (``out``, which
    may be q, or a new tensor; None without q). A row without a slot (a
    negative place, one past its table, a table entry outside the pool) is not
    stored. ``cos`` and ``sin`` must reach the longest sequence: a place past
    their last row is turned by that row's angles and stored all the same. Rows
    behind the last sequence are left out of the cache and of the result: they
    stay as they were in ``out``, and in a new tensor hold whatever its memory
    held, so a padded step gives its own ``out``.
    """
    desc, pk, mx = _append_plan(
        _meta(k), _meta(v), _meta(k_pages), _meta(v_pages), _meta(block_table), _meta(seq_lens),
        _meta(cu_seqlens), _meta(q), _meta(cos), _meta(sin), _meta(q_weight), _meta(k_weight),
        _meta(k_scales), _meta(v_scales), _meta(out), float(eps), 1 if interleaved else 0)
    if q is not None and out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lib = load_library()
    entry = (lib.neptune_kv_append_paged, desc, pk) if mx is None else \
        (lib.neptune_kv_append_paged_mx, desc, pk, mx)
    _launch(lib, k.device, *entry, k.data_ptr(), v.data_ptr(),
            _ptr(q), _ptr(q_weight), _ptr(k_weight), _ptr(cos), _ptr(sin), block_table.data_ptr(),
            _ptr(cu_seqlens), seq_lens.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            _ptr(k_scales), _ptr(v_scales), _ptr(out))
    return out


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _read_plan(k_pages, v_pages, block_table, seq_lens, cu_seqlens, k_scales, v_scales, k_out,
               v_out, tokens, dtype):
    """(descriptor, page descriptor, MXFP4 descriptor or None, rows' shape, their dtype)."""
    if tokens is None:
        if k_out is None and cu_seqlens is not None:
            raise ValueError("kv_read_paged: give tokens (or out) with cu_seqlens")
        tokens = k_out[0][0] if k_out is not None and len(k_out[0]) == 3 else seq_lens[0][0]
    pool = k_pages[2] if k_pages[2] in (torch.float16, torch.bfloat16) else torch.bfloat16
    pk, kv_dtype, B, D, mx = _pool_plan("kv_read_paged", pool, tokens, k_pages, v_pages,
                                        block_table, seq_lens, cu_seqlens, k_scales, v_scales)
    if dtype is None:
        dtype = pool if k_out is None else k_out[2]
    if dtype not in _TORCH_TO_DTYPE:
        raise ValueError(f"dtype must be one of {list(_TORCH_TO_DTYPE)}")
    shape = (tokens, k_pages[0][1], D)
    desc = _abi.KvReadDesc()
    if k_out is not None:
        desc.ko_stride[:] = _strides_th("k_out", k_out, shape[1], D, tokens, dtype)
        desc.vo_stride[:] = _strides_th("v_out", v_out, shape[1], D, tokens, dtype)
    _require_cuda(k_pages, v_pages, block_table, seq_lens, cu_seqlens, k_scales, v_scales, k_out,
                  v_out)
    desc.tokens, desc.batch, desc.heads_kv, desc.head_dim = tokens, B, shape[1], D
    desc.dtype, desc.kv_dtype = _TORCH_TO_DTYPE[dtype], kv_dtype
    return (ctypes.byref(desc), ctypes.byref(pk), None if mx is None else ctypes.byref(mx), shape,
            dtype)


def kv_read_paged(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    tokens: int | None = None,
    dtype: torch.dtype | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached keys and values as rows: what ``kv_append_paged`` wrote, read back.

    Pools, tables and lengths as there (16-bit, E4M3 or MXFP4 pools): row r of
    sequence b, cu_seqlens[b] <= r < cu_seqlens[b + 1], is the token at place
    seq_lens[b] - (cu_seqlens[b + 1] - r), so that cu_seqlens of whole lengths reads
    whole sequences, and the step's own the rows just appended; without it, each
    sequence's last token. ``tokens`` is the number of rows (cu_seqlens[B], known to
    the caller; the device's is not waited for). Returns (k, v) [tokens, Hkv, D] in
    ``dtype`` float32, float16 or bfloat16 (default: the pools', bfloat16 for codes),
    new or ``out`` = (k_out, v_out). A row without a slot is zeros; rows behind the last
    sequence stay as they were in ``out``, and in new tensors hold whatever their memory
    held.
    """
    if out is not None and not (isinstance(out, (tuple, list)) and len(out) == 2 and
                                all(isinstance(t, torch.Tensor) for t in out)):
        raise ValueError("out must be a pair of tensors (k_out, v_out)")
    k_out, v_out = (None, None) if out is None else out
    desc, pk, mx, shape, dtype = _read_plan(
        _meta(k_pages), _meta(v_pages), _meta(block_table), _meta(seq_lens), _meta(cu_seqlens),
        _meta(k_scales), _meta(v_scales), _meta(k_out), _meta(v_out),
        None if tokens is None else int(tokens), dtype)
    if out is None:
        k_out, v_out = (torch.empty(shape, dtype=dtype, device=k_pages.device) for _ in range(2))
    lib = load_library()
    _launch(lib, k_pages.device, lib.neptune_kv_read_paged, desc, pk, mx, k_pages.data_ptr(),
            v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), block_table.data_ptr(),
            _ptr(cu_seqlens), seq_lens.data_ptr(), k_out.data_ptr(), v_out.data_ptr())
    return k_out, v_out


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _attn_paged_plan(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, k_scales, v_scales,
                     out, max_seq_len, scale, softcap, slopes, window):
    """(descriptor, page descriptor, workspace bytes, None or the MXFP4 and the scores'
    descriptors, either of them None)."""
    if len(q[0]) != 3:
        raise ValueError("attention_paged takes q [tokens, Hq, D]")
    T, Hq, _ = q[0]
    pk, kv_dtype, B, D, mx = _pool_plan("attention_paged", q[2], T, k_pages, v_pages, block_table,
                                        seq_lens, cu_seqlens, k_scales, v_scales)
    _, Hk, psize, _ = k_pages[0]
    desc = _abi.AttnPagedDesc()
    desc.q_stride[:] = _strides_th("q", q, Hq, D, T, q[2])
    if out is not None:
        desc.o_stride[:] = _strides_th("out", out, Hq, D, T, q[2])
    desc.scale_log2 = scale_to_log2(scale, D)
    if scale is not None and desc.scale_log2 == 0.0:  # the library's default otherwise
        raise ValueError("attention_paged: scale must not be 0")
    score = None
    if softcap is not None or window is not None:
        if softcap is not None and not softcap > 0.0:
            raise ValueError("attention_paged: softcap must be positive")
        if window is not None and window < 1:
            raise ValueError("attention_paged: window must be at least 1")
        # (a window past 64 bits hides nothing: it must not wrap)
        score = _abi.ScoreDesc(min(window or 0, 2**63 - 1), softcap or 0.0, 0)
        if softcap is not None and score.softcap == 0.0:  # none to the library
            raise ValueError("attention_paged: softcap must lie between 2^-60 and 2^60")
    if slopes is not None and (slopes[2] != torch.float32 or tuple(slopes[0]) != (Hq,) or
                               not _contiguous(slopes)):
        raise ValueError(f"attention_paged: slopes must be a contiguous float32 [{Hq}] tensor")
    _require_cuda(q, k_pages, v_pages, block_table, seq_lens, cu_seqlens, k_scales, v_scales, out,
                  slopes)
    desc.tokens, desc.batch, desc.heads_q, desc.heads_kv, desc.head_dim = T, B, Hq, Hk, D
    desc.seq_kv = max_seq_len if max_seq_len is not None else pk.max_pages * psize
    desc.dtype, desc.kv_dtype = _TORCH_TO_DTYPE[q[2]], kv_dtype
    n = ctypes.c_size_t()
    lib = load_library()
    check(lib.neptune_attn_paged_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)), lib)
    ext = None
    if mx is not None or score is not None or slopes is not None:
        ext = (None if mx is None else ctypes.byref(mx),
               None if score is None else ctypes.byref(score))
    return ctypes.byref(desc), ctypes.byref(pk), n.value, ext


def attention_paged(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    max_seq_len: int | None = None,
    scale: float | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    window: int | None = None,
):
    """Causal attention of new tokens over a paged cache that holds them.

    q [T, Hq, D] float16 or bfloat16, the new tokens of all sequences one after
    the other, any number each: a chunk of a prompt, guessed tokens to check, a
    single token, none (``cu_seqlens`` and ``seq_lens`` as in
    ``kv_append_paged``, called before). k_pages / v_pages, block_table,
    k_scales / v_scales as in ``decode_paged`` (pools of q's dtype, or E4M3 with
    bfloat16 q), or MXFP4 pools as ``kv_append_paged`` writes them (their values are
    read in q's dtype: float16 has those past 65504 as infinite, and rounds those
    below 2^-14 to steps of 2^-24); page sizes that are multiples of 16; D 64 or 128.
    ``max_seq_len`` (default max_pages * page_size) bounds the lengths. A row
    sees its sequence up to its own place; one with a negative place sees
    nothing: output 0, log-sum-exp -inf. Rows behind the last sequence are not
    written: they stay as they were in ``out``, and in a new tensor, lse among
    them, hold whatever its memory held (a padded step gives its own ``out``,
    and reads no lse there). Returns o [T, Hq, D] (and lse [T, Hq] fp32 if
    asked).

    Scores x = q . k * scale become softcap * tanh(x / softcap) with ``softcap``; with
    ``slopes`` float32 [Hq], slopes[h] * (j - p) is added for a key at place j and a
    row at place p; with ``window`` a row sees that many keys at most, its own the last
    of them. Any of them together, over pools of any kind.

    The workspace is for the calls of the sizes it was asked for: fewer tokens
    may need a larger one, since keys are cut where tiles are few.
    """
    desc, pk, need, ext = _attn_paged_plan(
        _meta(q), _meta(k_pages), _meta(v_pages), _meta(block_table), _meta(seq_lens),
        _meta(cu_seqlens), _meta(k_scales), _meta(v_scales), _meta(out),
        None if max_seq_len is None else int(max_seq_len), None if scale is None else float(scale),
        None if softcap is None else float(softcap), _meta(slopes),
        None if window is None else int(window))
    _check_workspace(workspace, q.device)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    lib = load_library()
    tail = (block_table.data_ptr(), _ptr(cu_seqlens), seq_lens.data_ptr(), out.data_ptr(),
            _ptr(lse), _ptr(workspace),
            0 if workspace is None else workspace.numel() * workspace.element_size())
    if ext is None:
        _launch(lib, q.device, lib.neptune_attn_paged, desc, pk, q.data_ptr(), k_pages.data_ptr(),
                v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales), *tail)
    else:
        _launch(lib, q.device, lib.neptune_attn_paged_ext, desc, pk, *ext, q.data_ptr(),
                k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scales), _ptr(v_scales),
                _ptr(slopes), *tail)
    return (out, lse) if return_lse else out


def attention_paged_workspace_bytes(
    tokens: int, batch: int, heads_q: int, heads_kv: int, head_dim: int, max_seq_len: int,
    *, dtype: torch.dtype = torch.bfloat16, fp8: bool = False,
) -> int:
    """Bytes of ``attention_paged``'s workspace for such a call (0: none); MXFP4 pools, a
    cap, slopes and a window change none of it."""
    desc = _abi.AttnPagedDesc()
    desc.tokens, desc.batch, desc.heads_q, desc.heads_kv = tokens, batch, heads_q, heads_kv
    desc.head_dim, desc.seq_kv = head_dim, max_seq_len
    if dtype not in _TORCH_TO_DTYPE:
        raise ValueError(f"dtype must be one of {list(_TORCH_TO_DTYPE)}")
    desc.dtype = _TORCH_TO_DTYPE[dtype]
    desc.kv_dtype = _abi.DTYPE_FP8_E4M3 if fp8 else desc.dtype
    n = ctypes.c_size_t()
    lib = load_library()
    check(lib.neptune_attn_paged_workspace_bytes(ctypes.byref(desc), ctypes.byref(n)), lib)
    return n.value


@functools.lru_cache(maxsize=_PLANS, typed=True)
def _scan_plan(u, delta, A, B, C, D, z, delta_bias, delta_softplus):
    """The descriptor."""
    for name, m in (("u", u), ("delta", delta), ("B", B), ("C", C), ("z", z)):
        if m is not None and (m[2] != torch.bfloat16 or not _contiguous(m)):
            raise ValueError(f"{name} must be contiguous bfloat16")
    for name, m in (("A", A), ("D", D), ("delta_bias", delta_bias)):
        if m is not None and (m[2] != torch.float32 or not _contiguous(m)):
            raise ValueError(f"{name} must be contiguous float32")
    if len(u[0]) != 3 or len(A[0]) != 2:
        raise ValueError("selective_scan takes u [batch, dim, L] and A [dim, d_state]")
    bsz, dim, L = u[0]
    N = A[0][1]
    want = {"delta": (bsz, dim, L), "A": (dim, N), "B": (bsz, N, L), "C": (bsz, N, L),
            "z": (bsz, dim, L), "D": (dim,), "delta_bias": (dim,)}
    for name, m in (("delta", delta), ("A", A), ("B", B), ("C", C), ("z", z), ("D", D),
                    ("delta_bias", delta_bias)):
        if m is not None and tuple(m[0]) != want[name]:
            raise ValueError(f"selective_scan: {name} is {tuple(m[0])}, expected "
                             f"{want[name]}")
    _require_cuda(u, delta, A, B, C, D, z, delta_bias)
    return ctypes.byref(_abi.ScanDesc(bsz, dim, L, N, _abi.DTYPE_BF16, 1 if delta_softplus else 0))


def selective_scan(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    delta_bias: torch.Tensor | None = None,
    delta_softplus: bool = True,
) -> torch.Tensor:
    """Mamba-1 selective scan (selective_scan_fn argument order).

    u, delta, z [batch, dim, L] and B, C [batch, d_state, L] bf16; A
    [dim, d_state], D and delta_bias [dim] fp32. Returns y [batch, dim, L] bf16.
    """
    desc = _scan_plan(_meta(u), _meta(delta), _meta(A), _meta(B), _meta(C), _meta(D), _meta(z),
                      _meta(delta_bias), bool(delta_softplus))
    y = torch.empty_like(u)
    lib = load_library()
    _launch(lib, u.device, lib.neptune_selective_scan_fwd, desc, u.data_ptr(), delta.data_ptr(),
            A.data_ptr(), B.data_ptr(), C.data_ptr(), D.data_ptr() if D is not None else None,
            z.data_ptr() if z is not None else None,
            delta_bias.data_ptr() if delta_bias is not None else None, y.data_ptr())
    return y


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
