// abi.cpp — the extern "C" entry points of libneptune_hip.so
// (declared in include/neptune_hip.h).
//
// Every request is validated on the host before any HIP call, so argument
// errors are reported identically with or without a GPU. Failures return a
// status code and leave a message for neptune_last_error() on the calling
// thread; no C++ exception crosses the boundary. The reference reports the
// same classes of failure as RuntimeError (toolchain/runtime failure,
// src/neptune_mlir/translators/common.py:217-224) and NotImplementedError
// (valid input outside what the backend covers, common.py:187-197).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/neptune_hip.h"
#include "kernels.h"

using namespace neptune;

namespace {

thread_local std::string g_last_error;

neptune_status fail(neptune_status st, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return st;
}

neptune_status ok() {
  g_last_error.clear();
  return NEPTUNE_OK;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Resolve (batch, head, seq) strides; all-zero means contiguous.
bool resolve_strides(const int64_t in[3], int64_t heads, int64_t seq, int64_t dim,
                     int64_t out[3]) {
  if (in[0] == 0 && in[1] == 0 && in[2] == 0) {
    out[2] = dim;
    out[1] = seq * dim;
    out[0] = heads * seq * dim;
    return true;
  }
  for (int i = 0; i < 3; ++i) {
    if (in[i] <= 0) return false;
    out[i] = in[i];
  }
  return true;
}

neptune_status device_ready() {
  int n = 0;
  hipError_t e = hipGetDeviceCount(&n);
  if (e != hipSuccess || n <= 0)
    return fail(NEPTUNE_ERR_NO_DEVICE, "no HIP device available (%s)",
                e == hipSuccess ? "device count is 0" : hipGetErrorString(e));
  return NEPTUNE_OK;
}

neptune_status hip_result(hipError_t e, const char *what) {
  if (e != hipSuccess)
    return fail(NEPTUNE_ERR_HIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
  return ok();
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Split layout; identical rule in the CPU oracle (neptune_cpu_decode_layout).
void decode_layout(const neptune_decode_desc *d, int64_t *splits, int64_t *chunk) {
  int64_t want = d->num_splits;
  if (want <= 0) {
    int64_t groups = d->batch * d->heads_kv;
    want = cdiv(2048, groups);
    int64_t cap = cdiv(d->seq_kv, 256);
    if (want > cap) want = cap;
    if (want < 1) want = 1;
  }
  int64_t c = cdiv(cdiv(d->seq_kv, want), 64) * 64;
  *chunk = c;
  *splits = cdiv(d->seq_kv, c);
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// whether the byte ranges [a, a + na) and [b, b + nb) share a byte
bool overlaps(const void *a, size_t na, const void *b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return na && nb && x < y + nb && y < x + na;
}

neptune_status decode_check(const neptune_decode_desc *d) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: desc is NULL");
  if (d->batch <= 0 || d->heads_q <= 0 || d->heads_kv <= 0 || d->seq_kv <= 0 ||
      d->head_dim <= 0 || d->num_splits < 0 || d->scale_block < 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "decode: sizes must be positive (batch=%lld heads_q=%lld heads_kv=%lld "
                "seq_kv=%lld head_dim=%lld num_splits=%lld)",
                (long long)d->batch, (long long)d->heads_q, (long long)d->heads_kv,
                (long long)d->seq_kv, (long long)d->head_dim, (long long)d->num_splits);
  if (d->heads_q % d->heads_kv)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: heads_q (%lld) %% heads_kv (%lld) != 0",
                (long long)d->heads_q, (long long)d->heads_kv);
  if (d->q_dtype != NEPTUNE_DTYPE_BF16)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "decode: q_dtype must be BF16");
  if (d->kv_dtype != NEPTUNE_DTYPE_BF16 && d->kv_dtype != NEPTUNE_DTYPE_FP8_E4M3)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "decode: kv_dtype must be BF16 or FP8_E4M3");
  if (!(d->scale_log2 >= 0.0f) || !std::isfinite(d->scale_log2))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: scale_log2 must be finite and >= 0");
  return NEPTUNE_OK;
}

size_t decode_ws_bytes(const neptune_decode_desc *d, int64_t splits) {
  size_t rows = (size_t)d->batch * d->heads_q * splits;
  return align256(rows * d->head_dim * 4) + align256(rows * 2 * 4);
}

// the checks of an attention descriptor, and the launch it describes (no
// tensors)
neptune_status attn_resolve(const neptune_attn_desc *d, AttnLaunch *launch) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: desc is NULL");
  if (d->batch <= 0 || d->heads_q <= 0 || d->heads_kv <= 0 || d->seq_q <= 0 ||
      d->seq_kv <= 0 || d->head_dim <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "attn_fwd: sizes must be positive (batch=%lld heads_q=%lld heads_kv=%lld "
                "seq_q=%lld seq_kv=%lld head_dim=%lld)",
                (long long)d->batch, (long long)d->heads_q, (long long)d->heads_kv,
                (long long)d->seq_q, (long long)d->seq_kv, (long long)d->head_dim);
  if (d->heads_q % d->heads_kv)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: heads_q (%lld) %% heads_kv (%lld) != 0",
                (long long)d->heads_q, (long long)d->heads_kv);
  if (d->dtype != NEPTUNE_DTYPE_F32 && d->dtype != NEPTUNE_DTYPE_F16 &&
      d->dtype != NEPTUNE_DTYPE_BF16)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_fwd: dtype %d (need F32, F16 or BF16)",
                (int)d->dtype);
  if (!(d->scale_log2 >= 0.0f) || !std::isfinite(d->scale_log2))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: scale_log2 must be finite and >= 0");
  if (d->pipeline_stages < 0 || d->pipeline_stages > 3)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: pipeline_stages %d (need 0..3)",
                (int)d->pipeline_stages);
  if (d->k_dim_order != 0 && d->k_dim_order != 1)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: k_dim_order %d (need 0 or 1)",
                (int)d->k_dim_order);
  AttnLaunch &L = *launch;
  L.batch = d->batch; L.heads_q = d->heads_q; L.heads_kv = d->heads_kv;
  L.seq_q = d->seq_q; L.seq_kv = d->seq_kv; L.head_dim = d->head_dim;
  if (!resolve_strides(d->q_stride, d->heads_q, d->seq_q, d->head_dim, L.qs) ||
      !(d->k_dim_order ? resolve_strides(d->k_stride, d->heads_kv, d->head_dim, d->seq_kv, L.ks)
                       : resolve_strides(d->k_stride, d->heads_kv, d->seq_kv, d->head_dim, L.ks)) ||
      !resolve_strides(d->v_stride, d->heads_kv, d->seq_kv, d->head_dim, L.vs) ||
      !resolve_strides(d->o_stride, d->heads_q, d->seq_q, d->head_dim, L.os))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "attn_fwd: strides must be all zero (contiguous) or all positive");
  L.dtype = d->dtype;
  L.causal = d->causal ? 1 : 0;
  L.stages = d->pipeline_stages ? d->pipeline_stages : 2;
  L.k_dim_order = d->k_dim_order;
  L.scale_log2 = d->scale_log2 != 0.0f
                     ? d->scale_log2
                     : (float)(1.4426950408889634 / std::sqrt((double)d->head_dim));
  return NEPTUNE_OK;
}

// the attention entry points; ws: the caller has a workspace for the states of
// split keys
neptune_status attn_run(const neptune_attn_desc *d, const void *q, const void *k, const void *v,
                        void *o, float *lse, bool ws, void *workspace, size_t workspace_bytes,
                        void *stream) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: desc is NULL");
  if (!q || !k || !v || !o)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_fwd: q, k, v and o must be non-NULL");
  AttnLaunch L;
  neptune_status st = attn_resolve(d, &L);
  if (st != NEPTUNE_OK) return st;
  L.q = q; L.k = k; L.v = v; L.o = o; L.lse = lse;
  if (d->dtype != NEPTUNE_DTYPE_F32) {
    bool strides8 = true;
    for (int i = 0; i < 3; ++i)
      strides8 = strides8 && L.qs[i] % 8 == 0 && L.ks[i] % 8 == 0 && L.vs[i] % 8 == 0 &&
                 L.os[i] % 8 == 0;
    if (!strides8 || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
      return fail(NEPTUNE_ERR_UNSUPPORTED,
                  "attn_fwd: 16-bit tensors need 16-byte aligned base pointers and strides "
                  "that are multiples of 8 elements");
  }
  const char *why = "";
  if (!attn_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_fwd: %s", why);
  const AttnSplit split = attn_split(L, ws);
  if (split.bytes) {
    if (!workspace || workspace_bytes < split.bytes)
      return fail(NEPTUNE_ERR_WORKSPACE_TOO_SMALL, "attn_fwd: workspace %zu bytes, need %zu",
                  workspace ? workspace_bytes : (size_t)0, split.bytes);
    if (!aligned16(workspace))
      return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_fwd: workspace must be 16-byte aligned");
  }
  st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_attn_fwd(L, split, workspace, (hipStream_t)stream), "attn_fwd launch");
}

}  // namespace

extern "C" {

neptune_status neptune_hip_get_backend_info(neptune_backend_info *info) {
  if (!info) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "info is NULL");
  info->abi_version = NEPTUNE_HIP_ABI_VERSION;
  info->name = "NeptuneHTileHIP";
  info->gcn_arch = "gfx950";
  int v = -1;
  if (hipRuntimeGetVersion(&v) != hipSuccess) v = -1;
  info->hip_runtime_version = v;
  return ok();
}

const char *neptune_last_error(void) { return g_last_error.c_str(); }

int32_t neptune_device_count(void) {
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess) return 0;
  return n;
}

neptune_status neptune_attn_fwd(const neptune_attn_desc *d, const void *q, const void *k,
                                const void *v, void *o, float *lse, void *stream) {
  return attn_run(d, q, k, v, o, lse, false, nullptr, 0, stream);
}

neptune_status neptune_attn_workspace_bytes(const neptune_attn_desc *d, size_t *bytes) {
  if (!bytes) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_workspace_bytes: bytes is NULL");
  AttnLaunch L;
  neptune_status st = attn_resolve(d, &L);
  if (st != NEPTUNE_OK) return st;
  const char *why = "";
  if (!attn_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_fwd: %s", why);
  *bytes = attn_split(L, true).bytes;
  return ok();
}

neptune_status neptune_attn_fwd_ws(const neptune_attn_desc *d, const void *q, const void *k,
                                   const void *v, void *o, float *lse, void *workspace,
                                   size_t workspace_bytes, void *stream) {
  return attn_run(d, q, k, v, o, lse, true, workspace, workspace_bytes, stream);
}

neptune_status neptune_decode_workspace_bytes(const neptune_decode_desc *d, size_t *bytes) {
  if (!bytes) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode_workspace_bytes: bytes is NULL");
  neptune_status st = decode_check(d);
  if (st != NEPTUNE_OK) return st;
  int64_t splits, chunk;
  decode_layout(d, &splits, &chunk);
  *bytes = decode_ws_bytes(d, splits);
  return ok();
}

namespace {
// shared tail of the decode entry points (pk != nullptr: paged KV;
// scratch: the partials go to the library's static device scratch, and
// workspace / workspace_bytes are not used)
neptune_status decode_run(const neptune_decode_desc *d, const neptune_paged_kv_desc *pk,
                          const void *q, const void *k, const void *v, const float *k_scale,
                          const float *v_scale, const int32_t *block_table,
                          const int32_t *seq_lens, void *o, float *lse, bool scratch,
                          void *workspace, size_t workspace_bytes, void *stream) {
  if (!scratch && !workspace)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: workspace is NULL");
  int64_t splits, chunk;
  decode_layout(d, &splits, &chunk);
  const size_t need = decode_ws_bytes(d, splits);
  if (scratch && need > kDecodeScratchBytes)
    return fail(NEPTUNE_ERR_WORKSPACE_TOO_SMALL,
                "decode_noalloc: %lld splits x %lld rows need %zu bytes of partials, the static "
                "scratch holds %zu (use neptune_decode_splitk with a workspace)",
                (long long)splits, (long long)(d->batch * d->heads_q), need,
                kDecodeScratchBytes);
  if (!scratch && workspace_bytes < need)
    return fail(NEPTUNE_ERR_WORKSPACE_TOO_SMALL, "decode: workspace %zu bytes, need %zu",
                workspace_bytes, need);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || (!scratch && !aligned16(workspace)))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "decode: q, k, v and workspace must be 16-byte aligned");
  DecodeLaunch L;
  L.q = q; L.k = k; L.v = v; L.k_scale = k_scale; L.v_scale = v_scale;
  L.o = o; L.lse = lse;
  L.batch = d->batch; L.heads_q = d->heads_q; L.heads_kv = d->heads_kv;
  L.seq_kv = d->seq_kv; L.head_dim = d->head_dim;
  L.splits = splits; L.chunk = chunk;
  L.scale_block = d->scale_block > 0 ? d->scale_block : 64;
  L.n_scale_blocks = cdiv(d->seq_kv, L.scale_block);
  L.kv_dtype = d->kv_dtype;
  L.scale_log2 = d->scale_log2 != 0.0f
                     ? d->scale_log2
                     : (float)(1.4426950408889634 / std::sqrt((double)d->head_dim));
  if (pk) {
    L.block_table = block_table;
    L.seq_lens = seq_lens;
    L.page_size = pk->page_size;
    L.max_pages = pk->max_pages;
    L.num_pages = pk->num_pages;
    for (int i = 0; i < 3; ++i) {
      L.k_pstride[i] = pk->k_stride[i];
      L.v_pstride[i] = pk->v_stride[i];
    }
  }
  const char *why = "";
  if (!decode_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "decode: %s", why);
  neptune_status st = device_ready();
  if (st != NEPTUNE_OK) return st;
  if (scratch) {
    st = hip_result(decode_scratch((hipStream_t)stream, &workspace), "decode_noalloc: scratch address");
    if (st != NEPTUNE_OK) return st;
  }
  const size_t rows = (size_t)d->batch * d->heads_q * splits;
  L.part_o = (float *)workspace;
  L.part_ml = (float *)((char *)workspace + align256(rows * d->head_dim * 4));
  return hip_result(launch_decode(L, (hipStream_t)stream), "decode launch");
}
}  // namespace

neptune_status neptune_decode_splitk(const neptune_decode_desc *d, const void *q,
                                     const void *k, const void *v, const float *k_scale,
                                     const float *v_scale, void *o, float *lse,
                                     void *workspace, size_t workspace_bytes, void *stream) {
  neptune_status st = decode_check(d);
  if (st != NEPTUNE_OK) return st;
  if (!q || !k || !v || !o)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: q, k, v and o must be non-NULL");
  const bool fp8 = d->kv_dtype == NEPTUNE_DTYPE_FP8_E4M3;
  if (fp8 && (!k_scale || !v_scale))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode: fp8 KV needs k_scale and v_scale");
  return decode_run(d, nullptr, q, k, v, k_scale, v_scale, nullptr, nullptr, o, lse, false,
                    workspace, workspace_bytes, stream);
}

neptune_status neptune_decode_splitk_noalloc(const neptune_decode_desc *d, const void *q,
                                             const void *k, const void *v,
                                             const float *k_scale, const float *v_scale,
                                             void *o, float *lse, void *stream) {
  neptune_status st = decode_check(d);
  if (st != NEPTUNE_OK) return st;
  if (!q || !k || !v || !o)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode_noalloc: q, k, v and o must be non-NULL");
  if (d->kv_dtype == NEPTUNE_DTYPE_FP8_E4M3 && (!k_scale || !v_scale))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode_noalloc: fp8 KV needs k_scale and v_scale");
  return decode_run(d, nullptr, q, k, v, k_scale, v_scale, nullptr, nullptr, o, lse, true,
                    nullptr, 0, stream);
}

namespace {
// checks shared by the two paged entry points; esize: bytes per pool element
neptune_status paged_check(const char *fn, const neptune_decode_desc *d,
                           const neptune_paged_kv_desc *pk, const void *q, const void *k_pages,
                           const void *v_pages, const int32_t *block_table,
                           const int32_t *seq_lens, const void *o, int64_t esize) {
  neptune_status st = decode_check(d);
  if (st != NEPTUNE_OK) return st;
  if (!pk) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: pages desc is NULL", fn);
  if (!q || !k_pages || !v_pages || !block_table || !seq_lens || !o)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: q, pools, block_table, seq_lens and o must be non-NULL", fn);
  if (pk->num_pages <= 0 || pk->page_size <= 0 || pk->max_pages <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: num_pages, page_size and max_pages must be positive", fn);
  if (pk->max_pages * pk->page_size < d->seq_kv)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: max_pages (%lld) * page_size (%lld) < seq_kv (%lld)", fn,
                (long long)pk->max_pages, (long long)pk->page_size, (long long)d->seq_kv);
  // 16-byte copy units: strides in whole units
  const int64_t unit = 16 / esize;
  for (int i = 0; i < 3; ++i)
    if (pk->k_stride[i] <= 0 || pk->v_stride[i] <= 0 || pk->k_stride[i] % unit ||
        pk->v_stride[i] % unit)
      return fail(NEPTUNE_ERR_UNSUPPORTED,
                  "%s: pool strides must be positive multiples of %lld elements", fn,
                  (long long)unit);
  return NEPTUNE_OK;
}
}  // namespace

neptune_status neptune_decode_paged(const neptune_decode_desc *d, const neptune_paged_kv_desc *pk,
                                    const void *q, const void *k_pages, const void *v_pages,
                                    const int32_t *block_table, const int32_t *seq_lens, void *o,
                                    float *lse, void *workspace, size_t workspace_bytes,
                                    void *stream) {
  neptune_status st =
      paged_check("decode_paged", d, pk, q, k_pages, v_pages, block_table, seq_lens, o, 2);
  if (st != NEPTUNE_OK) return st;
  if (d->kv_dtype != NEPTUNE_DTYPE_BF16)
    return fail(NEPTUNE_ERR_UNSUPPORTED,
                "decode_paged: kv_dtype must be BF16 (fp8 pools: neptune_decode_paged_fp8)");
  return decode_run(d, pk, q, k_pages, v_pages, nullptr, nullptr, block_table, seq_lens, o, lse,
                    false, workspace, workspace_bytes, stream);
}

neptune_status neptune_decode_paged_fp8(const neptune_decode_desc *d,
                                        const neptune_paged_kv_desc *pk, const void *q,
                                        const uint8_t *k_pages, const uint8_t *v_pages,
                                        const float *k_scales, const float *v_scales,
                                        const int32_t *block_table, const int32_t *seq_lens,
                                        void *o, float *lse, void *workspace,
                                        size_t workspace_bytes, void *stream) {
  neptune_status st =
      paged_check("decode_paged_fp8", d, pk, q, k_pages, v_pages, block_table, seq_lens, o, 1);
  if (st != NEPTUNE_OK) return st;
  if (d->kv_dtype != NEPTUNE_DTYPE_FP8_E4M3)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "decode_paged_fp8: kv_dtype must be FP8_E4M3");
  if (!k_scales || !v_scales)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "decode_paged_fp8: k_scales and v_scales must be non-NULL");
  if (d->scale_block != 0 && d->scale_block != pk->page_size)
    return fail(NEPTUNE_ERR_UNSUPPORTED,
                "decode_paged_fp8: one scale per page: scale_block must be 0 or page_size "
                "(%lld), not %lld",
                (long long)pk->page_size, (long long)d->scale_block);
  neptune_decode_desc dd = *d;
  dd.scale_block = pk->page_size;
  return decode_run(&dd, pk, q, k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, o,
                    lse, false, workspace, workspace_bytes, stream);
}

neptune_status neptune_kv_quantize_fp8(int64_t batch, int64_t heads_kv, int64_t seq_kv,
                                       int64_t head_dim, int64_t scale_block, const void *src,
                                       uint8_t *codes, float *scales, void *stream) {
  if (!src || !codes || !scales)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "kv_quantize: src, codes and scales must be non-NULL");
  if (batch <= 0 || heads_kv <= 0 || seq_kv <= 0 || head_dim <= 0 || scale_block < 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "kv_quantize: sizes must be positive");
  if (batch * heads_kv * cdiv(seq_kv, scale_block > 0 ? scale_block : 64) > ((int64_t)1 << 31) - 1 ||
      seq_kv * head_dim > ((int64_t)1 << 31) - 1)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "kv_quantize: shape too large for one launch");
  QuantLaunch L;
  L.src = src; L.codes = codes; L.scales = scales;
  L.batch = batch; L.heads_kv = heads_kv; L.seq_kv = seq_kv; L.head_dim = head_dim;
  L.scale_block = scale_block > 0 ? scale_block : 64;
  L.n_scale_blocks = cdiv(seq_kv, L.scale_block);
  neptune_status st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_kv_quantize(L, (hipStream_t)stream), "kv_quantize launch");
}

namespace {

bool is_float(int32_t dtype, bool f32) {
  return dtype == NEPTUNE_DTYPE_F16 || dtype == NEPTUNE_DTYPE_BF16 ||
         (f32 && dtype == NEPTUNE_DTYPE_F32);
}

// Bytes from the first element to past the last of a [sizes.., row] tensor;
// 0 where that passes 2^60
size_t span(const int64_t *sizes, const int64_t *strides, int n, int64_t row, int64_t esize) {
  int64_t at = row, step;
  for (int i = 0; i < n; ++i)
    if (__builtin_mul_overflow(sizes[i] - 1, strides[i], &step) ||
        __builtin_add_overflow(at, step, &at))
      return 0;
  return at > ((int64_t)1 << 60) / esize ? 0 : (size_t)(at * esize);
}

// A strided tensor of an entry point: its rows' strides resolved (zero:
// contiguous), their sizes, its bytes
struct Strided {
  const char *name;
  const void *p;
  int64_t stride[3], size[3];
  int n;
  int64_t dim, esize;
  size_t bytes;
};

// [sizes[0], sizes[1], sizes[2], dim] with `n` strides in the descriptor's order
neptune_status resolve(const char *fn, const char *name, const void *p, const int64_t *in,
                       const int64_t *sizes, int n, int64_t dim, int64_t esize, Strided *t) {
  t->name = name;
  t->p = p;
  t->n = n;
  t->dim = dim;
  t->esize = esize;
  for (int i = 0; i < n; ++i) t->size[i] = sizes[i];
  if (!p) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: %s must be non-NULL", fn, name);
  bool zero = true;
  for (int i = 0; i < n; ++i) zero = zero && in[i] == 0;
  int64_t run = dim;
  for (int i = n - 1; i >= 0; --i) {
    t->stride[i] = zero ? run : in[i];
    if (sizes[i] == 1) {  // no step is taken along it
      t->stride[i] = 16 / esize;
      continue;
    }
    if (zero && __builtin_mul_overflow(run, sizes[i], &run))
      return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s is too large", fn, name);
    if (t->stride[i] <= 0)
      return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                  "%s: strides must be all zero (contiguous) or all positive", fn);
    if (t->stride[i] % (16 / esize))
      return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: strides must be multiples of 16 bytes", fn);
  }
  if (!aligned16(p))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s must be 16-byte aligned", fn, name);
  t->bytes = span(sizes, t->stride, n, dim, esize);
  if (!t->bytes) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s is too large", fn, name);
  return NEPTUNE_OK;
}

// Whether rows of two tensors share a byte. Their spans may cross where they do
// not: heads of q, k and v side by side in one projection. The distance of two
// rows is delta + sum of x_j step_j with x_j in [lo_j, hi_j] (a step that both
// tensors take counts once); largest step first, few x_j leave one that the
// smaller steps can still bring into (-b's row, a's row). Where strides are so
// tangled that it takes thousands of tries, the answer is yes. (Both span at most
// 2^60 bytes and cross, so 64 bits hold every sum.)
struct Steps {
  int n = 0, tries = 0;
  int64_t step[6], lo[6], hi[6];
  int64_t below, above;  // the open interval
  void add(int64_t by, int64_t first, int64_t last) {
    int i = 0;
    while (i < n && step[i] > by) ++i;
    if (i == n || step[i] != by) {
      for (int j = n++; j > i; --j) step[j] = step[j - 1], lo[j] = lo[j - 1], hi[j] = hi[j - 1];
      step[i] = by;
      lo[i] = hi[i] = 0;
    }
    lo[i] += first;
    hi[i] += last;
  }
  bool reach(int j, int64_t at) {
    if (++tries > 4096) return true;
    if (j == n) return at > below && at < above;
    int64_t least = 0, most = 0;  // of the smaller steps
    for (int i = j + 1; i < n; ++i) least += lo[i] * step[i], most += hi[i] * step[i];
    const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    // at + x step + [least, most] meets [below + 1, above - 1]
    const int64_t first = -floor_div(at + most - below - 1, step[j]);
    const int64_t last = floor_div(above - 1 - least - at, step[j]);
    for (int64_t x = first > lo[j] ? first : lo[j]; x <= last && x <= hi[j]; ++x)
      if (reach(j + 1, at + x * step[j])) return true;
    return false;
  }
};

bool meet(const Strided &a, const Strided &b) {
  if (!overlaps(a.p, a.bytes, b.p, b.bytes)) return false;
  Steps s;
  for (int i = 0; i < a.n; ++i)
    if (a.size[i] > 1) s.add(a.stride[i] * a.esize, 1 - a.size[i], 0);
  for (int i = 0; i < b.n; ++i)
    if (b.size[i] > 1) s.add(b.stride[i] * b.esize, 0, b.size[i] - 1);
  s.below = -(b.dim * b.esize);
  s.above = a.dim * a.esize;
  return s.reach(0, (int64_t)((uintptr_t)b.p - (uintptr_t)a.p));
}

// out must share no byte with in
neptune_status apart(const char *fn, const Strided &out, const Strided &in) {
  if (meet(out, in))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: %s overlaps %s", fn, out.name, in.name);
  return NEPTUNE_OK;
}

bool same_place(const Strided &a, const Strided &b, int n) {
  bool same = a.p == b.p;
  for (int i = 0; i < n; ++i) same = same && a.stride[i] == b.stride[i];
  return same;
}

// what the rotation and norm take beside their tensors
neptune_status rope_check(const char *fn, int64_t head_dim, int64_t rot_dim, int64_t table_len,
                          const float *cos, const float *sin, const float *q_weight,
                          const float *k_weight, int32_t interleaved, float eps) {
  if (rot_dim < 0 || rot_dim > head_dim || (rot_dim > 0 && table_len <= 0))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: rot_dim %lld (at most head_dim %lld) over tables of %lld rows", fn,
                (long long)rot_dim, (long long)head_dim, (long long)table_len);
  if (rot_dim > 0 && (!cos || !sin))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: cos and sin must be non-NULL", fn);
  if (interleaved != 0 && interleaved != 1)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: interleaved must be 0 or 1", fn);
  if (!(eps >= 0.0f) || !std::isfinite(eps))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: eps must be finite and >= 0", fn);
  if (!aligned16(cos) || !aligned16(sin) || !aligned16(q_weight) || !aligned16(k_weight))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: tables and weights must be 16-byte aligned", fn);
  return NEPTUNE_OK;
}

// the pools of a ragged batch's entry points
// (mx, scales: entry points that take MXFP4 pools)
neptune_status pools_check(const char *fn, const neptune_paged_kv_desc *pk, const void *k_pages,
                           const void *v_pages, const void *k_scales, const void *v_scales,
                           const int32_t *block_table, const int32_t *cu_seqlens,
                           const int32_t *seq_lens, int64_t tokens, int64_t batch,
                           int64_t heads_kv, int64_t head_dim, int32_t kv_dtype, Strided pools[2],
                           const neptune_mx_desc *mx = nullptr, Strided *scales = nullptr) {
  if (!pk) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: pages desc is NULL", fn);
  if (!block_table || !seq_lens)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: block_table and seq_lens must be non-NULL", fn);
  if (pk->num_pages <= 0 || pk->page_size <= 0 || pk->max_pages <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: num_pages, page_size and max_pages must be positive", fn);
  if (!cu_seqlens && tokens != batch)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: without cu_seqlens a sequence has one new token: tokens %lld, batch %lld", fn,
                (long long)tokens, (long long)batch);
  const bool fp8 = kv_dtype == NEPTUNE_DTYPE_FP8_E4M3, mx4 = kv_dtype == NEPTUNE_DTYPE_MXFP4;
  if (fp8 && (!k_scales || !v_scales))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: E4M3 pools need k_scales and v_scales", fn);
  if (mx4 && (!mx || !k_scales || !v_scales))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: MXFP4 pools need mx, k_scales and v_scales", fn);
  if (mx4 && head_dim % 32)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: MXFP4 pools need a head_dim of whole 32s", fn);
  const int64_t sizes[3] = {pk->num_pages, heads_kv, pk->page_size};
  const struct { const char *name; const void *p; const int64_t *stride; } in[2] = {
      {"k_pages", k_pages, pk->k_stride}, {"v_pages", v_pages, pk->v_stride}};
  for (int i = 0; i < 2; ++i) {
    for (int j = 0; j < 3; ++j)
      if (in[i].stride[j] <= 0)
        return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: pool strides must be positive", fn);
    neptune_status st = resolve(fn, in[i].name, in[i].p, in[i].stride, sizes, 3,
                                mx4 ? head_dim / 2 : head_dim, fp8 || mx4 ? 1 : 2, &pools[i]);
    if (st != NEPTUNE_OK) return st;
  }
  if (!mx4) return NEPTUNE_OK;
  // the scales' pools: whole rows of head_dim / 32 bytes
  const int64_t row = head_dim / 32;
  for (int i = 0; i < 2; ++i) {
    Strided &t = scales[i];
    const int64_t *stride = i ? mx->v_stride : mx->k_stride;
    t = {i ? "v_scales" : "k_scales", i ? v_scales : k_scales, {}, {}, 3, row, 1, 0};
    for (int j = 0; j < 3; ++j) {
      t.size[j] = sizes[j];
      t.stride[j] = sizes[j] == 1 ? row : stride[j];  // no step is taken along it
      if (t.stride[j] <= 0)
        return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: the scales' strides must be positive", fn);
      if (t.stride[j] % row || (uintptr_t)t.p % row)
        return fail(NEPTUNE_ERR_UNSUPPORTED,
                    "%s: %s: base and strides must be multiples of head_dim / 32 bytes", fn, t.name);
    }
    t.bytes = span(t.size, t.stride, 3, row, 1);
    if (!t.bytes) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s is too large", fn, t.name);
  }
  return NEPTUNE_OK;
}

Pool pool_of(int32_t kv_dtype) {
  return kv_dtype == NEPTUNE_DTYPE_MXFP4 ? MXFP4 : kv_dtype == NEPTUNE_DTYPE_FP8_E4M3 ? E4M3 : WIDE;
}

// the checks of an attn_paged descriptor, and the launch it describes (no tensors)
neptune_status attn_paged_resolve(const neptune_attn_paged_desc *d, PagedAttnLaunch *L) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_paged: desc is NULL");
  if (d->tokens <= 0 || d->batch <= 0 || d->heads_q <= 0 || d->heads_kv <= 0 || d->head_dim <= 0 ||
      d->seq_kv <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "attn_paged: sizes must be positive (tokens=%lld batch=%lld heads_q=%lld "
                "heads_kv=%lld head_dim=%lld seq_kv=%lld)",
                (long long)d->tokens, (long long)d->batch, (long long)d->heads_q,
                (long long)d->heads_kv, (long long)d->head_dim, (long long)d->seq_kv);
  if (d->heads_q % d->heads_kv)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_paged: heads_q (%lld) %% heads_kv (%lld) != 0",
                (long long)d->heads_q, (long long)d->heads_kv);
  if (!is_float(d->dtype, false))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_paged: dtype must be F16 or BF16");
  if (d->kv_dtype != d->dtype && pool_of(d->kv_dtype) == WIDE)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_paged: kv_dtype must be dtype, FP8_E4M3 or MXFP4");
  if (!(d->scale_log2 >= 0.0f) || !std::isfinite(d->scale_log2))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_paged: scale_log2 must be finite and >= 0");
  *L = PagedAttnLaunch();
  L->tokens = d->tokens; L->batch = d->batch; L->heads_q = d->heads_q; L->heads_kv = d->heads_kv;
  L->head_dim = d->head_dim; L->seq_kv = d->seq_kv; L->dtype = d->dtype;
  L->pool = pool_of(d->kv_dtype);
  L->page_size = 16;
  L->scale_log2 = d->scale_log2 != 0.0f
                      ? d->scale_log2
                      : (float)(1.4426950408889634 / std::sqrt((double)d->head_dim));
  return NEPTUNE_OK;
}

}  // namespace

neptune_status neptune_qk_norm_rope(const neptune_rope_desc *d, const void *q, const void *k,
                                    const float *q_weight, const float *k_weight, const float *cos,
                                    const float *sin, const int32_t *positions, void *qo, void *ko,
                                    void *stream) {
  const char *fn = "qk_norm_rope";
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: desc is NULL", fn);
  if (d->batch <= 0 || d->heads_q <= 0 || d->heads_kv <= 0 || d->seq <= 0 || d->head_dim <= 0 ||
      d->rot_dim <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: sizes must be positive (batch=%lld heads_q=%lld heads_kv=%lld seq=%lld "
                "head_dim=%lld rot_dim=%lld)",
                fn, (long long)d->batch, (long long)d->heads_q, (long long)d->heads_kv,
                (long long)d->seq, (long long)d->head_dim, (long long)d->rot_dim);
  if (!is_float(d->dtype, true))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: dtype must be F32, F16 or BF16", fn);
  if (!positions) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: positions must be non-NULL", fn);
  neptune_status st = rope_check(fn, d->head_dim, d->rot_dim, d->table_len, cos, sin, q_weight,
                                 k_weight, d->interleaved, d->eps);
  if (st != NEPTUNE_OK) return st;
  const int64_t esize = d->dtype == NEPTUNE_DTYPE_F32 ? 4 : 2;
  const int64_t sq[3] = {d->batch, d->heads_q, d->seq}, sk[3] = {d->batch, d->heads_kv, d->seq};
  Strided in[2], out[2];
  if ((st = resolve(fn, "q", q, d->q_stride, sq, 3, d->head_dim, esize, &in[0])) != NEPTUNE_OK ||
      (st = resolve(fn, "k", k, d->k_stride, sk, 3, d->head_dim, esize, &in[1])) != NEPTUNE_OK ||
      (st = resolve(fn, "qo", qo, d->qo_stride, sq, 3, d->head_dim, esize, &out[0])) != NEPTUNE_OK ||
      (st = resolve(fn, "ko", ko, d->ko_stride, sk, 3, d->head_dim, esize, &out[1])) != NEPTUNE_OK)
    return st;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (!(i == j && same_place(out[i], in[i], 3)) &&
          (st = apart(fn, out[i], in[j])) != NEPTUNE_OK)
        return st;
  if ((st = apart(fn, out[0], out[1])) != NEPTUNE_OK) return st;
  RopeLaunch L;
  L.q = q; L.k = k; L.qo = qo; L.ko = ko;
  L.q_weight = q_weight; L.k_weight = k_weight; L.cos = cos; L.sin = sin; L.positions = positions;
  L.batch = d->batch; L.heads_q = d->heads_q; L.heads_kv = d->heads_kv; L.seq = d->seq;
  L.head_dim = d->head_dim; L.rot_dim = d->rot_dim; L.table_len = d->table_len;
  for (int i = 0; i < 3; ++i) {
    L.qs[i] = in[0].stride[i]; L.ks[i] = in[1].stride[i];
    L.qos[i] = out[0].stride[i]; L.kos[i] = out[1].stride[i];
  }
  L.dtype = d->dtype; L.interleaved = d->interleaved; L.eps = d->eps;
  const char *why = "";
  if (!rope_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s", fn, why);
  st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_rope(L, (hipStream_t)stream), "qk_norm_rope launch");
}

namespace {
// both append entry points (mx: into MXFP4 pools, whose scales are written)
neptune_status append_run(const char *fn, const neptune_append_desc *d,
                          const neptune_paged_kv_desc *pk, bool to_mx, const neptune_mx_desc *mx,
                          const void *k, const void *v, const void *q, const float *q_weight,
                          const float *k_weight, const float *cos, const float *sin,
                          const int32_t *block_table, const int32_t *cu_seqlens,
                          const int32_t *seq_lens, void *k_pages, void *v_pages,
                          const void *k_scales, const void *v_scales, void *qo, void *stream) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: desc is NULL", fn);
  if (d->tokens <= 0 || d->batch <= 0 || d->heads_q < 0 || d->heads_kv <= 0 || d->head_dim <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: sizes must be positive (tokens=%lld batch=%lld heads_q=%lld heads_kv=%lld "
                "head_dim=%lld)",
                fn, (long long)d->tokens, (long long)d->batch, (long long)d->heads_q,
                (long long)d->heads_kv, (long long)d->head_dim);
  if (!is_float(d->dtype, false))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: dtype must be F16 or BF16", fn);
  if (to_mx ? d->kv_dtype != NEPTUNE_DTYPE_MXFP4
            : d->kv_dtype != d->dtype && d->kv_dtype != NEPTUNE_DTYPE_FP8_E4M3)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: kv_dtype must be %s", fn,
                to_mx ? "MXFP4" : "dtype or FP8_E4M3 (MXFP4: neptune_kv_append_paged_mx)");
  neptune_status st = rope_check(fn, d->head_dim, d->rot_dim, d->table_len, cos, sin, q_weight,
                                 k_weight, d->interleaved, d->eps);
  if (st != NEPTUNE_OK) return st;
  Strided pools[4], in[3], out;  // pools: K, V, and MXFP4's scales
  const int n_pools = to_mx ? 4 : 2;
  st = pools_check(fn, pk, k_pages, v_pages, k_scales, v_scales, block_table, cu_seqlens, seq_lens,
                   d->tokens, d->batch, d->heads_kv, d->head_dim, d->kv_dtype, pools, mx, pools + 2);
  if (st != NEPTUNE_OK) return st;
  const int64_t sq[2] = {d->tokens, d->heads_q}, sk[2] = {d->tokens, d->heads_kv};
  const int n_in = d->heads_q ? 3 : 2;
  if ((st = resolve(fn, "k", k, d->k_stride, sk, 2, d->head_dim, 2, &in[0])) != NEPTUNE_OK ||
      (st = resolve(fn, "v", v, d->v_stride, sk, 2, d->head_dim, 2, &in[1])) != NEPTUNE_OK)
    return st;
  if (d->heads_q) {
    if ((st = resolve(fn, "q", q, d->q_stride, sq, 2, d->head_dim, 2, &in[2])) != NEPTUNE_OK ||
        (st = resolve(fn, "qo", qo, d->qo_stride, sq, 2, d->head_dim, 2, &out)) != NEPTUNE_OK)
      return st;
    for (int j = 0; j < 3; ++j)
      if (!(j == 2 && same_place(out, in[2], 2)) && (st = apart(fn, out, in[j])) != NEPTUNE_OK)
        return st;
    for (int i = 0; i < n_pools; ++i)
      if ((st = apart(fn, out, pools[i])) != NEPTUNE_OK) return st;
  }
  for (int i = 0; i < n_pools; ++i) {
    for (int j = 0; j < n_in; ++j)
      if ((st = apart(fn, pools[i], in[j])) != NEPTUNE_OK) return st;
    for (int j = 0; j < i; ++j)
      if ((st = apart(fn, pools[j], pools[i])) != NEPTUNE_OK) return st;
  }
  RopeLaunch L;
  L.append = true;
  L.pool = pool_of(d->kv_dtype);
  L.q = q; L.k = k; L.v = v; L.qo = qo; L.ko = k_pages; L.vo = v_pages;
  L.q_weight = q_weight; L.k_weight = k_weight; L.cos = cos; L.sin = sin;
  L.cu_seqlens = cu_seqlens; L.seq_lens = seq_lens; L.block_table = block_table;
  if (to_mx) {
    L.k_bytes = (uint8_t *)k_scales;
    L.v_bytes = (uint8_t *)v_scales;
  } else {
    L.k_scales = (const float *)k_scales;
    L.v_scales = (const float *)v_scales;
  }
  L.batch = 1; L.seq = d->tokens; L.heads_q = d->heads_q; L.heads_kv = d->heads_kv;
  L.head_dim = d->head_dim; L.rot_dim = d->rot_dim; L.table_len = d->table_len;
  L.sequences = d->batch; L.page_size = pk->page_size; L.max_pages = pk->max_pages;
  L.num_pages = pk->num_pages;
  // (token, head) -> (batch, head, seq)
  const auto rows = [](const Strided &t, int64_t *s) {
    s[0] = 0;
    s[1] = t.stride[1];
    s[2] = t.stride[0];
  };
  rows(in[0], L.ks);
  rows(in[1], L.vs);
  if (d->heads_q) {
    rows(in[2], L.qs);
    rows(out, L.qos);
  }
  for (int i = 0; i < 3; ++i) {
    L.kos[i] = pools[0].stride[i];
    L.vos[i] = pools[1].stride[i];
    if (to_mx) {
      L.kss[i] = pools[2].stride[i];
      L.vss[i] = pools[3].stride[i];
    }
  }
  L.dtype = d->dtype; L.interleaved = d->interleaved; L.eps = d->eps;
  const char *why = "";
  if (!rope_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s", fn, why);
  st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_rope(L, (hipStream_t)stream), "kv_append_paged launch");
}
}  // namespace

neptune_status neptune_kv_append_paged(const neptune_append_desc *d,
                                       const neptune_paged_kv_desc *pk, const void *k,
                                       const void *v, const void *q, const float *q_weight,
                                       const float *k_weight, const float *cos, const float *sin,
                                       const int32_t *block_table, const int32_t *cu_seqlens,
                                       const int32_t *seq_lens, void *k_pages, void *v_pages,
                                       const float *k_scales, const float *v_scales, void *qo,
                                       void *stream) {
  return append_run("kv_append_paged", d, pk, false, nullptr, k, v, q, q_weight, k_weight, cos, sin,
                    block_table, cu_seqlens, seq_lens, k_pages, v_pages, k_scales, v_scales, qo,
                    stream);
}

neptune_status neptune_kv_append_paged_mx(const neptune_append_desc *d,
                                          const neptune_paged_kv_desc *pk,
                                          const neptune_mx_desc *mx, const void *k, const void *v,
                                          const void *q, const float *q_weight,
                                          const float *k_weight, const float *cos, const float *sin,
                                          const int32_t *block_table, const int32_t *cu_seqlens,
                                          const int32_t *seq_lens, void *k_pages, void *v_pages,
                                          uint8_t *k_scales, uint8_t *v_scales, void *qo,
                                          void *stream) {
  return append_run("kv_append_paged_mx", d, pk, true, mx, k, v, q, q_weight, k_weight, cos, sin,
                    block_table, cu_seqlens, seq_lens, k_pages, v_pages, k_scales, v_scales, qo,
                    stream);
}

neptune_status neptune_kv_read_paged(const neptune_kv_read_desc *d, const neptune_paged_kv_desc *pk,
                                     const neptune_mx_desc *mx, const void *k_pages,
                                     const void *v_pages, const void *k_scales,
                                     const void *v_scales, const int32_t *block_table,
                                     const int32_t *cu_seqlens, const int32_t *seq_lens, void *ko,
                                     void *vo, void *stream) {
  const char *fn = "kv_read_paged";
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: desc is NULL", fn);
  if (d->tokens <= 0 || d->batch <= 0 || d->heads_kv <= 0 || d->head_dim <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: sizes must be positive (tokens=%lld batch=%lld heads_kv=%lld head_dim=%lld)",
                fn, (long long)d->tokens, (long long)d->batch, (long long)d->heads_kv,
                (long long)d->head_dim);
  if (!is_float(d->dtype, true))
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: dtype must be F32, F16 or BF16", fn);
  if (!is_float(d->kv_dtype, false) && pool_of(d->kv_dtype) == WIDE)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: kv_dtype must be F16, BF16, FP8_E4M3 or MXFP4", fn);
  Strided pools[4], out[2];
  const Pool pool = pool_of(d->kv_dtype);
  neptune_status st = pools_check(fn, pk, k_pages, v_pages, k_scales, v_scales, block_table,
                                  cu_seqlens, seq_lens, d->tokens, d->batch, d->heads_kv,
                                  d->head_dim, d->kv_dtype, pools, mx, pools + 2);
  if (st != NEPTUNE_OK) return st;
  const int64_t sizes[2] = {d->tokens, d->heads_kv};
  const int64_t esize = d->dtype == NEPTUNE_DTYPE_F32 ? 4 : 2;
  if ((st = resolve(fn, "ko", ko, d->ko_stride, sizes, 2, d->head_dim, esize, &out[0])) != NEPTUNE_OK ||
      (st = resolve(fn, "vo", vo, d->vo_stride, sizes, 2, d->head_dim, esize, &out[1])) != NEPTUNE_OK ||
      (st = apart(fn, out[0], out[1])) != NEPTUNE_OK)
    return st;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < (pool == MXFP4 ? 4 : 2); ++j)
      if ((st = apart(fn, out[i], pools[j])) != NEPTUNE_OK) return st;
  if (pool == E4M3) {
    const size_t n = (size_t)pk->num_pages * (size_t)d->heads_kv * 4;
    for (int i = 0; i < 2; ++i)
      if (overlaps(out[i].p, out[i].bytes, k_scales, n) || overlaps(out[i].p, out[i].bytes, v_scales, n))
        return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: %s overlaps the scales", fn, out[i].name);
  }
  ReadLaunch L = {};
  L.k = k_pages; L.v = v_pages; L.k_scales = k_scales; L.v_scales = v_scales;
  L.block_table = block_table; L.cu_seqlens = cu_seqlens; L.seq_lens = seq_lens;
  L.ko = ko; L.vo = vo;
  L.tokens = d->tokens; L.sequences = d->batch; L.heads_kv = d->heads_kv; L.head_dim = d->head_dim;
  L.page_size = pk->page_size; L.max_pages = pk->max_pages; L.num_pages = pk->num_pages;
  for (int i = 0; i < 3; ++i) {
    L.kps[i] = pools[0].stride[i];
    L.vps[i] = pools[1].stride[i];
    if (pool == MXFP4) {
      L.kss[i] = pools[2].stride[i];
      L.vss[i] = pools[3].stride[i];
    }
  }
  for (int i = 0; i < 2; ++i) {
    L.kos[i] = out[0].stride[i];
    L.vos[i] = out[1].stride[i];
  }
  L.dtype = d->dtype; L.kv_dtype = d->kv_dtype; L.pool = pool;
  const char *why = "";
  if (!kv_read_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s", fn, why);
  st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_kv_read(L, (hipStream_t)stream), "kv_read_paged launch");
}

neptune_status neptune_attn_paged_workspace_bytes(const neptune_attn_paged_desc *d,
                                                  size_t *bytes) {
  if (!bytes)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "attn_paged_workspace_bytes: bytes is NULL");
  PagedAttnLaunch L;
  neptune_status st = attn_paged_resolve(d, &L);
  if (st != NEPTUNE_OK) return st;
  const char *why = "";
  if (!attn_paged_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_paged: %s", why);
  *bytes = attn_paged_bytes(L);
  return ok();
}

namespace {
// both entry points; the extended one takes mx, score and slopes
neptune_status attn_paged_run(const char *fn, const neptune_attn_paged_desc *d,
                              const neptune_paged_kv_desc *pk, const neptune_mx_desc *mx,
                              const neptune_score_desc *score, const void *q, const void *k_pages,
                              const void *v_pages, const void *k_scales, const void *v_scales,
                              const float *slopes, const int32_t *block_table,
                              const int32_t *cu_seqlens, const int32_t *seq_lens, void *o,
                              float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  PagedAttnLaunch L;
  neptune_status st = attn_paged_resolve(d, &L);
  if (st != NEPTUNE_OK) return st;
  if (score) {
    if (!(score->softcap >= 0.0f) || !std::isfinite(score->softcap))
      return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: softcap must be finite and >= 0", fn);
    // (its inverse and products with it stay ordinary numbers)
    if (score->softcap != 0.0f && (score->softcap < 0x1p-60f || score->softcap > 0x1p60f))
      return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: softcap must lie between 2^-60 and 2^60", fn);
    if (score->window < 0)
      return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "%s: window must be >= 0", fn);
    L.softcap = score->softcap;
    L.window = score->window;
  }
  L.slopes = slopes;
  Strided pools[4], tq, to;
  st = pools_check(fn, pk, k_pages, v_pages, k_scales, v_scales, block_table, cu_seqlens, seq_lens,
                   d->tokens, d->batch, d->heads_kv, d->head_dim, d->kv_dtype, pools, mx, pools + 2);
  if (st != NEPTUNE_OK) return st;
  if (pk->max_pages < cdiv(d->seq_kv, pk->page_size))
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "%s: max_pages (%lld) * page_size (%lld) < seq_kv (%lld)", fn,
                (long long)pk->max_pages, (long long)pk->page_size, (long long)d->seq_kv);
  const int64_t sizes[2] = {d->tokens, d->heads_q};
  if ((st = resolve(fn, "q", q, d->q_stride, sizes, 2, d->head_dim, 2, &tq)) != NEPTUNE_OK ||
      (st = resolve(fn, "o", o, d->o_stride, sizes, 2, d->head_dim, 2, &to)) != NEPTUNE_OK ||
      (st = apart(fn, to, tq)) != NEPTUNE_OK ||
      (st = apart(fn, to, pools[0])) != NEPTUNE_OK ||
      (st = apart(fn, to, pools[1])) != NEPTUNE_OK)
    return st;
  if (L.pool == MXFP4)
    for (int i = 2; i < 4; ++i)
      if ((st = apart(fn, to, pools[i])) != NEPTUNE_OK) return st;
  L.q = q; L.k = k_pages; L.v = v_pages; L.k_scales = k_scales; L.v_scales = v_scales;
  L.block_table = block_table; L.cu_seqlens = cu_seqlens; L.seq_lens = seq_lens;
  L.o = o; L.lse = lse; L.workspace = workspace;
  L.page_size = pk->page_size; L.max_pages = pk->max_pages; L.num_pages = pk->num_pages;
  for (int i = 0; i < 2; ++i) {
    L.qs[i] = tq.stride[i];
    L.os[i] = to.stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    L.kps[i] = pools[0].stride[i];
    L.vps[i] = pools[1].stride[i];
    if (L.pool == MXFP4) {
      L.kss[i] = pools[2].stride[i];
      L.vss[i] = pools[3].stride[i];
    }
  }
  const char *why = "";
  if (!attn_paged_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: %s", fn, why);
  const size_t need = attn_paged_bytes(L);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return fail(NEPTUNE_ERR_WORKSPACE_TOO_SMALL, "%s: workspace %zu bytes, need %zu", fn,
                  workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned16(workspace))
      return fail(NEPTUNE_ERR_UNSUPPORTED, "%s: workspace must be 16-byte aligned", fn);
  }
  st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_attn_paged(L, (hipStream_t)stream), "attn_paged launch");
}
}  // namespace

neptune_status neptune_attn_paged(const neptune_attn_paged_desc *d,
                                  const neptune_paged_kv_desc *pk, const void *q,
                                  const void *k_pages, const void *v_pages, const float *k_scales,
                                  const float *v_scales, const int32_t *block_table,
                                  const int32_t *cu_seqlens, const int32_t *seq_lens, void *o,
                                  float *lse, void *workspace, size_t workspace_bytes,
                                  void *stream) {
  if (d && d->kv_dtype == NEPTUNE_DTYPE_MXFP4)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "attn_paged: MXFP4 pools: neptune_attn_paged_ext");
  return attn_paged_run("attn_paged", d, pk, nullptr, nullptr, q, k_pages, v_pages, k_scales,
                        v_scales, nullptr, block_table, cu_seqlens, seq_lens, o, lse, workspace,
                        workspace_bytes, stream);
}

neptune_status neptune_attn_paged_ext(const neptune_attn_paged_desc *d,
                                      const neptune_paged_kv_desc *pk, const neptune_mx_desc *mx,
                                      const neptune_score_desc *score, const void *q,
                                      const void *k_pages, const void *v_pages,
                                      const void *k_scales, const void *v_scales,
                                      const float *slopes, const int32_t *block_table,
                                      const int32_t *cu_seqlens, const int32_t *seq_lens, void *o,
                                      float *lse, void *workspace, size_t workspace_bytes,
                                      void *stream) {
  return attn_paged_run("attn_paged_ext", d, pk, mx, score, q, k_pages, v_pages, k_scales, v_scales,
                        slopes, block_table, cu_seqlens, seq_lens, o, lse, workspace,
                        workspace_bytes, stream);
}


neptune_status neptune_selective_scan_fwd(const neptune_scan_desc *d, const void *u,
                                          const void *delta_raw, const float *A, const void *B,
                                          const void *C, const float *D, const void *z,
                                          const float *delta_bias, void *y, void *stream) {
  if (!d) return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "selective_scan: desc is NULL");
  if (!u || !delta_raw || !A || !B || !C || !y)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT,
                "selective_scan: u, delta, A, B, C and y must be non-NULL");
  if (d->batch <= 0 || d->dim <= 0 || d->seq_len <= 0 || d->d_state <= 0)
    return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "selective_scan: sizes must be positive");
  if (d->io_dtype != NEPTUNE_DTYPE_BF16)
    return fail(NEPTUNE_ERR_UNSUPPORTED, "selective_scan: io_dtype must be BF16");
  ScanLaunch L;
  L.u = u; L.delta_raw = delta_raw; L.B = B; L.C = C; L.z = z;
  L.A = A; L.D = D; L.delta_bias = delta_bias; L.y = y;
  L.batch = d->batch; L.dim = d->dim; L.seq_len = d->seq_len; L.d_state = d->d_state;
  L.delta_softplus = d->delta_softplus ? 1 : 0;
  const char *why = "";
  if (!scan_supported(L, &why)) return fail(NEPTUNE_ERR_UNSUPPORTED, "selective_scan: %s", why);
  // y is written while later steps of the inputs are still being read, and
  // holds per-chunk state before the outputs: it may share no input byte
  // (sizes are below 2^63 once scan_supported has passed)
  const size_t rows = (size_t)d->batch * (size_t)d->seq_len * 2;
  const size_t act = rows * (size_t)d->dim, bc = rows * (size_t)d->d_state;
  const struct { const void *p; size_t n; const char *name; } in[] = {
      {u, act, "u"},
      {delta_raw, act, "delta"},
      {z, z ? act : 0, "z"},
      {B, bc, "B"},
      {C, bc, "C"},
      {A, (size_t)d->dim * (size_t)d->d_state * 4, "A"},
      {D, D ? (size_t)d->dim * 4 : 0, "D"},
      {delta_bias, delta_bias ? (size_t)d->dim * 4 : 0, "delta_bias"}};
  for (const auto &t : in)
    if (overlaps(y, act, t.p, t.n))
      return fail(NEPTUNE_ERR_INVALID_ARGUMENT, "selective_scan: y overlaps %s", t.name);
  neptune_status st = device_ready();
  if (st != NEPTUNE_OK) return st;
  return hip_result(launch_selective_scan(L, (hipStream_t)stream), "selective_scan launch");
}

}  // extern "C"
