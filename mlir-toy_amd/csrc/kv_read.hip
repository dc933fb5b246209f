// kv_read.hip — tokens of a paged KV cache read back as rows, for gfx950.
//
// Not in the reference. Row r of a ragged batch is its sequence's token at the place
// that kv_append_paged gives such a row; its keys and values, all KV heads, come back
// as the values that the pool holds: 16-bit elements, E4M3 codes times their page's
// and head's scale, E2M1 codes times 2^(e - 127), e the byte of their 32 elements
// (255: NaN), formed in fp32 and rounded once to the rows' type.
//
// D / 8 lanes have a row, eight elements each: 4, 8 or 16 bytes in, 16 or 32 out. A group
// of lanes takes HPG heads of one token, keys and values, all loaded before the first is
// widened: the place (a search among the sequences, a length, a table's entry) is worked
// out once for 2 HPG rows.
//
// Bound: HBM, mostly the rows written; few rows by the chain of loads and the launch.
// Measured in a replayed graph (8 heads of 128 to bf16 rows): 65536 tokens from MXFP4
// 66 us (5.2 TB/s; a copy 5.0), 32768 from bf16 pages 41 (6.5), 16 tokens 3.6 (an empty
// copy 2.0).
#include <type_traits>

#include "device_common.h"
#include "kernels.h"
#include "paged_rows.h"

namespace neptune {
namespace {

constexpr int NT = 256;

struct ReadSide {
  const char *in;
  const uint8_t *bytes;  // MXFP4: scales
  const float *scales;   // E4M3
  char *out;
  int64_t ps[3], ss[3];  // (page, head, place), bytes
  int64_t os[2];         // (token, head), bytes
};

struct ReadArgs {
  ReadSide side[2];
  const int32_t *cu, *lens, *btab;
  int32_t tokens, B, heads, runs, ps, maxp, npages;
  uint32_t runs_inv;
  bool pool_f16;
};

// eight fp32 values as rows of O hold them
template <class O>
struct Out;
template <>
struct Out<float> {
  __device__ static inline void store(char *p, f32x4 a, f32x4 b) {
    *(f32x4 *)p = a;
    *(f32x4 *)(p + 16) = b;
  }
};
template <class E>
struct Out16 {
  __device__ static inline void store(char *p, f32x4 a, f32x4 b) {
    *(u32x4 *)p = u32x4{E::pack2(a[0], a[1]), E::pack2(a[2], a[3]), E::pack2(b[0], b[1]),
                        E::pack2(b[2], b[3])};
  }
};
template <>
struct Out<Bf16Tag> : Out16<Bf16Tag> {};
template <>
struct Out<F16Tag> : Out16<F16Tag> {};

template <class O, int D, int POOL, int HPG>
__global__ __launch_bounds__(NT) void kv_read(ReadArgs a) {
  constexpr int LPR = D / 8;
  typedef typename std::conditional<
      POOL == WIDE, u32x4, typename std::conditional<POOL == E4M3, u32x2, uint32_t>::type>::type raw;
  const int lane = threadIdx.x & 63, l = threadIdx.x % LPR;
  const uint32_t gid = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const int at = (int)divide(gid, a.runs, a.runs_inv), run = (int)gid - at * a.runs;
  const int tok = min(at, a.tokens - 1);
  bool write = at < a.tokens;
  int b = tok, left = 1;
  if (a.cu) {
    b = sequence_of<LPR>(a.cu, a.B, lane, tok, chunk_end(a.cu, a.B, lane));
    write = write && b < a.B && a.cu[0] <= tok;  // rows behind the last sequence stay as they were
    b = min(b, a.B - 1);
    left = a.cu[b + 1] - tok;
  }
  const int t = a.lens[b] - left;
  const int index = (int)((uint32_t)max(t, 0) / (uint32_t)a.ps), place = max(t, 0) - index * a.ps;
  int page = -1;
  if (t >= 0 && index < a.maxp) page = a.btab[(int64_t)b * a.maxp + index];
  const bool held = page >= 0 && page < a.npages;  // a row without a slot is zeros
  page = held ? page : 0;

  raw x[2][HPG];
  float scale[2][HPG];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const ReadSide &m = a.side[s];
      const int h = min(run + i * a.runs, a.heads - 1);
      const char *row = m.in + page * m.ps[0] + (held ? place : 0) * m.ps[2] + h * m.ps[1];
      x[s][i] = *(const raw *)(row + (int)sizeof(raw) * l);
      if constexpr (POOL == E4M3) scale[s][i] = m.scales[(int64_t)page * a.heads + h];
      if constexpr (POOL == MXFP4)
        scale[s][i] = __uint_as_float(
            (uint32_t)m.bytes[page * m.ss[0] + (held ? place : 0) * m.ss[2] + h * m.ss[1] + (l >> 2)]
            << 23);
    }
  if (!write) return;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const ReadSide &m = a.side[s];
      const int h = run + i * a.runs;
      if (h >= a.heads) continue;
      f32x4 lo = {0, 0, 0, 0}, hi = lo;
      if (held) {
        if constexpr (POOL == MXFP4) {
          const f32x2 c0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[s][i], scale[s][i], 0);
          const f32x2 c1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[s][i], scale[s][i], 1);
          const f32x2 c2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[s][i], scale[s][i], 2);
          const f32x2 c3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(x[s][i], scale[s][i], 3);
          lo = f32x4{c0[0], c0[1], c1[0], c1[1]};
          hi = f32x4{c2[0], c2[1], c3[0], c3[1]};
        } else if constexpr (POOL == E4M3) {
          const f32x2 c0 = e4m3x2_to_f32<false>(x[s][i][0]), c1 = e4m3x2_to_f32<true>(x[s][i][0]);
          const f32x2 c2 = e4m3x2_to_f32<false>(x[s][i][1]), c3 = e4m3x2_to_f32<true>(x[s][i][1]);
          lo = f32x4{c0[0], c0[1], c1[0], c1[1]} * scale[s][i];
          hi = f32x4{c2[0], c2[1], c3[0], c3[1]} * scale[s][i];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t e = (uint16_t)(x[s][i][j >> 1] >> (16 * (j & 1)));
            const float v = a.pool_f16 ? F16Tag::to_f32(e) : Bf16Tag::to_f32(e);
            if (j < 4)
              lo[j] = v;
            else
              hi[j - 4] = v;
          }
        }
      }
      constexpr int SIZE = std::is_same<O, float>::value ? 4 : 2;
      Out<O>::store(m.out + tok * m.os[0] + h * m.os[1] + 8 * SIZE * l, lo, hi);
    }
}

template <class O, int D, int POOL>
hipError_t launch_hpg(ReadArgs a, hipStream_t s) {
  constexpr int GPB = NT / (D / 8);  // groups of lanes per work-group
  auto go = [&](auto H) {
    constexpr int HPG = decltype(H)::value;
    a.runs = (a.heads + HPG - 1) / HPG;
    a.runs_inv = 0xffffffffu / (uint32_t)a.runs;
    const uint32_t blocks = (uint32_t)(((int64_t)a.tokens * a.runs + GPB - 1) / GPB);
    hipLaunchKernelGGL((kv_read<O, D, POOL, HPG>), dim3(blocks), dim3(NT), 0, s, a);
  };
  // Codes: several heads a group where that leaves two work-groups for every CU. 8 heads of
  // 128 from MXFP4, 65536, 16384, 4096 and 1024 tokens: 66, 16.5, 7.0 and 4.9 us, one head
  // a group 100, 19.4, 7.1 and 4.3; E4M3 74, 17.9, 7.2 and 5.0, one head 100, 19.6, 6.9 and
  // 4.3. 16-bit rows fill a group's loads alone: one head 22.0 and 7.3 for 16384 and 4096,
  // four 23.0 and 8.5.
  if constexpr (POOL != WIDE)
    if (a.heads > 1 && (int64_t)a.tokens * a.heads >= 2048 * GPB) {
      go(std::integral_constant<int, 4>{});
      return hipGetLastError();
    }
  go(std::integral_constant<int, 1>{});
  return hipGetLastError();
}

template <class O>
hipError_t launch_o(const ReadArgs &a, int64_t head_dim, Pool pool, hipStream_t s) {
  if (head_dim == 64)
    return pool == MXFP4  ? launch_hpg<O, 64, MXFP4>(a, s)
           : pool == E4M3 ? launch_hpg<O, 64, E4M3>(a, s)
                          : launch_hpg<O, 64, WIDE>(a, s);
  return pool == MXFP4  ? launch_hpg<O, 128, MXFP4>(a, s)
         : pool == E4M3 ? launch_hpg<O, 128, E4M3>(a, s)
                        : launch_hpg<O, 128, WIDE>(a, s);
}

}  // namespace

bool kv_read_supported(const ReadLaunch &L, const char **why) {
  if (L.head_dim != 64 && L.head_dim != 128) {
    *why = "the paged cache holds head_dim 64 or 128";
    return false;
  }
  // a group of lanes per (token, head) at most, counted in 32 bits; a dispatch
  // covers at most 2^32 - 1 work-items
  if (L.tokens > INT32_MAX || L.heads_kv > 1 << 20 ||
      L.tokens * L.heads_kv > ((int64_t)1 << 31) / (L.head_dim / 8)) {
    *why = "tokens * heads too large for one launch";
    return false;
  }
  if (L.num_pages > INT32_MAX || L.max_pages > INT32_MAX || L.page_size > INT32_MAX ||
      L.sequences > INT32_MAX - 64) {
    *why = "tables of 2^31 rows or pages and more";
    return false;
  }
  if (L.cu_seqlens && L.sequences > 1 << 16) {  // every group of lanes looks through them
    *why = "cu_seqlens of more than 65536 sequences";
    return false;
  }
  return true;
}

hipError_t launch_kv_read(const ReadLaunch &L, hipStream_t s) {
  ReadArgs a = {};
  const int64_t size = L.pool == WIDE ? 2 : 1, osize = L.dtype == 0 ? 4 : 2;
  const void *const in[2] = {L.k, L.v}, *const scales[2] = {L.k_scales, L.v_scales};
  void *const out[2] = {L.ko, L.vo};
  const int64_t *const ps[2] = {L.kps, L.vps}, *const ss[2] = {L.kss, L.vss},
                *const os[2] = {L.kos, L.vos};
  for (int i = 0; i < 2; ++i) {
    ReadSide &m = a.side[i];
    m.in = (const char *)in[i];
    m.bytes = (const uint8_t *)scales[i];
    m.scales = (const float *)scales[i];
    m.out = (char *)out[i];
    for (int j = 0; j < 3; ++j) {
      m.ps[j] = ps[i][j] * size;
      m.ss[j] = ss[i][j];
    }
    for (int j = 0; j < 2; ++j) m.os[j] = os[i][j] * osize;
  }
  a.cu = L.cu_seqlens; a.lens = L.seq_lens; a.btab = L.block_table;
  a.tokens = (int32_t)L.tokens;
  a.B = (int32_t)L.sequences;
  a.heads = (int32_t)L.heads_kv;
  a.ps = (int32_t)L.page_size;
  a.maxp = (int32_t)L.max_pages;
  a.npages = (int32_t)L.num_pages;
  a.pool_f16 = L.kv_dtype == 1;
  if (L.dtype == 0) return launch_o<float>(a, L.head_dim, L.pool, s);
  if (L.dtype == 1) return launch_o<F16Tag>(a, L.head_dim, L.pool, s);
  return launch_o<Bf16Tag>(a, L.head_dim, L.pool, s);
}

}  // namespace neptune
