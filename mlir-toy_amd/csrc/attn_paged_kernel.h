// attn_paged_kernel.h — the kernels of attention of a ragged batch of new tokens over a paged KV
// cache, for gfx950.
//
// Not in the reference; the recurrence is the HTile one
// (tests/data/flash_attention_htile.mlir:40-143) per query row:
//   O_r = sum_{j <= t} 2^(s_rj - m) v_j / l,   s_rj = q_r . k_j scale log2(e),
//   l = sum_j 2^(s_rj - m),   lse_r = (m + log2 l) ln 2,
// with t the row's place in its sequence. 16-bit pools, E4M3 codes with a scale per
// page and KV head, or MXFP4: E2M1 codes, two to a byte, with an E8M0 byte for every
// 32 elements of a place. A score may be capped, s -> c tanh(s / c) ahead of log2(e),
// biased by slope_h (j - t), and dropped where j <= t - window (MOD; shape()).
//
// Tiles and items. The rows of a KV head's whole group, token by token, form a
// sequence's run of rows (row r: token r / group, head r % group), cut into tiles
// of 128: K and V are then read once for the group, and the causal edge of a tile
// spans 128 / group tokens only. The lengths are on the device, so the launch
// has an upper bound of work-groups and each finds its item (sequence, tile,
// split of the keys) itself from cu_seqlens and seq_lens (make_plan, find_item).
//
// A work-group is that of attn_fwd_tile.hip: 4 waves of 32 rows, 64-key blocks,
// S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_32x32x16, two LDS slots per
// operand, block j+1's QK^T in the MFMA stream of block j's P.V. A block's 64
// keys are four runs of 16, one per wave, each within a page (the page size is a
// multiple of 16): the run's page comes by v_readlane from a window of 64
// block-table entries, so no load waits on a load. E4M3 codes pass through
// registers and are widened to bf16 (exact) on their way to LDS, once for the
// work-group's four waves; the K scale meets the scores, the V scale P before
// its rounding. MXFP4 codes are widened under their scales there, exact in bf16, and the
// products then are the 16-bit ones. Tiles of at most 32 rows take the narrow form
// (narrow_item; MXFP4: narrow_mx).
//
// One rounding is not the plain form's: P goes to 16 bits for P.V, the operands that
// the matrix instructions take (as a sum of two 16-bit numbers it would cost twice the
// products). The sums l and O are fp32, l of p before the rounding. The result is then
// off by 0.0021-0.0024 of its norm (f16 0.00027) where rounding the output alone gives
// 0.0017 (0.00021). A maximum that lags (kSlack) changes none of it: p's relative
// rounding is the same at 2^8 as at 1, and f16 holds both.
//
// Bound: chunks by the matrix cores beside softmax VALU and copies, as that kernel;
// tiles of few rows by HBM; small launches by the chain lengths - table - K and V -
// states, at 0.7 us a link, and the second launch. Measured (us, in a replayed graph;
// 32 heads of 128 over 8 unless said): 4 x 4096 causal 520-540, 1000 over 30000 460-478
// (1050-1080 TFLOP/s; a bf16 GEMM of 8192^3 1344-1433), 2000 over 6000 E4M3 244
// (bf16 222; head_dim 64 179 and 150; pages of 16 291), 32 x 1 over 8000 164-169 (6.2-6.4
// TB/s), E4M3 96, MXFP4 54, 16 x 1-4 over 8000 69-71, 1 over 32768 29, MXFP4 18, 1 over 64
// 6.1-6.5. MXFP4 chunks take 537 where bf16 takes 517 (4 x 4096): what widening costs
// beside the matrix cores. Shaped scores, 1000 over 12000, 16 heads of 128 over 16, f16:
// plain 116, biased 128, capped 150, windowed to 4096 64 (E4M3 124, 149, 175, 77; f16 of
// head_dim 64 84, 109, 134, 58); four ragged chunks over up to 5000, 32 heads over 8:
// plain 125, MXFP4 133, capped MXFP4 178.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_tile.h"
#include "kernels.h"

namespace neptune {
namespace {

// Inclusive sum over the wave's lanes, by DPP moves
__device__ inline int wave_scan(int x) {
  auto step = [&](auto ctrl, auto rows) {
    x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf,
                                     false);
  };
  typedef std::integral_constant<int, 0xf> all;
  step(std::integral_constant<int, 0x111>{}, all{});  // row_shr 1, 2, 4, 8
  step(std::integral_constant<int, 0x112>{}, all{});
  step(std::integral_constant<int, 0x114>{}, all{});
  step(std::integral_constant<int, 0x118>{}, all{});
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast 15
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast 31
  return x;
}
__device__ inline int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// three loads in flight at once
__device__ inline void together(int &x, int &y, int &z) {
  asm volatile("" : "+v"(x), "+v"(y), "+v"(z));
}

}  // namespace
}  // namespace neptune

#include "attn_plan.h"

namespace neptune {
namespace {

typedef int v2i32 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i32 lds_v2i32;

// bf16 bits of 4 E4M3 codes (exact)
__device__ inline u32x2 widen4(uint32_t c) {
  const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false);
  const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true);
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// E's bits of 8 E2M1 codes under a scale, 2^(e - 127) for a byte e (255: NaN), two
// codes an instruction: exact in bf16 down to 2^-126, in f16 from 2^-24 to 65504
template <class E>
__device__ inline u32x4 widen8(uint32_t c, float scale) {
  u32x4 r;
  if constexpr (std::is_same<E, Bf16Tag>::value) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3));
  }
  return r;
}
// byte i of x as such a scale
__device__ inline float scale_byte(uint32_t x, int i) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ubfe(x, 8 * i, 8) << 23);
}
// The kernel's argument, read again: scalars kept from its first lines on pass what a
// wave has registers for, and were fetched out of vector lanes in the loops (66 of 330
// vector instructions a step of narrow_mx)
__device__ inline const PagedArgs &arguments() {
  auto p = (const __attribute__((address_space(4))) PagedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedArgs *)p;
}
// base + page * stride + place * tok of an MXFP4 pool: a page's offset is a product of 32
// by 32 bits, a place's within it fits 32 (attn_paged_supported), four scalar
// instructions where 64-bit strides take ten
__device__ inline const char *mx_at(const char *base, int page, int64_t stride, int place,
                                    int64_t tok) {
  return base + (uint64_t)(uint32_t)page * (uint32_t)stride + (uint32_t)place * (uint32_t)tok;
}
// x, at its use: loads in flight round a loop are carried whole. (Carried element by
// element they were copied at the loop's end, and so waited for.)
template <class T>
__device__ inline T whole(T x) {
  asm volatile("" : "+v"(x));
  return x;
}
// x, a lane's 32-bit offset from a scalar base, at its use: widened ahead of a loop it
// takes two registers, and the loads 64-bit sums
__device__ inline uint32_t offset(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
// A row's scales as a load brings them, all of a row at once: 32 bits for four, for two
// 16 that are not an integer to the compiler (it carries a small integer round a loop
// widened, and so waits at the loop's end for what is in flight)
template <int HD>
using row_scales = typename std::conditional<HD == 128, uint32_t, _Float16>::type;
// scale i of them
template <class T>
__device__ inline float scale_of(T x, int i) {
  uint32_t bytes;
  if constexpr (sizeof(T) == 4)
    bytes = whole(x);
  else
    bytes = __builtin_bit_cast(uint16_t, whole(x));
  return scale_byte(bytes, i);
}
// a number of the lane's bits: bit i of it is the lane's bit (bits >> 4 i) & 15
__device__ inline int lane_bits(int lane, int bits) {
  int x = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < 2 || bits >> 8) x |= ((lane >> ((bits >> (4 * i)) & 15)) & 1) << i;
  return x;
}

// Scores that are not plain products, in log2 units: cap tanh(x / cap) with x = s sc,
// then slope (key - place). Element r is key c0 + 8 (r >> 2) + (r & 3) after the lane's
// first, which lies d0 after the row's place.
//
// Up to |y| = 3/8, y = x / cap, tanh(y) is y times a polynomial of y^2 (fitted at
// Chebyshev nodes: off by 6e-8, in fp32 1.5e-7, 5e-8 rms), beyond it 1 - 2 / (e^2y + 1),
// whose cancellation would cost a small score its last bits. Scores of ordinary heads
// keep to an eighth of such caps as 30 and 50, so a wave forms the second only for blocks
// that need it.
template <int N, class V>
__device__ inline void shape(const PagedArgs &a, float slope2, float sc, float d0, int c0, V &s) {
  if (a.cap2 != 0.0f) {
    const float u = sc * a.cap_inv;
    float big = 0.0f;
    V y;
#pragma unroll
    for (int r = 0; r < N; ++r) {
      y[r] = s[r] * u;
      big = fmaxf(big, fabsf(y[r]));
      const float w = y[r] * y[r];
      float p = fmaf(w, a.capp[3], a.capp[2]);
      p = fmaf(w, p, a.capp[1]);
      s[r] = y[r] * fmaf(w, p, a.capp[0]);
    }
    if (__any(big > kCapPoly)) {
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const float e = fast_exp2(y[r] * (2.0f * kLog2e));
        const float t = fmaf(-2.0f * a.cap2, __builtin_amdgcn_rcpf(e + 1.0f), a.cap2);
        s[r] = fabsf(y[r]) > kCapPoly ? t : s[r];
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < N; ++r) s[r] *= sc;
  }
  if (a.slopes) {
#pragma unroll
    for (int r = 0; r < N; ++r)
      s[r] = fmaf(slope2, d0 + (float)(c0 + 8 * (r >> 2) + (r & 3)), s[r]);
  }
}

// Whether some row's maximum is so large that p = 2^(s sc - m) needs its products rounded, as
// the maximum's was. One fma takes the exact product: the largest p is then off 1 by half a
// step of m in the exponent, and all of the row's with it. Below 2^24 that is 2^+-0.5; from
// 2^31 on (f16: 2^28) it may be more than the type holds, and rows came out infinite or empty.
// (Costs up to 1%: 6 x 32-130 head_dim-64 tokens over 1500 20.0 / 20.1 us, MXFP4 capped chunks
// 176.6 / 178.4, E4M3 chunks 167.6 / 169.7; 4 x 4096 nothing.)
__device__ inline bool huge(float m) { return __any(fabsf(m) >= 0x1p24f); }

// The scale that V's scales are taken relative to where they meet P: that of the
// first page looked at, in lane 0 of vscv. P is rounded to 16 bits with the ratio
// in it, so its large values, at most 1, stay next to 1 and below, where bf16's
// relative step is smallest, and 1 stays exact; the usual scales, amax / 448 with
// amax near 4, lie just above 2^-7, where it is largest (a row over few keys: off by
// 0.0027 of its norm with the bare scales, 0.0021 so; the output's rounding alone is
// 0.0017). Within 2^+-16, so that no ratio leaves the range of an ordinary float.
__device__ inline float scale_unit(float vscv) {
  const float v = __builtin_bit_cast(
      float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vscv), 0));
  return v >= 0x1p-16f && v <= 0x1p16f ? v : 1.0f;
}
// (v_rcp_f32 inverts it: 1 ulp)
__device__ inline float scalar(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// Infinities and NaN of V behind the mask. A masked key's p is 0, but 0 times them
// is NaN, and a matrix product cannot leave a key out for some of its rows. So in
// blocks that any row of a tile does not see whole, V is looked over in LDS before
// its use, such values (hardly ever: a new token whose V overflowed) become 0, and
// the rows that do see them have them added at the end (add_special). All-ones
// exponents (E4M3: all-ones magnitudes) carry into the bit above them.
template <class E, bool FP8>
struct Special {
  static constexpr uint32_t ONES = FP8 ? 0x7f7f7f7fu
                                       : std::is_same<E, Bf16Tag>::value ? 0x7f807f80u : 0x7c007c00u;
  static constexpr uint32_t UNIT = FP8 ? 0x01010101u
                                       : std::is_same<E, Bf16Tag>::value ? 0x00800080u : 0x04000400u;
  static constexpr uint32_t TOP = FP8 ? 0x80808080u : 0x80008000u;
  __device__ static inline uint32_t marks(uint32_t x) { return ((x & ONES) + UNIT) & TOP; }
  __device__ static inline uint32_t marks(u32x4 x) {
    return marks(x[0]) | marks(x[1]) | marks(x[2]) | marks(x[3]);
  }
  __device__ static inline u32x4 without(u32x4 x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = marks(x[i]);
      x[i] &= ~(FP8 ? (m >> 7) * 0xffu : (m >> 15) * 0xffffu);
    }
    return x;
  }
  // takes them out of N KiB of LDS; whether there were any
  template <int N>
  __device__ static inline bool scrub(const uint8_t *p, int lane) {
    u32x4 *at = (u32x4 *)p + lane;
    u32x4 x[N];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = at[64 * i];
#pragma unroll
    for (int i = 0; i < N; ++i) m |= marks(x[i]);
    const bool found = __any(m != 0);
    if (__builtin_expect(found, 0)) {
#pragma unroll
      for (int i = 0; i < N; ++i) at[64 * i] = without(x[i]);
    }
    return found;
  }
};

// add(i, e, x) for the special values x of V's keys lo .. hi - 1 that the row at pos sees,
// elements e of the lane's runs of four: head_dim RUN i + 4 g + e
template <class E, int HD, int POOL, int RUN, int VECTORS, class O>
__device__ inline void add_special(const PagedArgs &a, const Item &it, int hk, int lo, int hi,
                                   int pos, int g, O add) {
  const int from = a.window ? pos - a.window : -1;  // the last key before the row's
  const int32_t *tab = a.btab + (int64_t)it.b * a.maxp;
#pragma unroll 1
  for (int j = lo; j < hi; ++j) {
    int index, rest;
    page_of(a, j >> 4, &index, &rest);
    const int page = min(max(tab[index], 0), a.npages - 1);
    const int place = rest * 16 + (j & 15);
    const char *v = a.v + hk * a.vps1 + page * a.vps0 + (int64_t)place * a.vtok;
    const uint8_t *vs = POOL == MXFP4
                            ? a.vmx + hk * a.vss1 + page * a.vss0 + (int64_t)place * a.vstok
                            : nullptr;
#pragma unroll
    for (int i = 0; i < VECTORS; ++i) {
      const int d = RUN * i + 4 * g;
      u32x4 four;
      if constexpr (POOL == MXFP4)
        four = widen8<E>(*(const uint16_t *)(v + d / 2), scale_byte(vs[d / 32], 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x;
        if constexpr (POOL == MXFP4)
          x = E::to_f32((uint16_t)(four[e >> 1] >> (16 * (e & 1))));
        else if constexpr (POOL == E4M3)
          x = (((const uint8_t *)v)[d + e] & 0x7f) == 0x7f ? __builtin_nanf("") : 0.0f;
        else
          x = E::to_f32(((const uint16_t *)v)[d + e]);
        if (j <= pos && j > from && !(fabsf(x) <= 3.4e38f)) add(i, e, x);
      }
      __builtin_amdgcn_sched_barrier(0);  // few registers at a time
    }
  }
}
// (o of the 32-row forms: element 4 rq + e of o[nb] is head_dim 32 nb + 8 rq + 4 g + e)
template <class E, int HD, int POOL>
__device__ inline void add_special(const PagedArgs &a, const Item &it, int hk, int lo, int hi,
                                   int pos, int g, f32x16 (&o)[HD / 32]) {
  add_special<E, HD, POOL, 8, HD / 8>(a, it, hk, lo, hi, pos, g, [&](int i, int e, float x) {
    o[i >> 2][4 * (i & 3) + e] += x;
  });
}

// A tile of at most 32 rows (generated or guessed tokens, a chunk's last few): the
// wide form would compute in one wave of four and hold 32 KB in flight between
// barriers, and such an item is bound by memory. Here the four waves share out
// the item's keys in steps of 32, each streaming its own through 16 KB of LDS
// with no barrier: K of step i + N is issued once step i's scores are formed, V
// once its P.V is (N slots per operand: 1 for 16-bit head_dim 128, 2 or 4 for
// smaller rows), so a wave has copies in flight at all times. E4M3 codes stay codes in
// LDS and are widened as operands are read. The running max moves with every
// step, so a row's largest p is 1. At the end the waves' states merge in LDS, a
// quarter of the head_dim each.
template <class E, int HD, int POOL, bool MOD>
__device__ inline void narrow_item(const PagedArgs &a, const Item &it, int hk, int w, int lane,
                                   int kb0, int nv, const uint8_t *smem, f32x2 *mlbox) {
  typedef typename E::vec8 V8;
  constexpr bool FP8 = POOL == E4M3;
  constexpr int STEP = 32;
  constexpr int RB = HD * (FP8 ? 1 : 2);        // bytes of a row
  constexpr int TILE = STEP * RB;
  constexpr int REGION = 16384;                 // LDS per wave
  constexpr int N = REGION / (2 * TILE);        // slots per operand
  constexpr int UNITS = RB / 16, RPC = 64 / UNITS;  // 16-byte units per row, rows per 1 KiB chunk
  constexpr int CH = TILE / 1024;               // chunks per tile
  constexpr int NST = HD / 16, NB = HD / 32;
  const int lq = lane & 31, g = lane >> 5;
  const uint8_t *const mine = smem + w * REGION;
  auto kslot = [&](int i) { return mine + (i % N) * TILE; };
  auto vslot = [&](int i) { return mine + (N + i % N) * TILE; };
  // 256 bytes hold 1, 2 or 4 rows: the unit that row r's unit u goes to
  auto kswz = [](int r) {
    return UNITS == 16 ? r & 15 : UNITS == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  };
  auto vswz = [](int r) {
    return FP8 ? (UNITS == 8 ? (r >> 1) & 7 : (r >> 2) & 3)
               : (UNITS == 16 ? (r & 3) << 2 : ((r >> 1) & 1) << 2);
  };

  const int off = it.len - it.n, base_row = it.tile * BM;
  const int rows = min(it.n * a.group - base_row, NARROW);
  const int row = base_row + min(lq, rows - 1);
  const int tok = quotient(row, a.group, a.group_inv), hr = row - tok * a.group;
  const int pos = off + tok;
  const int lo = __builtin_amdgcn_readfirstlane(off + quotient(base_row, a.group, a.group_inv));
  const int last = off + quotient(base_row + rows - 1, a.group, a.group_inv);  // the last row's place
  // the wave's steps of the item's
  const int s0 = max(2 * kb0, MOD && a.window ? max(lo - a.window + 1, 0) / STEP : 0);
  const int s1 = min(2 * (kb0 + nv), last < 0 ? 0 : last / STEP + 1);
  const int share = (max(s1 - s0, 0) + 3) >> 2;
  const int t0 = __builtin_amdgcn_readfirstlane(s0 + w * share);
  const int ns = __builtin_amdgcn_readfirstlane(max(min(t0 + share, s1) - t0, 0));

  const char *kp = a.k + hk * a.kps1, *vp = a.v + hk * a.vps1;
  const int32_t *tab = a.btab + (int64_t)it.b * a.maxp;
  const int last_run = (it.len - 1) >> 4;
  // No other tile of the sequence reads these keys, so their copies pass the caches by
  // (32 x 1 over 8000, pages apart, 171 us, with them kept 191; E4M3 95, 109). Sequences
  // may share pages, which a tile cannot tell from its own table: each then reads them
  // again, at 2-3% more than through the caches (32 x 1 over the same 8000 tokens 69 us,
  // kept 67; 64 x 1 over 2000 40.2, 39.1).
  const bool once = it.tiles == 1;
  int tab0 = 0, tabv = 0, sc0 = 0;
  float kscv = 0.0f, vscv = 0.0f;
  auto load_tab = [&](int first) {
    tab0 = first;
    const int j = first + lane;
    tabv = j < a.maxp ? tab[j] : 0;
  };
  auto load_scales = [&](int first) {
    sc0 = first;
    const int j = first + lane;
    const int page = min(max(j < a.maxp ? tab[j] : 0, 0), a.npages - 1);
    kscv = a.ksc[(int64_t)page * a.Hk + hk];
    vscv = a.vsc[(int64_t)page * a.Hk + hk];
  };
  if (ns > 0) {
    int index, rest;
    page_of(a, min(2 * t0, last_run), &index, &rest);
    load_tab(index);
    if constexpr (FP8) load_scales(index);
  }
  u32x4 qf[NST];
  {
    const uint16_t *qp = a.q + (int64_t)(it.row0 + tok) * a.qs0 +
                         (int64_t)(hk * a.group + hr) * a.qs1 + 8 * g;
#pragma unroll
    for (int st = 0; st < NST; ++st)
      qf[st] = lq < rows ? *(const u32x4 *)(qp + 16 * st) : u32x4{0, 0, 0, 0};
  }
  float slope2 = 0.0f;
  if constexpr (MOD)
    if (a.slopes) slope2 = a.slopes[hk * a.group + hr] * kLog2e;
  settle(slope2);
  settle(kscv);
  settle(vscv);
  const float unit = FP8 ? scale_unit(vscv) : 1.0f, unit_inv = FP8 ? scalar(__builtin_amdgcn_rcpf(unit)) : 1.0f;
#pragma unroll
  for (int st = 0; st < NST; ++st) settle(qf[st]);
  settle(tabv);

  // one operand's copy of step i: two runs of 16 rows, each within a page, rows
  // behind the sequence's end from its last
  const int crow = lane / UNITS, cunit = lane & (UNITS - 1);
  auto copy = [&](int i, auto is_v, const uint8_t *tile) {
    constexpr bool V = decltype(is_v)::value;
    const int64_t tokb = V ? a.vtok : a.ktok;
    static_for<2>([&](auto H) {
      constexpr int h = decltype(H)::value;
      const int run = min(2 * (t0 + i) + h, last_run);
      int index, rest;
      page_of(a, run, &index, &rest);
      if (index - tab0 >= 64) {
        load_tab(max(index - 1, 0));  // V's first run may lie a page before K's second
        settle(tabv);
      }
      int page = __builtin_amdgcn_readlane(tabv, index - tab0);
      page = min(max(page, 0), a.npages - 1);
      const char *src = (V ? vp + page * a.vps0 : kp + page * a.kps0) + (int64_t)(rest * 16) * tokb;
      const int most = it.len - 1 - run * 16;
      auto issue = [&](auto nt) {
#pragma unroll
        for (int c = 0; c < CH / 2; ++c) {
          const int r = crow + RPC * c;  // of the run
          const int u = cunit ^ (V ? vswz(16 * h + r) : kswz(16 * h + r));
          dma16<decltype(nt)::value>(src, (uint32_t)(min(r, most) * tokb + u * 16),
                                     lds_offset(tile + (h * CH / 2 + c) * 1024));
        }
      };
      if (once)
        issue(std::true_type{});
      else
        issue(std::false_type{});
    });
  };
  auto copy_k = [&](int i) { copy(i, std::false_type{}, kslot(i)); };
  auto copy_v = [&](int i) { copy(i, std::true_type{}, vslot(i)); };

  f32x16 o[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.0f;
  float m = kNegFltMax, lsum = 0.0f;
  static_for<N>([&](auto J) {
    if (decltype(J)::value < ns) {
      copy_k(decltype(J)::value);
      copy_v(decltype(J)::value);
    }
  });
  bool special = false;
  // waits until the copies issued after a tile are all that is in flight: `pairs`
  // whole steps' (at most N - 1) and X tiles
  auto wait_tiles = [&](int pairs, auto extra) {
    constexpr int X = decltype(extra)::value;
    static_for<N>([&](auto P) {
      constexpr int n = decltype(P)::value;
      if (min(pairs, N - 1) == n) __builtin_amdgcn_s_waitcnt(waitcnt_vm(CH * (2 * n + X)));
    });
    asm volatile("" ::: "memory");  // no read of the tile before the wait
  };

  for (int i = 0; i < ns; ++i) {
    const int later = ns - 1 - i;
    const int key0 = (t0 + i) * STEP;
    wait_tiles(later, std::integral_constant<int, 1>{});  // K(i) is there
    f32x16 s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    {
      const uint8_t *kt = kslot(i) + lq * RB;
#pragma unroll
      for (int st = 0; st < NST; ++st) {
        u32x4 A;
        if constexpr (FP8) {
          const u32x2 c = *(const u32x2 *)(kt + ((st ^ kswz(lq)) << 4) + 8 * g);
          const u32x2 x = widen4(c[0]), y = widen4(c[1]);
          A = u32x4{x[0], x[1], y[0], y[1]};
        } else {
          A = *(const u32x4 *)(kt + (((2 * st + g) ^ kswz(lq)) << 4));
        }
        s = E::mfma32(as_vec8<V8>(A), as_vec8<V8>(qf[st]), s);
      }
    }
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);  // K(i) has been read
    if (later >= N) copy_k(i + N);
    float vs[2] = {1.0f, 1.0f};
    if constexpr (FP8) {
      // the scales of both runs: K's before the mask, V's with P
      static_for<2>([&](auto H) {
        constexpr int h = decltype(H)::value;
        int index, rest;
        page_of(a, min(2 * (t0 + i) + h, last_run), &index, &rest);
        if (index - sc0 >= 64) {
          load_scales(index);
          settle(kscv);
          settle(vscv);
        }
        const float ks = a.scale2 * __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kscv), index - sc0));
        vs[h] = unit_inv * __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vscv), index - sc0));
#pragma unroll
        for (int r = 0; r < 8; ++r) s[8 * h + r] *= ks;
      });
    } else if constexpr (!MOD) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= a.scale2;
    }
    const int lim = pos - key0 - 4 * g;  // element r holds key 4 g + 8 (r >> 2) + (r & 3)
    if constexpr (MOD) shape<16>(a, slope2, FP8 ? 1.0f : a.scale2, (float)-lim, 0, s);
    bool masked = key0 + STEP - 1 > lo;
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
    }
    if constexpr (MOD)
      if (a.window && key0 + a.window <= last) {  // some row's window begins behind its keys
        masked = true;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + (r & 3) <= lim - a.window) s[r] = -INFINITY;
      }
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = pair_max(mx);
    if (__any(mx > m)) {
      const float m_new = fmaxf(m, mx);
      const float alpha = fast_exp2(m - m_new);
      lsum *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nb][r] *= alpha;
      m = m_new;
    }
    u32x4 pf[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = fast_exp2(s[8 * c + 2 * j] - m), p1 = fast_exp2(s[8 * c + 2 * j + 1] - m);
        lsum += p0 + p1;
        // rounded to 16 bits (above), V's scale with it; a masked key's page may hold any
        pf[c][j] = FP8 ? E::pack2(p0 == 0.0f ? 0.0f : p0 * vs[c], p1 == 0.0f ? 0.0f : p1 * vs[c])
                       : E::pack2(p0, p1);
      }
    if (later >= N)
      wait_tiles(N - 1, std::integral_constant<int, 1>{});  // V(i) is there, K(i + N) after it
    else
      wait_tiles(later, std::integral_constant<int, 0>{});
    const uint8_t *vt = vslot(i);
    auto v_operand = [&](int c, int nb) {
      const int s16 = lane & 15, dh = (lane >> 4) & 1;
      if constexpr (FP8) {
        // lane pair (2 j, 2 j + 1) of 16 names the row of k-slot j
        const int j = s16 >> 1, r = 16 * c + 4 * g + (j & 3) + 8 * (j >> 2);
        const v2i32 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i32 *)as_lds(
            vt + r * RB + (((2 * nb + dh) ^ vswz(r)) << 4) + 8 * (s16 & 1)));
        const u32x2 y = widen4((uint32_t)x[0]), z = widen4((uint32_t)x[1]);
        return u32x4{y[0], y[1], z[0], z[1]};
      } else {
        const int j = s16 >> 2, r = 16 * c + 4 * g + j;
        const uint8_t *p = vt + r * RB + (((4 * nb + 2 * dh) ^ vswz(j)) << 4) + 8 * (s16 & 3);
        const u32x2 y = __builtin_bit_cast(u32x2, lds_read_tr16(p));
        const u32x2 z = __builtin_bit_cast(u32x2, lds_read_tr16(p + 8 * RB));
        return u32x4{y[0], y[1], z[0], z[1]};
      }
    };
    if (masked) special |= Special<E, FP8>::template scrub<CH>(vt, lane);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        o[nb] = E::mfma32(as_vec8<V8>(v_operand(c, nb)), as_vec8<V8>(pf[c]), o[nb]);
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);  // V(i) has been read
    if (later >= N) copy_v(i + N);
  }

  if (__builtin_expect(special, 0))
    add_special<E, HD, POOL>(a, it, hk,
                             MOD && a.window ? t0 * STEP : max(t0 * STEP, lo / STEP * STEP),
                             min((t0 + ns) * STEP, it.len), pos, g, o);
  if constexpr (FP8) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[nb] *= unit;
  }
  // the waves' states, merged lane by lane, NB of a row's 4 NB vectors a wave
  const float ltot = pair_sum(lsum);
  f32x4 *const box = (f32x4 *)mine + lane;
#pragma unroll
  for (int v = 0; v < 4 * NB; ++v)
    box[v * 64] = f32x4{o[v >> 2][4 * (v & 3)], o[v >> 2][4 * (v & 3) + 1],
                        o[v >> 2][4 * (v & 3) + 2], o[v >> 2][4 * (v & 3) + 3]};
  mlbox[w * 64 + lane] = f32x2{m, ltot};
  __syncthreads();
  float M = kNegFltMax, L = 0.0f, wgt[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) M = fmaxf(M, mlbox[k * 64 + lane][0]);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const f32x2 ml = mlbox[k * 64 + lane];
    wgt[k] = fast_exp2(ml[0] - M);
    L = fmaf(wgt[k], ml[1], L);
  }
  if (lq >= rows) return;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const int64_t t = it.row0 + tok;
  const int64_t part = ((int64_t)(it.part + it.split) * a.Hk + hk) * a.prows + lq;
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    const int v = w * NB + k, d = 32 * (v >> 2) + 8 * (v & 3) + 4 * g;
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 y = *((const f32x4 *)(smem + j * REGION) + v * 64 + lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(wgt[j], y[e], x[e]);
    }
    if (it.splits > 1)
      *(f32x4 *)(a.po + part * HD + d) = x;
    else
      *(u32x2 *)(a.o + t * a.os0 + (int64_t)(hk * a.group + hr) * a.os1 + d) =
          u32x2{E::pack2(x[0] * inv, x[1] * inv), E::pack2(x[2] * inv, x[3] * inv)};
  }
  if (w == 0 && g == 0) {
    if (it.splits > 1)
      *(f32x2 *)(a.pml + part * 2) = f32x2{M, L};
    else if (a.lse)
      a.lse[t * a.Hq + hk * a.group + hr] = L == 0.0f ? -INFINITY : row_lse(M, L);
  }
}

// The same over MXFP4 pools, with products of 16 by 16 by 32: a decoded token's few heads
// fill a quarter of 16 rows, not an eighth of 32, so scores and products cost half. NQ
// tiles of 16 rows. Lane (c, g) of 16 by 4 holds S^T's keys 4 g + r of each run of 16 for
// row c, and O^T's head_dim 16 nd + 4 g + r.
//
// A step is 32 keys, two runs of 16; its codes come in registers, a step ahead. K: a lane
// takes 32 (head_dim 64: 16) elements of one row of each run, and one scale, as the
// products' operands (which element a k-slot holds is free, as long as Q's agree). V goes
// through LDS widened, and is read transposed; keys 16 t + 4 g + r take k-slot
// 8 g + 4 t + r, where P has them. A run lies within a page, so a load's base is scalar and
// its offsets are the same all along. Bound by the loads' latency where a wave has few
// steps, by HBM where it has many (8 heads of 128, 4 queries each, in a replayed graph):
// 1 by 4000 keys 11.3 us, 32 by 4000 32.0 us, 32 by 8000 53.9 us. Steps of 64 keys: 12.6,
// 33.4, 54.3; three steps of 32 in flight, in a loop unrolled as often, were slower by the
// code's length, 1 by 400 8.6 us against 8.2.
template <class E, int HD, bool MOD, int NQ>
__device__ inline void narrow_mx(const Item &it, int hk, int w, int lane, int kb0, int nv,
                                 const uint8_t *smem, f32x2 *mlbox) {
  const PagedArgs &a = arguments();
  typedef typename E::vec8 V8;
  constexpr int STEP = 32, RUNS = STEP / 16;
  constexpr int RB = HD * 2;        // bytes of V's rows in LDS
  constexpr int REGION = 16384;     // LDS per wave: V's tile, and its state at the end
  constexpr int ND = HD / 16;       // 16-wide head_dim tiles of O^T
  constexpr int KS = HD / 32;       // k-steps of S^T
  constexpr int LB = HD / 8;        // bytes of codes a lane takes of a row
  typedef typename std::conditional<HD == 128, u32x4, u32x2>::type codes_t;
  const int c16 = lane & 15, g = lane >> 4;
  const uint8_t *const mine = smem + w * REGION;
  // 16-byte units of a row of V: eight rows' neighbouring pairs, which half a wave reads
  // transposed at once, lie in different banks, and so do the single ones of rows 0, 1, 8
  // and 9 (head_dim 64: 0 and 8) apart, which eight lanes write
  auto vswz = [](int r) {
    return (HD == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  };

  const int off = it.len - it.n, base_row = it.tile * BM;
  const int rows = min(it.n * a.group - base_row, NARROW);
  int tok[NQ], hr[NQ], pos[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int row = base_row + min(16 * q + c16, rows - 1);
    tok[q] = quotient(row, a.group, a.group_inv);
    hr[q] = row - tok[q] * a.group;
    pos[q] = off + tok[q];
  }
  const int lo = __builtin_amdgcn_readfirstlane(off + quotient(base_row, a.group, a.group_inv));
  const int last = off + quotient(base_row + rows - 1, a.group, a.group_inv);  // the last row's place
  // the wave's steps of the item's
  const int s0 = max(2 * kb0, MOD && a.window ? max(lo - a.window + 1, 0) / STEP : 0);
  const int s1 = min(2 * (kb0 + nv), last < 0 ? 0 : last / STEP + 1);
  const int share = (max(s1 - s0, 0) + 3) >> 2;
  const int t0 = __builtin_amdgcn_readfirstlane(s0 + w * share);
  const int ns = __builtin_amdgcn_readfirstlane(max(min(t0 + share, s1) - t0, 0));

  const char *kp = a.k + hk * a.kps1, *vp = a.v + hk * a.vps1;
  const char *ksp = (const char *)a.kmx + hk * a.kss1, *vsp = (const char *)a.vmx + hk * a.vss1;
  const int32_t *tab = a.btab + (int64_t)it.b * a.maxp;
  const int last_run = (it.len - 1) >> 4;
  int tab0 = 0, tabv = 0;
  auto load_tab = [&](int first) {
    tab0 = first;
    const int j = first + lane;
    tabv = j < a.maxp ? tab[j] : 0;
  };
  if (ns > 0) {
    int index, rest;
    page_of(a, min(RUNS * t0, last_run), &index, &rest);
    load_tab(index);
  }
  // Q: k-step u's 8 elements are those of K's operand
  u32x4 qf[NQ][KS];
  float slope2[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const uint16_t *qp = a.q + (int64_t)(it.row0 + tok[q]) * a.qs0 +
                         (int64_t)(hk * a.group + hr[q]) * a.qs1 + 2 * LB * g;
#pragma unroll
    for (int u = 0; u < KS; ++u)
      qf[q][u] = 16 * q + c16 < rows ? *(const u32x4 *)(qp + 8 * u) : u32x4{0, 0, 0, 0};
    slope2[q] = 0.0f;
    if constexpr (MOD)
      if (a.slopes) slope2[q] = a.slopes[hk * a.group + hr[q]] * kLog2e;
  }

  // a lane's row of a run, and where it lies in it: K's row c16, its quarter g; V's in an
  // order that keeps apart the eight neighbouring lanes that write at once, over 128 bytes
  const int vq = lane_bits(lane, HD == 128 ? 0x30 : 0x10);
  const int vrow = lane_bits(lane, HD == 128 ? 0x2541 : 0x2543);
  codes_t kc[RUNS], vc[RUNS];
  row_scales<HD> ks[RUNS], vs[RUNS];
  // A run's 16 rows all lie in its page, those behind the sequence's end too: what they
  // hold meets scores that are masked (K), or becomes nothing under a scale of 2^-127 (V).
  const uint32_t koff = c16 * (uint32_t)a.ktok + LB * g, voff = vrow * (uint32_t)a.vtok + LB * vq;
  const uint32_t ksoff = c16 * (uint32_t)a.kstok, vsoff = vrow * (uint32_t)a.vstok;
  const int kblk = HD == 128 ? g : g >> 1, vblk = HD == 128 ? vq : vq >> 1;
  // pages of an even number of runs: a step lies within one, and its place is looked up once
  const bool same = !(a.ps16 & 1);
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int run = RUNS * (t0 + i);
    int index, rest;
    page_of(a, min(run, last_run), &index, &rest);
    const char *at[4];  // the run's first place: K, its scales, V, its scales
#pragma unroll
    for (int h = 0; h < RUNS; ++h) {
      const bool more = run + h <= last_run;  // (behind the end: the last run again)
      if (h && same) {
        at[0] += more ? 16 * (uint32_t)a.ktok : 0;
        at[1] += more ? 16 * (uint32_t)a.kstok : 0;
        at[2] += more ? 16 * (uint32_t)a.vtok : 0;
        at[3] += more ? 16 * (uint32_t)a.vstok : 0;
      } else {
        if (h && more && ++rest == a.ps16) {
          rest = 0;
          ++index;
        }
        if (index - tab0 >= 64) {
          load_tab(max(index - 1, 0));  // the step's first run may lie a page before
          settle(tabv);
        }
        int page = __builtin_amdgcn_readlane(tabv, index - tab0);
        page = min(max(page, 0), a.npages - 1);
        const int place = rest * 16;
        at[0] = mx_at(kp, page, a.kps0, place, a.ktok);
        at[1] = mx_at(ksp, page, a.kss0, place, a.kstok);
        at[2] = mx_at(vp, page, a.vps0, place, a.vtok);
        at[3] = mx_at(vsp, page, a.vss0, place, a.vstok);
      }
      kc[h] = *(const codes_t *)(at[0] + offset(koff));
      ks[h] = *(const row_scales<HD> *)(at[1] + offset(ksoff));
      vc[h] = *(const codes_t *)(at[2] + offset(voff));
      vs[h] = *(const row_scales<HD> *)(at[3] + offset(vsoff));
    }
  };
  const int vput = vrow * RB + (((LB / 4 * vq) ^ vswz(vrow)) << 4);
  // V's first operand: row 4 g + j, the run's second 16 rows on
  const int vj = 4 * g + (c16 >> 2);
  const int vget0 = vj * RB + ((((c16 >> 1) & 1) ^ vswz(vj)) << 4) + 8 * (c16 & 1);

  f32x4 o[NQ][ND];
  float m[NQ], lsum[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) o[q][nd] = f32x4{0, 0, 0, 0};
    m[q] = kNegFltMax;
    lsum[q] = 0.0f;
  }
  bool special = false;
  if (ns > 0) fetch(0);
  // (Q was asked for before: waited for here, not in the loop for all)
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
#pragma unroll
    for (int u = 0; u < KS; ++u) settle(qf[q][u]);
    settle(slope2[q]);
  }

  for (int i = 0; i < ns; ++i) {
    const int key0 = (t0 + i) * STEP;
    f32x4 s[NQ][RUNS];
#pragma unroll
    for (int h = 0; h < RUNS; ++h) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][h] = f32x4{0, 0, 0, 0};
      const codes_t codes = whole(kc[h]);
      const float scale = scale_of(ks[h], kblk);
#pragma unroll
      for (int u = 0; u < KS; ++u) {
        const u32x4 A = widen8<E>(codes[u], scale);
#pragma unroll
        for (int q = 0; q < NQ; ++q)
          s[q][h] = E::mfma16(as_vec8<V8>(A), as_vec8<V8>(qf[q][u]), s[q][h]);
      }
    }
    int to = vput;  // (one register for the stores' addresses)
    asm volatile("" : "+v"(to));
#pragma unroll
    for (int h = 0; h < RUNS; ++h) {
      const codes_t codes = whole(vc[h]);
      const float held = scale_of(vs[h], vblk);
      const float scale = key0 + 16 * h + vrow < it.len ? held : 0.0f;
#pragma unroll
      for (int u = 0; u < LB / 4; ++u)
        *(u32x4 *)(uint8_t *)(mine + 16 * h * RB + (to ^ (u << 4))) = widen8<E>(codes[u], scale);
    }
    __builtin_amdgcn_sched_barrier(0);
    fetch(min(i + 1, ns - 1));
    __builtin_amdgcn_sched_barrier(0);
    bool masked = key0 + STEP - 1 > lo;
    u32x4 pf[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int lim = pos[q] - key0 - 4 * g;  // element (h, r) holds key 4 g + 16 h + r
      float sc = a.scale2;
      if constexpr (MOD) {
#pragma unroll
        for (int h = 0; h < RUNS; ++h) shape<4>(a, slope2[q], sc, (float)-lim, 16 * h, s[q][h]);
        sc = 1.0f;
      }
      if (key0 + STEP - 1 > lo) {
#pragma unroll
        for (int h = 0; h < RUNS; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * h + r > lim) s[q][h][r] = -INFINITY;
      }
      if constexpr (MOD)
        if (a.window && key0 + a.window <= last) {  // some row's window begins behind its keys
          masked = true;
#pragma unroll
          for (int h = 0; h < RUNS; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * h + r <= lim - a.window) s[q][h][r] = -INFINITY;
        }
      float rs;
      auto expo = [&]() {
#pragma unroll
        for (int h = 0; h < RUNS; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float p0 = fast_exp2(fmaf(s[q][h][2 * j], sc, -m[q]));
            const float p1 = fast_exp2(fmaf(s[q][h][2 * j + 1], sc, -m[q]));
            rs = h + j == 0 ? p0 : rs + p0;
            rs += p1;
            pf[q][2 * h + j] = E::pack2(p0, p1);  // 16 bits, for P.V alone
          }
      };
      auto products = [&]() {  // rounded, where huge() asks for it
        if (!MOD && __builtin_expect(huge(m[q]), 0)) {
#pragma unroll
          for (int h = 0; h < RUNS; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[q][h][r] *= sc;
          sc = 1.0f;
        }
      };
      // past the first step the max is formed only where a lane's sum passes 2^kSlack: up
      // to that m keeps
      bool full = i == 0;
      if (!full) {
        products();
        expo();
        full = __any(!(rs <= kSumCap));
      }
      if (full) {
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < RUNS; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[q][h][r]);
        const float m_new = fmaxf(m[q], max_xor32(max_xor16(mx)) * sc);
        const float alpha = fast_exp2(m[q] - m_new);
        lsum[q] *= alpha;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[q][nd][r] *= alpha;
        m[q] = m_new;
        products();
        expo();
      }
      lsum[q] += rs;
    }
    asm volatile("" ::: "memory");  // no read of V before its stores
    if (masked) {
#pragma unroll 1
      for (int h = 0; h < RUNS; ++h)
        special |= Special<E, false>::template scrub<HD / 32>(mine + 16 * h * RB, lane);
      asm volatile("" ::: "memory");
    }
    int from = vget0;
    asm volatile("" : "+v"(from));
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) {
      const uint8_t *p = mine + (from ^ (nd << 5));
      const u32x2 x = __builtin_bit_cast(u32x2, lds_read_tr16(p));
      const u32x2 y = __builtin_bit_cast(u32x2, lds_read_tr16(p + 16 * RB));
      const u32x4 A = {x[0], x[1], y[0], y[1]};
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        o[q][nd] = E::mfma16(as_vec8<V8>(A), as_vec8<V8>(pf[q]), o[q][nd]);
    }
    asm volatile("" ::: "memory");  // nor the next V's stores before these reads
  }

  if (__builtin_expect(special, 0)) {
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      add_special<E, HD, MXFP4, 16, ND>(
          a, it, hk, MOD && a.window ? t0 * STEP : max(t0 * STEP, lo / STEP * STEP),
          min((t0 + ns) * STEP, it.len), pos[q], g, [&](int i, int e, float x) { o[q][i][e] += x; });
  }
  // the waves' states, merged lane by lane, a quarter of a row's vectors a wave
  constexpr int VECTORS = NQ * ND;
  f32x4 *const box = (f32x4 *)mine + lane;
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) box[v * 64] = o[v / ND][v % ND];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const float ltot = sum_xor32(sum_xor16(lsum[q]));
    if (g == 0) mlbox[(w * NQ + q) * 16 + c16] = f32x2{m[q], ltot};
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float M = kNegFltMax, L = 0.0f, wgt[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) M = fmaxf(M, mlbox[(k * NQ + q) * 16 + c16][0]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x2 ml = mlbox[(k * NQ + q) * 16 + c16];
      wgt[k] = fast_exp2(ml[0] - M);
      L = fmaf(wgt[k], ml[1], L);
    }
    if (16 * q + c16 >= rows) continue;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int64_t t = it.row0 + tok[q];
    const int64_t part = ((int64_t)(it.part + it.split) * a.Hk + hk) * a.prows + 16 * q + c16;
#pragma unroll
    for (int k = 0; k < ND / 4; ++k) {
      const int nd = w * (ND / 4) + k, d = 16 * nd + 4 * g;
      f32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 y = *((const f32x4 *)(smem + j * REGION) + (q * ND + nd) * 64 + lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(wgt[j], y[e], x[e]);
      }
      if (it.splits > 1)
        *(f32x4 *)(a.po + part * HD + d) = x;
      else
        *(u32x2 *)(a.o + t * a.os0 + (int64_t)(hk * a.group + hr[q]) * a.os1 + d) =
            u32x2{E::pack2(x[0] * inv, x[1] * inv), E::pack2(x[2] * inv, x[3] * inv)};
    }
    if (w == 0 && g == 0) {
      if (it.splits > 1)
        *(f32x2 *)(a.pml + part * 2) = f32x2{M, L};
      else if (a.lse)
        a.lse[t * a.Hq + hk * a.group + hr[q]] = L == 0.0f ? -INFINITY : row_lse(M, L);
    }
  }
}

template <class E, int HD, int POOL, bool MOD>
__global__ __launch_bounds__(NT, 2) void attn_paged(PagedArgs args) {
  typedef typename E::vec8 V8;
  constexpr bool FP8 = POOL == E4M3, MX = POOL == MXFP4;
  constexpr bool CODES = FP8 || MX;  // widened on their way to LDS
  // (E4M3's scores have a scale for each page; head_dim 64 forms every block's maximum)
  constexpr bool FOLD = MOD && HD == 128 && !FP8;
  // Biases grow towards the row's own place: from there back, the first block sets the
  // maximum, and none after it raises it far
  constexpr bool BACK = MOD;

  typedef TileLoader<HD> TL;
  constexpr int TILE = TL::TILE_BYTES;
  constexpr int ROWB = HD * 2;   // bytes per LDS row
  constexpr int NST = HD / 16;   // QK^T k-steps
  constexpr int NB = HD / 32;    // 32-wide head_dim blocks of O^T
  constexpr int NQK = 2 * NST, NPV = 4 * NB;  // MFMAs per key block
  constexpr int CHUNKS = TL::CHUNKS, RPC = TL::RPC;
  // K slots 0 and 1, then V slots 0 and 1; block t uses slot t & 1
  __shared__ __attribute__((aligned(16))) uint8_t smem[65536];
  __shared__ f32x2 mlbox[NT];
  __shared__ int special[4];  // by wave: V of a masked block held infinities or NaN
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31, g = lane >> 5;
  auto kslot = [&](int t) { return smem + (t & 1) * TILE; };
  auto vslot = [&](int t) { return smem + (2 + (t & 1)) * TILE; };

  // kv heads fastest: with a multiple of 8 of them, id % 8 (the XCD) fixes the
  // head modulo 8 and the tiles of a head share an L2
  const Plan plan = make_plan(args, lane);
  const int idx = quotient((int)blockIdx.x, args.Hk, args.Hk_inv);
  const int hk = (int)blockIdx.x - idx * args.Hk;
  Item it;
  if (!find_item<MX>(args, plan, lane, idx, 0, &it)) return;
  const PagedArgs &a = MX ? arguments() : args;
  const int rows = it.n * a.group;
  const int off = it.len - it.n;  // place of the sequence's first new token
  const int r0 = it.tile * BM + w * 32;

  // this lane's row: query head hk * group + hr of token tok, at place pos
  const int row = r0 + lq;
  const int tok = quotient(min(row, rows - 1), a.group, a.group_inv), hr = min(row, rows - 1) - tok * a.group;
  const int pos = off + tok;
  // blocks seen by rows up to r: through the place of its token
  auto blocks_to = [&](int r) {
    const int last = off + quotient(min(r, rows - 1), a.group, a.group_inv);
    return last < 0 ? 0 : last / BN + 1;
  };
  const int all = blocks_to(it.tile * BM + BM - 1);
  const int lo_tile = __builtin_amdgcn_readfirstlane(
      off + quotient(it.tile * BM, a.group, a.group_inv));
  // blocks before the first row's window
  const int before = MOD && a.window ? max(lo_tile - a.window + 1, 0) / BN : 0;
  const int span = max(all - before, 0);
  const int per = it.splits > 1 ? (span + it.splits - 1) / it.splits : span;
  const int kb0 = __builtin_amdgcn_readfirstlane(before + it.split * per);
  const int nv = __builtin_amdgcn_readfirstlane(min(max(all - kb0, 0), per));
  if (rows - it.tile * BM <= NARROW) {
    if constexpr (MX) {
      if (rows - it.tile * BM <= 16)
        narrow_mx<E, HD, MOD, 1>(it, hk, w, lane, kb0, nv, smem, mlbox);
      else
        narrow_mx<E, HD, MOD, 2>(it, hk, w, lane, kb0, nv, smem, mlbox);
    } else {
      narrow_item<E, HD, POOL, MOD>(a, it, hk, w, lane, kb0, nv, smem, mlbox);
    }
    return;
  }
  if (lane == 0) special[w] = 0;
  auto block = [&](int t) { return BACK ? nv - 1 - t : t; };  // of the t-th step
  const int nkw = __builtin_amdgcn_readfirstlane(
      r0 < rows ? min(max(blocks_to(r0 + 31) - kb0, 0), nv) : 0);
  const int lo_w = __builtin_amdgcn_readfirstlane(off + quotient(min(r0, rows - 1), a.group, a.group_inv));
  const int hi_w = __builtin_amdgcn_readfirstlane(off + quotient(min(r0 + 31, rows - 1), a.group, a.group_inv));

  const char *kp = a.k + hk * a.kps1, *vp = a.v + hk * a.vps1;
  const int32_t *tab = a.btab + (int64_t)it.b * a.maxp;
  const int last_key = it.len - 1;

  // the window of the block table: lane j holds entry tab0 + j; the copies' pages
  // only ever move on (BACK: back)
  int tab0 = 0, tabv = 0;
  auto load_tab = [&](int first) {
    tab0 = first;
    const int j = first + lane;
    tabv = j < a.maxp ? tab[j] : 0;
  };
  // the wave's run of block t: its byte offset in each pool, the tokens of it that
  // exist less one (a run behind the end takes the last run), its page, and its
  // first place there
  auto run_at = [&](int t, int64_t *ko, int64_t *vo, int *most, int *in, int *at) {
    int run = (kb0 + block(t)) * (BN / 16) + w;
    const int key = min(run * 16, last_key & ~15);
    run = key >> 4;
    int index, rest;
    page_of(a, run, &index, &rest);
    if (BACK ? index < tab0 : index - tab0 >= 64) {
      load_tab(BACK ? max(index - 63, 0) : index);
      settle(tabv);
    }
    int page = __builtin_amdgcn_readlane(tabv, index - tab0);
    page = min(max(page, 0), a.npages - 1);
    *ko = page * a.kps0 + (int64_t)(rest * 16) * a.ktok;
    *vo = page * a.vps0 + (int64_t)(rest * 16) * a.vtok;
    *most = last_key - key;
    *in = page;
    *at = rest * 16;
  };

  // 16-bit pools: chunk c of the wave's copy is rows RPC c + lane / UNITS of its
  // run, straight into LDS; rows behind the sequence's end re-read its last
  const int crow = lane / TL::UNITS, cunit = lane & (TL::UNITS - 1);
  uint32_t koff[CHUNKS], voff[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int r = 16 * w + crow + RPC * c;
    koff[c] = (uint32_t)((crow + RPC * c) * a.ktok + (cunit ^ tile_swizzle<HD, false>(r)) * 16);
    voff[c] = (uint32_t)((crow + RPC * c) * a.vtok + (cunit ^ tile_swizzle<HD, true>(r)) * 16);
  }
  auto copy = [&](const char *base, const uint32_t *offs, int64_t tokb, int most, bool is_v,
                  const uint8_t *tile) {
    if (most >= 15) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        dma16_sbase(base, offs[c], lds_offset(tile + (CHUNKS * w + c) * 1024));
    } else {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int r = crow + RPC * c;
        const int u = cunit ^ (is_v ? tile_swizzle<HD, true>(16 * w + r)
                                    : tile_swizzle<HD, false>(16 * w + r));
        dma16(base, (uint32_t)(min(r, most) * tokb + u * 16),
              lds_offset(tile + (CHUNKS * w + c) * 1024));
      }
    }
  };
  // E4M3 pools: 16 codes per lane and load, two 16-byte units of bf16. The rows of
  // 16 lanes, which one cycle writes to LDS, have units of both parities: K's by
  // its swizzle, V's by an order of rows that alternates bit 2 and a swizzle that
  // brings that bit in (without it half the LDS cycles were conflicts; counted, a
  // quarter of them still are, none with 16-bit pools)
  constexpr int LPR8 = HD / 16, ROWS8 = 64 / LPR8, N8 = 16 / ROWS8;
  const int krow8 = lane / LPR8;
  const int vrow8 = HD == 128 ? krow8 >> 1 | (krow8 & 1) << 2
                              : (krow8 & 9) | (krow8 & 2) << 1 | (krow8 & 4) >> 1;
  auto vswz8 = [](int r) { return tile_swizzle<HD, true>(r) | ((r >> 2) & 1); };
  u32x4 k8[N8], v8[N8];
  auto load8 = [&](const char *base, int64_t tokb, int most, int row8, u32x4 *dst) {
#pragma unroll
    for (int c = 0; c < N8; ++c) {
      const int r = row8 + ROWS8 * c;
      dst[c] = *(const u32x4 *)(base + (uint32_t)(min(r, most) * (int)tokb + (lane % LPR8) * 16));
    }
  };
  // where a lane's first 16 bytes go in a tile; the other half of its codes is the
  // neighbouring unit, and its second row 8 rows on (K's swizzle then differs in
  // unit bit 3). Kept as one register each and worked out anew for every tile: the
  // matrix products need the registers
  auto place8 = [&](int row8, int z) {
    return (16 * w + row8) * ROWB + (((2 * (lane % LPR8)) ^ z) << 4);
  };
  int kput = place8(krow8, tile_swizzle<HD, false>(16 * w + krow8));
  int vput = place8(vrow8, vswz8(16 * w + vrow8));
  auto store8 = [&](const u32x4 *src, const uint8_t *tile, bool is_v) {
    int at = is_v ? vput : kput;
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int c = 0; c < N8; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x2 lo = widen4(src[c][2 * h]), hi = widen4(src[c][2 * h + 1]);
        *(u32x4 *)(uint8_t *)(tile + ROWS8 * c * ROWB + (at ^ (16 * h) ^ (is_v ? 0 : 128 * c))) =
            u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
  };
  // MXFP4 pools: a lane takes a quarter of a row's codes, with their scale. Eight
  // neighbouring lanes write at once, over 128 bytes: two quarters (head_dim 64: four) of
  // rows whose swizzle differs in the unit's lowest bits
  const int mpart = lane_bits(lane, HD == 128 ? 0x30 : 0x10);
  const int mrow = lane_bits(lane, HD == 128 ? 0x5421 : 0x5423);
  const int mvrow = lane_bits(lane, HD == 128 ? 0x2154 : 0x5243);
  constexpr int MB = HD / 8;  // bytes of codes a lane takes
  typedef typename std::conditional<HD == 128, u32x4, u32x2>::type mx_t;
  mx_t kmx, vmx;
  row_scales<HD> ksb = {}, vsb = {};
  const char *const ksp = MX ? (const char *)a.kmx + hk * a.kss1 : nullptr;
  const char *const vsp = MX ? (const char *)a.vmx + hk * a.vss1 : nullptr;
  const int mblk = HD == 128 ? mpart : mpart >> 1;
  auto mxswz = [](int r) { return tile_swizzle<HD, true>(r) | ((r >> 2) & 3); };
  const int kmput = (16 * w + mrow) * ROWB +
                    (((MB / 4 * mpart) ^ tile_swizzle<HD, false>(16 * w + mrow)) << 4);
  const int vmput = (16 * w + mvrow) * ROWB + (((MB / 4 * mpart) ^ mxswz(mvrow)) << 4);
  const uint32_t kmoff = mrow * (uint32_t)a.ktok + mpart * MB, ksoff = mrow * (uint32_t)a.kstok;
  const uint32_t vmoff = mvrow * (uint32_t)a.vtok + mpart * MB, vsoff = mvrow * (uint32_t)a.vstok;
  // the wave's run of a block: its page and first place in it (of its rows behind the
  // end: narrow_mx). V's run of a block is K's, looked up before.
  int mpage = 0, mplace = 0;
  auto look_mx = [&](int t) {
    int64_t ko, vo;
    int most;
    run_at(t, &ko, &vo, &most, &mpage, &mplace);
  };
  auto load_k_mx = [&]() {
    kmx = *(const mx_t *)(mx_at(kp, mpage, a.kps0, mplace, a.ktok) + offset(kmoff));
    ksb = *(const row_scales<HD> *)(mx_at(ksp, mpage, a.kss0, mplace, a.kstok) + offset(ksoff));
  };
  auto load_v_mx = [&]() {
    vmx = *(const mx_t *)(mx_at(vp, mpage, a.vps0, mplace, a.vtok) + offset(vmoff));
    vsb = *(const row_scales<HD> *)(mx_at(vsp, mpage, a.vss0, mplace, a.vstok) + offset(vsoff));
  };
  auto store_mx = [&](mx_t codes, float scale, const uint8_t *tile, int put) {
    asm volatile("" : "+v"(put));
#pragma unroll
    for (int u = 0; u < MB / 4; ++u)
      *(u32x4 *)(uint8_t *)(tile + (put ^ (u << 4))) = widen8<E>(codes[u], scale);
  };
  auto put_k_mx = [&](int t) { store_mx(whole(kmx), scale_of(ksb, mblk), kslot(t), kmput); };
  auto put_v_mx = [&](int t) {
    const int key = (kb0 + block(t)) * BN + 16 * w + mvrow;
    const float held = scale_of(vsb, mblk);
    store_mx(whole(vmx), key <= last_key ? held : 0.0f, vslot(t), vmput);
  };
  auto load_k = [&](int t) {
    int64_t ko, vo;
    int most, page, at;
    run_at(t, &ko, &vo, &most, &page, &at);
    if constexpr (FP8)
      load8(kp + ko, a.ktok, most, krow8, k8);
    else
      copy(kp + ko, koff, a.ktok, most, false, kslot(t));
  };
  auto load_v = [&](int t) {
    int64_t ko, vo;
    int most, page, at;
    run_at(t, &ko, &vo, &most, &page, &at);
    if constexpr (FP8)
      load8(vp + vo, a.vtok, most, vrow8, v8);
    else
      copy(vp + vo, voff, a.vtok, most, true, vslot(t));
  };
  // E4M3: what load_k / load_v have in registers to LDS
  auto put_k = [&](int t) {
    if constexpr (FP8) store8(k8, kslot(t), false);
  };
  auto put_v = [&](int t) {
    if constexpr (FP8) store8(v8, vslot(t), true);
  };
  auto put_next = [&](int jb) {
    if constexpr (MX) {
      // in every block (past the last into slots that none reads, of the last again): a
      // branch around the loads would have their registers copied, and so waited for,
      // behind it
      put_v_mx(jb + 1);
      put_k_mx(jb + 2);
      load_v_mx();
      look_mx(min(jb + 3, nv - 1));
      load_k_mx();
    } else {
      if (jb + 1 < nv) put_v(jb + 1);
      if (jb + 2 < nv) put_k(jb + 2);
    }
  };
  // the wave's own rows of a V tile, before the others read them (16-bit pools:
  // their copy has landed; E4M3: they have been stored)
  const int hi_tile = __builtin_amdgcn_readfirstlane(
      off + quotient(min(it.tile * BM + BM, rows) - 1, a.group, a.group_inv));
  auto scrub_v = [&](int t) {
    const int key = (kb0 + block(t)) * BN;
    const bool cut = MOD && a.window && key + a.window <= hi_tile;  // at some row's window
    if (key + BN - 1 <= lo_tile && !cut) return;
    asm volatile("" ::: "memory");  // no read before the copy's wait
    const bool found =
        Special<E, false>::template scrub<CHUNKS>(vslot(t) + CHUNKS * w * 1024, lane);
    if (found && lane == 0) special[w] = 1;
  };
  if (nv > 0) {
    int index, rest;
    page_of(a, BACK ? min((kb0 + nv) * (BN / 16) - 1, last_key >> 4) : kb0 * (BN / 16), &index, &rest);
    load_tab(BACK ? max(index - 63, 0) : index);
  }

  // Q^T operand: k-step st covers head_dim 16 st + 8 g .. +7 of the row
  u32x4 qf[NST];
  {
    const uint16_t *qp = a.q + (int64_t)(it.row0 + tok) * a.qs0 +
                         (int64_t)(hk * a.group + hr) * a.qs1 + 8 * g;
#pragma unroll
    for (int st = 0; st < NST; ++st)
      qf[st] = row < rows ? *(const u32x4 *)(qp + 16 * st) : u32x4{0, 0, 0, 0};
  }
  // E4M3: the scales of the block-table entries sc0 .. sc0 + 63, a lane each
  int sc0 = 0;
  float kscv = 0.0f, vscv = 0.0f;
  auto load_scales = [&](int first) {
    sc0 = first;
    const int j = first + lane;
    const int page = min(max(j < a.maxp ? tab[j] : 0, 0), a.npages - 1);
    kscv = a.ksc[(int64_t)page * a.Hk + hk];
    vscv = a.vsc[(int64_t)page * a.Hk + hk];
  };
  if constexpr (FP8) {
    if (nv > 0) load_scales(tab0);
    settle(kscv);
    settle(vscv);
  }
  const float unit = FP8 ? scale_unit(vscv) : 1.0f, unit_inv = FP8 ? scalar(__builtin_amdgcn_rcpf(unit)) : 1.0f;
  float slope2 = 0.0f;
  if constexpr (MOD)
    if (a.slopes) slope2 = a.slopes[hk * a.group + hr] * kLog2e;
  settle(slope2);
  // Q and the table land before the first copy is issued
#pragma unroll
  for (int st = 0; st < NST; ++st) settle(qf[st]);
  settle(tabv);
  if (nv > 0) {
    if constexpr (MX) {
      look_mx(0);
      load_k_mx();
      load_v_mx();
      put_k_mx(0);
      look_mx(min(1, nv - 1));
      load_k_mx();
      put_v_mx(0);
      put_k_mx(1);
      load_v_mx();
      look_mx(min(2, nv - 1));
      load_k_mx();
    } else {
      load_k(0);
      load_v(0);
      put_k(0);
      if (nv > 1) load_k(1);
      put_v(0);
      if (nv > 1) put_k(1);
    }
  }

  // per-lane LDS byte offsets of the operand reads
  int ka[NST];  // K: row lq (+32 kb), logical unit 2 st + g
#pragma unroll
  for (int st = 0; st < NST; ++st)
    ka[st] = lq * ROWB + (((2 * st + g) ^ tile_swizzle<HD, false>(lq)) << 4);
  int va[NB];  // V^T: transpose read, rows 4 g + i (+16 c + 8 t), columns 32 nb + 16 dh + 4 q
  {
    const int s16 = lane & 15, i = s16 >> 2, q = s16 & 3, dh = (lane >> 4) & 1;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      va[nb] = (4 * g + i) * ROWB +
               (((4 * nb + 2 * dh + (q >> 1)) ^ (tile_swizzle<HD, true>(i) | (CODES ? g : 0))) << 4) +
               8 * (q & 1);
  }

  f32x16 o[NB];
  f32x16 s[2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.0f;
  float m = kNegFltMax, lsum = 0.0f;
  bool large = false;
  const f32x16 zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  // The A operand of MFMA i = 2 st + kb of S^T = K.Q^T (32 keys x 16 head_dim)
  auto k_operand = [&](const uint8_t *kt, int i) {
    return *(const u32x4 *)(kt + (i & 1) * 32 * ROWB + ka[i >> 1]);
  };
  // S^T of one key block, its first two A operands already read (k0, k1)
  auto qk_from = [&](const uint8_t *kt, const u32x4 &k0, const u32x4 &k1) {
    // operand reads run three MFMAs ahead. The order is spelled out, not left to
    // the scheduler, which gave up on it where registers were short: E4M3 pools
    // then waited for every read (2000 new rows behind 6000, 32 heads of 128 over
    // 8: 277 us against 257)
    u32x4 next[4] = {k0, k1, k_operand(kt, 2)};
#pragma unroll
    for (int i = 0; i < NQK; ++i) {
      if (i + 3 < NQK) next[(i + 3) & 3] = k_operand(kt, i + 3);
      __builtin_amdgcn_sched_barrier(0);
      s[i & 1] = E::mfma32(as_vec8<V8>(next[i & 3]), as_vec8<V8>(qf[i >> 1]),
                           i < 2 ? zero16 : s[i & 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The A operand of P.V step st (V^T: head_dim rows 32 nb .., keys 16 c ..)
  auto v_operand = [&](const uint8_t *vt, int st) {
    const int c = st / NB, nb = st % NB;
    const u32x2 a0 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + 16 * c * ROWB + va[nb]));
    // (MXFP4's swizzle has bit 3 of the row in bit 1)
    const u32x2 a1 = __builtin_bit_cast(
        u32x2, lds_read_tr16(vt + (16 * c + 8) * ROWB + (va[nb] ^ (MX ? 32 : 0))));
    return u32x4{a0[0], a0[1], a1[0], a1[1]};
  };

  wait_vmem();
  if (nv > 0) scrub_v(0);
  __syncthreads();
  if (nv > 0 && block(0) < nkw) qk_from(kslot(0), k_operand(kslot(0), 0), k_operand(kslot(0), 1));
  __syncthreads();  // every wave is done with K slot 0 before it is refilled

  for (int jb = 0; jb < nv; ++jb) {
    // K of block jb + 2 goes to the slot block jb's K has left, V of block
    // jb + 1 to the slot of block jb - 1's V (E4M3: in registers until the softmax
    // is done, and written then, which the matrix products hide: 247 us against 254)
    if (!MX && jb + 1 < nv) load_v(jb + 1);
    if (!MX && jb + 2 < nv) load_k(jb + 2);
    const bool live = block(jb) < nkw;
    const bool next_live = jb + 1 < nv && block(jb + 1) < nkw;
    const uint8_t *const vt = vslot(jb);
    u32x4 vp0 = {}, vp1 = {}, pf[4] = {};
    if (live) {
      // the first two V^T operands of this block's P.V, read before the softmax
      // (codes and shaped scores leave no registers for them until then)
      if constexpr (!(CODES && MOD)) {
        vp0 = v_operand(vt, 0);
        vp1 = v_operand(vt, 1);
      }
      const int key0 = (kb0 + block(jb)) * BN;
      float sc = a.scale2;
      // E4M3: V's scales (over scale_unit) meet P. Over a block within one page K's scale goes with
      // the score scale and V's into the exponent (lv), so they cost no operation
      // an element; the sum is then of scaled p, and unscaled by one product (iv).
      // Across pages, or where the exponent would not hold V's scale or K's is not
      // positive and finite, each run's are multiplied in: K's here, before the mask
      // (such a scale must not meet -inf), V's with P.
      float vs[4] = {1.0f, 1.0f, 1.0f, 1.0f}, v0 = 1.0f, lv = 0.0f, iv = 1.0f;
      bool apart = false;
      if constexpr (FP8) {
        int index, rest;
        page_of(a, key0 >> 4, &index, &rest);
        if (BACK ? index < sc0 : index + 3 - sc0 >= 64) {
          load_scales(BACK ? max(index - 60, 0) : index);
          // here, not where they are read: that would drain the loads above too
          settle(kscv);
          settle(vscv);
        }
        auto scale_at = [&](float v, int i) {
          return __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i - sc0));
        };
        const int runs = last_key / 16 - (key0 >> 4);  // runs behind the end take the last one's
        const float k0 = sc * scale_at(kscv, index);
        v0 = unit_inv * scale_at(vscv, index);
        apart = (rest + 3 >= a.ps16 && runs > 0) || !(v0 >= 0x1p-64f && v0 <= 0x1p64f) ||
                !(k0 > 0.0f && k0 <= 3.4e38f);
        if (apart) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float ks = sc * scale_at(kscv, index);
            vs[c] = unit_inv * scale_at(vscv, index);
#pragma unroll
            for (int r = 0; r < 8; ++r) s[c >> 1][8 * (c & 1) + r] *= ks;
            if (c < runs && ++rest == a.ps16) {
              rest = 0;
              ++index;
            }
          }
          sc = 1.0f;
        } else {
          sc = k0;
          lv = __builtin_amdgcn_logf(v0);
          iv = __builtin_amdgcn_rcpf(v0);
        }
      }
      // element (kb, r) holds key key0 + 4 g + c with c = 32 kb + 8 (r >> 2)
      // + (r & 3): it is masked when c passes the row's own place
      const int lim = pos - key0 - 4 * g;
      const bool edge = MOD && a.window && key0 + a.window <= hi_w;  // of some row's window
      float rs = 0.0f;
      // Capped and biased scores, of blocks that every row sees whole and whose maxima
      // stay where they were: the cap's polynomial and the bias are part of the exponent,
      // 5 vector instructions an element and 1, where shape() takes 8 and 3
      bool done = false;
      if constexpr (FOLD) {
        done = jb > 0 && key0 + BN - 1 <= lo_w && !edge;
        if (done && a.cap2 != 0.0f) {
          float big = 0.0f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(s[kb][r]));
          done = !__any(!(big <= a.cap_most));
        }
        if (done) {
          // (NaN where huge(), so that the block is done the other way: a comparison and a
          // branch here cost the biased chunk 5%)
          const float nm = fmaf(m * 0x1p104f, 0.0f, -m);
          const float b0 = fmaf(slope2, (float)-lim, nm);
          auto expo_of = [&](auto score) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int kb = c >> 1, r = 8 * (c & 1) + 2 * i, at = 32 * kb + 8 * (r >> 2) + (r & 3);
                const float p0 = fast_exp2(score(s[kb][r], (float)at));
                const float p1 = fast_exp2(score(s[kb][r + 1], (float)(at + 1)));
                rs = c + i == 0 ? p0 : rs + p0;
                rs += p1;
                pf[c][i] = E::pack2(p0, p1);
              }
          };
          auto capped = [&](float x, float b) {
            const float w = x * x;
            float p = fmaf(w, a.capq[3], a.capq[2]);
            p = fmaf(w, p, a.capq[1]);
            return fmaf(x, fmaf(w, p, a.capq[0]), b);
          };
          if (a.cap2 != 0.0f && a.slopes)
            expo_of([&](float x, float c) { return capped(x, fmaf(slope2, c, b0)); });
          else if (a.cap2 != 0.0f)
            expo_of([&](float x, float) { return capped(x, nm); });
          else if (a.slopes)
            expo_of([&](float x, float c) { return fmaf(x, sc, fmaf(slope2, c, b0)); });
          else
            expo_of([&](float x, float) { return fmaf(x, sc, nm); });
          done = !__any(!(rs <= kSumCap));
        }
      }
      if (!FOLD || !done) {
        if constexpr (MOD) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) shape<16>(a, slope2, sc, (float)-lim, 32 * kb, s[kb]);
          sc = 1.0f;
        }
        if (key0 + BN - 1 > lo_w) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * kb + 8 * (r >> 2) + (r & 3) > lim) s[kb][r] = -INFINITY;
        }
        if (edge) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * kb + 8 * (r >> 2) + (r & 3) <= lim - a.window) s[kb][r] = -INFINITY;
        }
        // p = 2^(s sc - m) for the block, packed for P.V, and the lane's sum
        auto expo = [&]() {
          const float nm = FP8 ? lv - m : -m;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int kb = c >> 1, hh = c & 1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p0 = fast_exp2(fmaf(s[kb][8 * hh + 2 * i], sc, nm));
              const float p1 = fast_exp2(fmaf(s[kb][8 * hh + 2 * i + 1], sc, nm));
              rs = c + i == 0 ? p0 : rs + p0;
              rs += p1;
              pf[c][i] = E::pack2(p0, p1);  // 16 bits, for P.V alone
            }
          }
          if constexpr (FP8) {
            rs *= iv;
            if (apart) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float p0 = fast_exp2(fmaf(s[c >> 1][8 * (c & 1) + 2 * i], sc, nm));
                  const float p1 = fast_exp2(fmaf(s[c >> 1][8 * (c & 1) + 2 * i + 1], sc, nm));
                  // (a masked key's page may hold any scale)
                  pf[c][i] = E::pack2(p0 == 0.0f ? 0.0f : p0 * vs[c], p1 == 0.0f ? 0.0f : p1 * vs[c]);
                }
            }
          }
        };
        auto raise_max = [&](float slack) {  // m to the block's max where that passes m + slack
          float mx = -INFINITY;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
          mx = pair_max(mx);
          const float m_blk = mx * sc;
          if (__any(m_blk > m + slack)) {
            const float m_new = fmaxf(m, m_blk);
            const float alpha = fast_exp2(m - m_new);
            lsum *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int r = 0; r < 16; ++r) o[nb][r] *= alpha;
            m = m_new;
            if constexpr (!MOD || FP8) large = huge(m);
          }
        };
        auto products = [&]() {  // rounded, where huge() asks for it
          if ((!MOD || FP8) && __builtin_expect(large, 0)) {
            if constexpr (!MOD) {
#pragma unroll
              for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[kb][r] *= sc;
              sc = 1.0f;
            }
            if (FP8 && !apart) {  // such an exponent has no room for V's scale
              apart = true;
#pragma unroll
              for (int c = 0; c < 4; ++c) vs[c] = v0;
              lv = 0.0f;
              iv = 1.0f;
            }
          }
        };
        if constexpr (HD == 64) {
          raise_max(0.0f);
          products();
          expo();
        } else {
          // the block max is only formed when it can matter: past the first block,
          // a lane sum of at most 2^kSlack bounds every p by it, and m keeps
          bool full = jb == 0;
          if (!full) {
            products();
            expo();
            full = __any(!(rs <= kSumCap));
          }
          if (full) {
            // (BACK: the first block may show a row few keys; a maximum left below the
            // next ones' would bring every block here)
            raise_max(BACK ? 0.0f : kSlack);
            products();
            expo();
          }
        }
      }
      lsum += rs;
    }
    if constexpr (CODES) put_next(jb);
    if (live) {
      // O^T += V^T P^T, then the next block's S^T, at raised issue priority
      __builtin_amdgcn_s_setprio(1);
      // (reads run two MFMAs ahead, as above; the last are the next block's first two
      // K operands: past the last block those are stale and dropped)
      if constexpr (CODES && MOD) {
        vp0 = v_operand(vt, 0);
        vp1 = v_operand(vt, 1);
      }
      u32x4 next[4] = {vp0, vp1};
#pragma unroll
      for (int st = 0; st < NPV; ++st) {
        next[(st + 2) & 3] = st + 2 < NPV ? v_operand(vt, st + 2)
                                          : k_operand(kslot(jb + 1), st + 2 - NPV);
        __builtin_amdgcn_sched_barrier(0);
        o[st % NB] = E::mfma32(as_vec8<V8>(next[st & 3]), as_vec8<V8>(pf[st / NB]), o[st % NB]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (next_live) qk_from(kslot(jb + 1), next[NPV & 3], next[(NPV + 1) & 3]);
      __builtin_amdgcn_s_setprio(0);
    } else if (BACK && next_live) {  // the wave's rows end before this block's keys
      const uint8_t *kt = kslot(jb + 1);
      qk_from(kt, k_operand(kt, 0), k_operand(kt, 1));
    }
    if constexpr (!CODES) wait_vmem();
    if (jb + 1 < nv) scrub_v(jb + 1);
    __syncthreads();
  }

  if constexpr (FP8) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) o[nb] *= unit;
  }
  const float ltot = pair_sum(lsum);
  if (__builtin_expect(special[0] | special[1] | special[2] | special[3], 0))
    add_special<E, HD, POOL>(a, it, hk, (MOD && a.window ? kb0 : max(kb0, lo_tile / BN)) * BN,
                             min((kb0 + nv) * BN, it.len), pos, g, o);
  if (row >= rows) return;
  if (it.splits > 1) {  // this split's state, for attn_paged_combine
    const int64_t part =
        ((int64_t)(it.part + it.split) * a.Hk + hk) * a.prows + (row - it.tile * BM);
    if (nv > 0) {
      float *op = a.po + part * HD + 4 * g;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int rq = 0; rq < 4; ++rq)
          *(f32x4 *)(op + 32 * nb + 8 * rq) =
              f32x4{o[nb][4 * rq], o[nb][4 * rq + 1], o[nb][4 * rq + 2], o[nb][4 * rq + 3]};
    }
    if (g == 0) *(f32x2 *)(a.pml + part * 2) = f32x2{m, ltot};
    return;
  }
  // O = acc / l, rounded to the input type (by a product: 1.5 ulp of fp32 off at most,
  // and an infinity stays one)
  const float inv = ltot == 0.0f ? 0.0f : 1.0f / ltot;
  const int64_t t = it.row0 + tok;
  uint16_t *op = a.o + t * a.os0 + (int64_t)(hk * a.group + hr) * a.os1 + 4 * g;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const u32x2 pk = {E::pack2(o[nb][4 * rq] * inv, o[nb][4 * rq + 1] * inv),
                        E::pack2(o[nb][4 * rq + 2] * inv, o[nb][4 * rq + 3] * inv)};
      *(u32x2 *)(op + 32 * nb + 8 * rq) = pk;
    }
  if (g == 0 && a.lse)
    a.lse[t * a.Hq + hk * a.group + hr] = ltot == 0.0f ? -INFINITY : row_lse(m, ltot);
}

// Combine of the cut tiles' states: M = max m_s, l = sum 2^(m_s - M) l_s, O = sum
// 2^(m_s - M) O_s / l. HD / 4 lanes per row, four elements each, and SG groups of
// them per row, group g taking splits g, g + SG, .. four at a time; a work-group
// takes `take` rows of a tile. A split with l_s = 0 (no visible key) may have left
// no O_s and is passed over.
template <class E, int HD, int SG>
__global__ __launch_bounds__(NT) void attn_paged_combine(PagedArgs a, int take) {
  constexpr int LPR = HD / 4, ROWS = NT / LPR / SG;
  __shared__ float st[SG > 1 ? NT : 1][6];
  const int lane = threadIdx.x & 63;
  const int grp = threadIdx.x / LPR, sg = grp % SG, d = 4 * (threadIdx.x % LPR);
  const Plan plan = make_plan(a, lane);
  const int idx = quotient((int)blockIdx.x, a.Hk, a.Hk_inv), hk = (int)blockIdx.x - idx * a.Hk;
  Item it;
  if (!find_item(a, plan, lane, idx, take, &it)) return;
  const int r0 = it.split;
  const int rows = min(min(it.n * a.group - it.tile * BM, BM), r0 + take);
  const int64_t step = (int64_t)a.Hk * a.prows;
  for (int rr = r0; rr < rows; rr += ROWS) {
    const int r = rr + grp / SG;
    const bool live = r < rows;
    const int64_t part = ((int64_t)it.part * a.Hk + hk) * a.prows + min(r, rows - 1);
    float M = kNegFltMax, l = 0.0f;
    f32x4 acc = {0, 0, 0, 0};
    auto join = [&](float m1, float l1, f32x4 o1) {
      if (l1 == 0.0f) return;
      const float m_new = fmaxf(M, m1);
      const float w0 = fast_exp2(M - m_new), w1 = fast_exp2(m1 - m_new);
      l = l * w0 + l1 * w1;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = acc[k] * w0 + o1[k] * w1;
      M = m_new;
    };
    for (int s = sg; s < it.splits; s += 4 * SG) {
      f32x2 ml[4];
      f32x4 os[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t at = part + min(s + i * SG, it.splits - 1) * step;
        ml[i] = *(const f32x2 *)(a.pml + at * 2);
        os[i] = *(const f32x4 *)(a.po + at * HD + d);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s + i * SG < it.splits) join(ml[i][0], ml[i][1], os[i]);
    }
    if constexpr (SG > 1) {
      float *mine = st[threadIdx.x];
      mine[0] = M;
      mine[1] = l;
#pragma unroll
      for (int k = 0; k < 4; ++k) mine[2 + k] = acc[k];
      __syncthreads();
    }
    if (sg == 0 && live) {
#pragma unroll
      for (int i = 1; i < SG; ++i) {
        const float *o = st[threadIdx.x + i * LPR];
        join(o[0], o[1], f32x4{o[2], o[3], o[4], o[5]});
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int row = it.tile * BM + r;
      const int tok = quotient(row, a.group, a.group_inv);
      const int h = hk * a.group + row - tok * a.group;
      const int64_t t = it.row0 + tok;
      *(u32x2 *)(a.o + t * a.os0 + h * a.os1 + d) =
          u32x2{E::pack2(acc[0] * inv, acc[1] * inv), E::pack2(acc[2] * inv, acc[3] * inv)};
      if (d == 0 && a.lse) a.lse[t * a.Hq + h] = l == 0.0f ? -INFINITY : row_lse(M, l);
    }
    if constexpr (SG > 1) __syncthreads();  // the states are read before the next rows'
  }
}

// a window that no sequence outgrows hides nothing
inline bool windowed(const PagedAttnLaunch &L) { return L.window > 0 && L.window < L.seq_kv; }
inline bool shaped(const PagedAttnLaunch &L) { return windowed(L) || L.slopes || L.softcap > 0.0f; }

inline PagedArgs paged_args(const PagedAttnLaunch &L) {
  PagedArgs a = {};
  const int64_t size = L.pool == WIDE ? 2 : 1;
  a.q = (const uint16_t *)L.q;
  a.k = (const char *)L.k;
  a.v = (const char *)L.v;
  a.ksc = (const float *)L.k_scales;
  a.vsc = (const float *)L.v_scales;
  a.btab = L.block_table;
  a.cu = L.cu_seqlens;
  a.lens = L.seq_lens;
  a.o = (uint16_t *)L.o;
  a.lse = L.lse;
  a.qs0 = L.qs[0]; a.qs1 = L.qs[1];
  a.os0 = L.os[0]; a.os1 = L.os[1];
  a.kps0 = L.kps[0] * size; a.kps1 = L.kps[1] * size; a.ktok = L.kps[2] * size;
  a.vps0 = L.vps[0] * size; a.vps1 = L.vps[1] * size; a.vtok = L.vps[2] * size;
  a.kmx = (const uint8_t *)L.k_scales;
  a.vmx = (const uint8_t *)L.v_scales;
  a.kss0 = L.kss[0]; a.kss1 = L.kss[1]; a.kstok = L.kss[2];
  a.vss0 = L.vss[0]; a.vss1 = L.vss[1]; a.vstok = L.vss[2];
  a.T = (int32_t)L.tokens;
  a.B = (int32_t)L.batch;
  a.Hq = (int32_t)L.heads_q;
  a.Hk = (int32_t)L.heads_kv;
  a.group = (int32_t)(L.heads_q / L.heads_kv);
  a.Lmax = (int32_t)L.seq_kv;
  a.maxp = (int32_t)L.max_pages;
  a.npages = (int32_t)L.num_pages;
  a.ps16 = (int32_t)(L.page_size / 16);
  a.ps16_inv = 0xffffffffu / (uint32_t)a.ps16;
  a.group_inv = 0xffffffffu / (uint32_t)a.group;
  a.Hk_inv = 0xffffffffu / (uint32_t)a.Hk;
  const Room room = room_of(L);
  a.items = (int32_t)room.items;
  a.slots = (int32_t)room.slots;
  a.parts = (int32_t)room.parts;
  a.prows = (int32_t)part_rows(L);
  a.longest = long_first(L);
  a.po = (float *)L.workspace;
  a.pml = a.po + (size_t)a.parts * L.heads_kv * a.prows * L.head_dim;
  a.scale2 = L.scale_log2;
  if (windowed(L)) {
    a.window = (int32_t)L.window;
    const int64_t keys = L.window - 1 + (BM - 1) / a.group + 2;  // a tile's rows' windows
    a.blocks_1 = (uint32_t)((keys + BN - 2) / BN + 2);
  }
  a.slopes = L.slopes;
  if (L.softcap > 0.0f) {
    a.cap2 = L.softcap * kLog2e;
    a.cap_inv = 1.0f / a.cap2;
    const float c[4] = {0x1.fffffep-1f, -0x1.5551cap-2f, 0x1.1011b4p-3f, -0x1.8b7eacp-5f};
    // of the products themselves, where the powers of u stay ordinary numbers, and so do
    // their products with the cap (an infinite factor would bring scores to -inf)
    const double u = (double)L.scale_log2 / a.cap2;
    double power = u * a.cap2;
    for (int i = 0; i < 4; ++i) {
      a.capp[i] = c[i] * a.cap2;
      a.capq[i] = (float)(c[i] * power);
      power *= u * u;
    }
    a.cap_most = u >= 0x1p-16 && u <= 0x1p16 && std::isfinite(a.capq[3]) ? (float)(kCapPoly / u)
                                                                         : -1.0f;
  }
  return a;
}

template <class E, int HD, int POOL, bool MOD>
hipError_t launch_t(const PagedArgs &a, const PagedAttnLaunch &L, hipStream_t s) {
  hipLaunchKernelGGL((attn_paged<E, HD, POOL, MOD>), dim3((unsigned)(a.items * L.heads_kv)), dim3(NT), 0,
                     s, a);
  if (a.parts) {
    auto combine = [&](auto G) {
      constexpr int SG = decltype(G)::value;
      constexpr int ROWS = NT / (HD / 4) / SG;
      // rows of cut tiles at most; runs of them, short ones (a wait for memory
      // each) as long as the GPU holds the work-groups at once
      const int64_t tiles = a.parts / 2;
      const int64_t rows = std::min<int64_t>(L.tokens * a.group, tiles * BM);
      const int64_t ends = std::min(std::min(L.batch, tiles), rows);  // a run short of `take` each
      int take = ROWS;
      auto runs = [&]() { return (rows + (take - 1) * ends) / take; };
      while (take < BM && runs() * L.heads_kv > 2048) take *= 2;
      hipLaunchKernelGGL((attn_paged_combine<E, HD, SG>), dim3((unsigned)(runs() * L.heads_kv)),
                         dim3(NT), 0, s, a, take);
    };
    if (combine_groups(L, room_of(L)) == 8)
      combine(std::integral_constant<int, 8>{});
    else
      combine(std::integral_constant<int, 1>{});
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace neptune
