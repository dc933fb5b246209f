// rope.hip — query/key norm with position rotation, and the paged cache append
// that does both on the way, for gfx950.
//
// Not in the reference. Per head row x of D elements at position p:
//   y = x w / sqrt(mean(x^2) + eps)             where a norm weight w is given
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s) with c, s = cos, sin [p][pair]
// for the R/2 pairs of the first R elements: (i, i + R/2), or (2i, 2i + 1)
// interleaved. All of it in fp32, rounded once at the store; an E4M3 pool takes
// the nearest code of the value's fp32 quotient by its page's scale.
//
// D/8 lanes hold a row, eight elements each. Lane l of the rotated part holds
// both sides of pairs 4l .. 4l+3, so a rotation never leaves the lane: two
// 4-element runs R/2 apart, or eight neighbours interleaved, with one float4 of
// cos and of sin either way. Weights and angles make two factors per element, once
// for a token: z_e = r (y_e P_e + y_partner Q_e), r the row's 1 / rms.
//
// A group of lanes takes HPG heads of one token, all loaded before the first is
// used; position, page, angles and factors are then worked out once for them.
// Neighbouring groups take neighbouring heads of the token, and a work-group's rows
// are all queries, all keys or all values, so bases, strides and weights are
// scalar. HPG 4 where that leaves work-groups for every CU, else 1.
//
// Bound: HBM for prompts, the chain of dependent loads (sequence, length, page or
// angles) and the launch below. Measured (us; a copy of as many bytes): 16384
// tokens of 32 + 8 bf16 heads with norms 64-67 (63), 15000 tokens into a token-major
// cache 38-45 (42), 8 x up to 250 into E4M3 pages 8.9 (5.1), 16 tokens 3.2 and 32 tokens
// appended 3.6 (an empty copy 2.0). Factors per element, scalar bases by operand and the
// rows' loads behind the chain's first took 38, 22, 0.1 and 0.2 off the 16-bit ones.
#include <type_traits>

#include "device_common.h"
#include "kernels.h"

namespace neptune {
namespace {

constexpr int NT = 256;

// One 4-element run in storage and in fp32
struct F32Elem {
  typedef f32x4 raw;
  static constexpr int SIZE = 4;
  __device__ static inline f32x4 load(raw r) { return r; }
  __device__ static inline raw store(f32x4 x) { return x; }
  // two neighbouring runs
  __device__ static inline void load8(const char *p, raw &a, raw &b) {
    a = *(const raw *)p;
    b = *(const raw *)(p + 16);
  }
  __device__ static inline void store8(char *p, raw a, raw b) {
    *(raw *)p = a;
    *(raw *)(p + 16) = b;
  }
};
template <class E>
struct Elem16 {
  typedef u32x2 raw;
  static constexpr int SIZE = 2;
  __device__ static inline f32x4 load(raw r) {
    return f32x4{E::to_f32((uint16_t)r[0]), E::to_f32((uint16_t)(r[0] >> 16)),
                 E::to_f32((uint16_t)r[1]), E::to_f32((uint16_t)(r[1] >> 16))};
  }
  __device__ static inline raw store(f32x4 x) {
    return raw{E::pack2(x[0], x[1]), E::pack2(x[2], x[3])};
  }
  __device__ static inline void load8(const char *p, raw &a, raw &b) {
    const u32x4 v = *(const u32x4 *)p;
    a = raw{v[0], v[1]};
    b = raw{v[2], v[3]};
  }
  __device__ static inline void store8(char *p, raw a, raw b) {
    *(u32x4 *)p = u32x4{a[0], a[1], b[0], b[1]};
  }
};

// One operand: rows in, rows out (keys and values of an append: the pool)
struct RopeSide {
  const char *in;
  char *out;
  const float *w, *scales;  // norm weight; scales of an E4M3 pool (nullable)
  int64_t is[3], os[3];     // byte strides (batch, head, token); pool (page, head, place)
  int32_t heads, runs;      // runs: groups of lanes per token
  uint32_t runs_inv;
  uint32_t first;           // the operand's first work-group
};

struct RopeArgs {
  RopeSide side[3];  // queries, keys, values (append)
  const float *cos, *sin;
  const int32_t *pos;              // qk_norm_rope: position of each token
  const int32_t *cu, *lens, *btab; // append
  int32_t S, tokens;
  uint32_t S_inv;
  int32_t half, P, interleaved;    // pairs rotated, table rows
  int32_t B, ps, maxp, npages;
  float eps, inv_dim;
};

// floor(x / d), inv = floor((2^32 - 1) / d): the estimate is that or one less
__device__ inline uint32_t divide(uint32_t x, uint32_t d, uint32_t inv) {
  const uint32_t q = __umulhi(x, inv);
  return x - q * d >= d ? q + 1 : q;
}

// sum over aligned groups of N (4, 8 or 16) lanes, in every lane: DPP moves
template <int N>
__device__ inline float group_sum(float x) {
  auto add = [&](auto ctrl) {
    x += __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                           0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xb1>{});                       // quad_perm [1,0,3,2]
  add(std::integral_constant<int, 0x4e>{});                       // quad_perm [2,3,0,1]
  if constexpr (N >= 8) add(std::integral_constant<int, 0x141>{});   // row_half_mirror
  if constexpr (N >= 16) add(std::integral_constant<int, 0x140>{});  // row_mirror
  return x;
}

// 1 / sqrt(x) by v_rsq_f32 (1 ulp), which reads subnormal numbers as 0: those, the mean
// squares of rows near 2^-64 with an eps as small, are scaled up first
__device__ inline float inverse_root(float x) {
  const bool small = x < 0x1p-100f;
  return __builtin_amdgcn_rsqf(small ? x * 0x1p100f : x) * (small ? 0x1p50f : 1.0f);
}

// Eight E4M3 codes of the fp32 quotients x / scale: nearest even, saturated (the
// instruction turns what passes 448 into NaN, so it is cut off first). The product
// with 1 / scale is off by up to 1.5 steps of fp32, which moves quotients from the
// middle between two codes (25 = 1.3671875 / 0.0546875 came out as 26, not 24; of bf16
// values under scales k / 128, 0.04%). One residual step brings it within a step, and
// a second one makes it the rounded quotient (Markstein: the reciprocal is correctly
// rounded, the residual of such a quotient exact) where nothing leaves the range of
// ordinary floats. Where it may, in a page's scale or a quotient, the wave divides; a
// page of scale 0 holds zeros, NaN stays NaN (the minimum of the other path would
// swallow it). Measured (us, the product alone / this): 8 x up to 250 tokens 8.4 / 8.8,
// 16000 tokens of 32 heads 122 / 126; division throughout takes 1.13 and 1.10 times the
// product's time.
__device__ inline u32x2 codes8(f32x4 a, f32x4 b, float scale) {
  const float inv = 1.0f / scale;
  float x[8], y[8], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = i < 4 ? a[i & 3] : b[i & 3];
    y[i] = x[i] * inv;
    sum += fabsf(y[i]);
  }
  if (__any(!(sum <= 1e38f && fabsf(scale) >= 0x1p-64f && fabsf(scale) <= 0x1p64f))) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = scale == 0.0f ? 0.0f : x[i] / scale;
      y[i] = y[i] > 448.0f ? 448.0f : y[i];
      y[i] = y[i] < -448.0f ? -448.0f : y[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = fmaf(fmaf(-y[i], scale, x[i]), inv, y[i]);
      y[i] = fmaf(fmaf(-y[i], scale, x[i]), inv, y[i]);
      y[i] = __builtin_amdgcn_fmed3f(y[i], -448.0f, 448.0f);
    }
  }
  u32x2 c;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], lo, true);
  }
  return c;
}

// KIND: 0 queries, 1 keys, 2 values
template <class E, int D, bool APPEND, bool FP8, int HPG, int KIND>
__device__ inline void rows(const RopeArgs &a) {
  typedef typename E::raw raw;
  constexpr int LPR = D / 8;
  constexpr bool TO_POOL = APPEND && KIND > 0;
  const int lane = threadIdx.x & 63, l = threadIdx.x % LPR;
  const RopeSide &x = a.side[KIND];
  const uint32_t gid = (blockIdx.x - x.first) * (NT / LPR) + threadIdx.x / LPR;
  const int at = (int)divide(gid, x.runs, x.runs_inv), run = (int)gid - at * x.runs;
  const int tok = min(at, a.tokens - 1);
  bool live = at < a.tokens;

  // An append's chain to the token's place and slot begins here; the rows are
  // loaded behind its first link, so that they arrive while it is followed. (The
  // one link of a plain rotation does better behind the rows: 76 / 82 us, 16384
  // tokens, one head a group.)
  const int t0 = APPEND ? 0 : (int)divide(tok, a.S, a.S_inv), t1 = APPEND ? tok : tok - t0 * a.S;
  int t, page = -1, place = 0, end = 0x7fffffff;
  const int chunk = (a.B + 63) >> 6;  // sequences a lane stands for in the search
  if constexpr (APPEND)
    if (a.cu && lane * chunk < a.B) end = a.cu[min((lane + 1) * chunk, a.B)];

  // this lane's two runs of four elements, the rotated ones' pairs 4l ..; flat: all
  // lanes' runs are neighbours
  const bool flat = KIND == 2 || a.interleaved || a.half == 0;
  const bool turns = KIND < 2 && 4 * l < a.half;
  const int offa = turns && !flat ? 4 * l : 8 * l;
  const int offb = turns && !flat ? 4 * l + a.half : 8 * l + 4;
  const char *src = x.in + (APPEND ? 0 : t0 * x.is[0]) + t1 * x.is[2];
  raw xa[HPG], xb[HPG];
  auto row_in = [&](int i) { return src + min(run + i * x.runs, x.heads - 1) * x.is[1]; };
  if (flat) {
#pragma unroll
    for (int i = 0; i < HPG; ++i) E::load8(row_in(i) + 8 * E::SIZE * l, xa[i], xb[i]);
  } else {
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      xa[i] = *(const raw *)(row_in(i) + offa * E::SIZE);
      xb[i] = *(const raw *)(row_in(i) + offb * E::SIZE);
    }
  }

  float scale[HPG];
  if constexpr (!APPEND) t = a.pos[tok];
  if constexpr (APPEND) {
    int b = tok, left = 1;
    if (a.cu) {
      // the sequence: as many ends lie at or before the row. Among 64 ends of whole
      // chunks, then among those of the chunk that the row is in (1024
      // single tokens 6.9 us, 2048 10.6; with a step per 64 sequences 9.7 and 19.3)
      constexpr int GROUPS = 64 / LPR;
      int row[GROUPS], at[GROUPS];
      b = 0;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        row[g] = __builtin_amdgcn_readlane(tok, g * LPR);
        at[g] = chunk * __builtin_popcountll(__ballot(end <= row[g]));
        if (lane / LPR == g) b = at[g];
      }
      if (chunk > 1)
        for (int j = lane; j - lane < chunk; j += 64) {
          int ends[GROUPS];
#pragma unroll
          for (int g = 0; g < GROUPS; ++g)
            ends[g] = j < chunk && at[g] + j < a.B ? a.cu[at[g] + j + 1] : 0x7fffffff;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const int n = __builtin_popcountll(__ballot(ends[g] <= row[g]));
            if (lane / LPR == g) b += n;
          }
        }
      live = live && b < a.B && a.cu[0] <= tok;  // rows behind the last sequence stay as they were
      b = min(b, a.B - 1);
      left = a.cu[b + 1] - tok;
    }
    t = a.lens[b] - left;
    if constexpr (KIND > 0) {
      const int index = (int)((uint32_t)max(t, 0) / (uint32_t)a.ps);
      place = max(t, 0) - index * a.ps;
      if (t >= 0 && index < a.maxp) page = a.btab[(int64_t)b * a.maxp + index];
      // a key or value without a slot is not stored
      live = live && page >= 0 && page < a.npages;
      if constexpr (FP8)
#pragma unroll
        for (int i = 0; i < HPG; ++i)
          scale[i] = live ? x.scales[(int64_t)page * x.heads + min(run + i * x.runs, x.heads - 1)]
                          : 1.0f;
    }
  }

  // the factors of the lane's elements, and of their partners: the other run's
  // element, or (interleaved) the neighbour
  f32x4 pa = {1, 1, 1, 1}, pb = {1, 1, 1, 1}, qa = {0, 0, 0, 0}, qb = {0, 0, 0, 0};
  if constexpr (KIND < 2) {
    // all four loads are in flight before the first is waited for
    f32x4 c = pa, s = qa;
    if (a.half) {
      const int64_t row = (int64_t)min(max(t, 0), a.P - 1) * a.half + min(4 * l, a.half - 4);
      c = *(const f32x4 *)(a.cos + row);
      s = *(const f32x4 *)(a.sin + row);
    }
    if (x.w) {
      pa = *(const f32x4 *)(x.w + offa);
      pb = *(const f32x4 *)(x.w + offb);
    }
    asm volatile("" : "+v"(c), "+v"(s), "+v"(pa), "+v"(pb));
    if (turns) {
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qa[2 * j] = -pa[2 * j + 1] * s[j];
          qa[2 * j + 1] = pa[2 * j] * s[j];
          qb[2 * j] = -pb[2 * j + 1] * s[2 + j];
          qb[2 * j + 1] = pb[2 * j] * s[2 + j];
          pa[2 * j] *= c[j];
          pa[2 * j + 1] *= c[j];
          pb[2 * j] *= c[2 + j];
          pb[2 * j + 1] *= c[2 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qa[j] = -pb[j] * s[j];
          qb[j] = pa[j] * s[j];
          pa[j] *= c[j];
          pb[j] *= c[j];
        }
      }
    }
  }

  char *dst = TO_POOL ? x.out + page * x.os[0] + place * x.os[2]
                                 : x.out + (APPEND ? 0 : t0 * x.os[0]) + t1 * x.os[2];
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int h = run + i * x.runs;
    f32x4 ya = E::load(xa[i]), yb = E::load(xb[i]);
    if constexpr (KIND < 2) {  // values pass as they are
      float r = 1.0f;
      if (x.w) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(ya[j], ya[j], fmaf(yb[j], yb[j], ss));
        r = inverse_root(fmaf(group_sum<LPR>(ss), a.inv_dim, a.eps));
      }
      f32x4 za, zb;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (a selection, not a branch: elements behind rot_dim have no partner)
        const float oa = a.interleaved ? ya[j ^ 1] : yb[j], ob = a.interleaved ? yb[j ^ 1] : ya[j];
        za[j] = ya[j] * pa[j];
        zb[j] = yb[j] * pb[j];
        if (turns) {
          za[j] = fmaf(oa, qa[j], za[j]);
          zb[j] = fmaf(ob, qb[j], zb[j]);
        }
      }
      ya = za * r;
      yb = zb * r;
    }
    if (!live || h >= x.heads) continue;
    char *p = dst + h * x.os[1];
    if constexpr (FP8 && TO_POOL) {
      const u32x2 c = codes8(ya, yb, scale[i]);
      if (flat) {
        *(u32x2 *)(p + 8 * l) = c;
      } else {
        *(uint32_t *)(p + offa) = c[0];
        *(uint32_t *)(p + offb) = c[1];
      }
    } else {
      if (flat) {
        E::store8(p + 8 * E::SIZE * l, E::store(ya), E::store(yb));
      } else {
        *(raw *)(p + offa * E::SIZE) = E::store(ya);
        *(raw *)(p + offb * E::SIZE) = E::store(yb);
      }
    }
  }
}

template <class E, int D, bool APPEND, bool FP8, int HPG>
__global__ __launch_bounds__(NT) void norm_rope(RopeArgs a) {
  if (blockIdx.x < a.side[1].first)
    rows<E, D, APPEND, FP8, HPG, 0>(a);
  else if (!APPEND || blockIdx.x < a.side[2].first)
    rows<E, D, APPEND, FP8, HPG, 1>(a);
  else if constexpr (APPEND)
    rows<E, D, APPEND, FP8, HPG, 2>(a);
}

template <class E, int D, bool APPEND, bool FP8>
hipError_t launch_hpg(RopeArgs a, hipStream_t s) {
  constexpr int GPB = NT / (D / 8);  // groups of lanes per work-group
  auto go = [&](auto H) {
    constexpr int HPG = decltype(H)::value;
    uint32_t blocks = 0;
    for (int i = 0; i < (APPEND ? 3 : 2); ++i) {
      RopeSide &x = a.side[i];
      x.first = blocks;
      if (!x.heads) continue;
      x.runs = (x.heads + HPG - 1) / HPG;
      x.runs_inv = 0xffffffffu / (uint32_t)x.runs;
      blocks += (uint32_t)(((int64_t)a.tokens * x.runs + GPB - 1) / GPB);
    }
    hipLaunchKernelGGL((norm_rope<E, D, APPEND, FP8, HPG>), dim3(blocks), dim3(NT), 0, s, a);
  };
  // Several heads a group spare it most of its instructions, but leave fewer
  // work-groups: from 8 for every CU on. Measured (us, 1 / 2 / 4 / 8 heads): 16384
  // tokens of 32 + 8 heads 75 / 70 / 66 / 64; of 16 + 4 head_dim-64 heads 18.7 /
  // 16.1 / 15.0 / 14.2; 2000 tokens of 32 + 8 11.1 / 10.4 / 9.8 / 10.9; 1300 into
  // E4M3 pages 10.6 / 9.3 / 9.4 / 10.4; below, 500 tokens 4.3 / 4.2 / 4.9 / 5.5; 16
  // 2.75 / 2.9 / 3.4 / 4.4.
  const int64_t heads = a.side[0].heads + (APPEND ? 2 : 1) * (int64_t)a.side[1].heads;
  if (a.tokens * heads >= 2048 * GPB)
    go(std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 1>{});
  return hipGetLastError();
}

template <class E, int D>
hipError_t launch_d(const RopeArgs &a, bool append, bool fp8, hipStream_t s) {
  if constexpr (E::SIZE == 2 && D >= 64) {
    if (append) return fp8 ? launch_hpg<E, D, true, true>(a, s) : launch_hpg<E, D, true, false>(a, s);
  }
  return launch_hpg<E, D, false, false>(a, s);
}

template <class E>
hipError_t launch_e(const RopeArgs &a, int64_t head_dim, bool append, bool fp8, hipStream_t s) {
  switch (head_dim) {
    case 32: return launch_d<E, 32>(a, append, fp8, s);
    case 64: return launch_d<E, 64>(a, append, fp8, s);
    default: return launch_d<E, 128>(a, append, fp8, s);
  }
}

}  // namespace

bool rope_supported(const RopeLaunch &L, const char **why) {
  if (L.head_dim != 32 && L.head_dim != 64 && L.head_dim != 128) {
    *why = "head_dim must be 32, 64 or 128";
    return false;
  }
  if (L.append && L.head_dim == 32) {
    *why = "the paged cache holds head_dim 64 or 128";
    return false;
  }
  if (L.rot_dim % 8) {
    *why = "rot_dim must be a multiple of 8";
    return false;
  }
  // a group of lanes per (token, head) at most, counted in 32 bits; a dispatch
  // covers at most 2^32 - 1 work-items
  const int64_t heads = L.heads_q + (L.append ? 2 : 1) * L.heads_kv;
  const int64_t tokens = L.batch * L.seq;
  if (L.batch > INT32_MAX || L.seq > INT32_MAX || heads > 1 << 20 || tokens > INT32_MAX ||
      tokens * heads > ((int64_t)1 << 31) / (L.head_dim / 8)) {
    *why = "tokens * heads too large for one launch";
    return false;
  }
  if (L.table_len > INT32_MAX || L.num_pages > INT32_MAX || L.max_pages > INT32_MAX ||
      L.page_size > INT32_MAX || L.sequences > INT32_MAX - 64) {
    *why = "tables of 2^31 rows or pages and more";
    return false;
  }
  if (L.cu_seqlens && L.sequences > 1 << 16) {  // every group of lanes looks through them
    *why = "cu_seqlens of more than 65536 sequences";
    return false;
  }
  return true;
}

hipError_t launch_rope(const RopeLaunch &L, hipStream_t s) {
  RopeArgs a = {};
  const int64_t size = L.dtype == 0 ? 4 : 2, kv = L.fp8 ? 1 : size;
  a.side[0] = {(const char *)L.q, (char *)L.qo, L.q_weight, nullptr};
  a.side[1] = {(const char *)L.k, (char *)L.ko, L.k_weight, L.k_scales};
  a.side[2] = {(const char *)L.v, (char *)L.vo, nullptr, L.v_scales};
  const int64_t *const in[3] = {L.qs, L.ks, L.vs}, *const out[3] = {L.qos, L.kos, L.vos};
  for (int i = 0; i < 3; ++i) {
    a.side[i].heads = (int32_t)(i ? L.heads_kv : L.heads_q);
    for (int j = 0; j < 3; ++j) {
      a.side[i].is[j] = in[i][j] * size;
      a.side[i].os[j] = out[i][j] * (L.append && i ? kv : size);
    }
  }
  a.cos = L.cos; a.sin = L.sin;
  a.pos = L.positions; a.cu = L.cu_seqlens; a.lens = L.seq_lens; a.btab = L.block_table;
  a.S = (int32_t)L.seq;
  a.tokens = (int32_t)(L.batch * L.seq);
  a.S_inv = 0xffffffffu / (uint32_t)a.S;
  a.half = (int32_t)(L.rot_dim / 2);
  a.P = (int32_t)L.table_len;
  a.interleaved = L.interleaved;
  a.B = (int32_t)L.sequences;
  a.ps = (int32_t)L.page_size;
  a.maxp = (int32_t)L.max_pages;
  a.npages = (int32_t)L.num_pages;
  a.eps = L.eps;
  a.inv_dim = 1.0f / (float)L.head_dim;
  if (L.dtype == 0) return launch_e<F32Elem>(a, L.head_dim, false, false, s);
  if (L.dtype == 1) return launch_e<Elem16<F16Tag>>(a, L.head_dim, L.append, L.fp8, s);
  return launch_e<Elem16<Bf16Tag>>(a, L.head_dim, L.append, L.fp8, s);
}

}  // namespace neptune
