// rope.hip — query/key norm with position rotation, and the paged cache append
// that does both on the way, for gfx950.
//
// Not in the reference. Per head row x of D elements at position p:
//   y = x w / sqrt(mean(x^2) + eps)             where a norm weight w is given
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s) with c, s = cos, sin [p][pair]
// for the R/2 pairs of the first R elements: (i, i + R/2), or (2i, 2i + 1)
// interleaved. All of it in fp32, rounded once at the store; an E4M3 pool takes
// the nearest code of the fp32 value over its page's scale.
//
// D/8 lanes hold a row, eight elements each. Lane l of the rotated part holds
// both sides of pairs 4l .. 4l+3, so a rotation never leaves the lane: two
// 4-element runs R/2 apart, or eight neighbours interleaved, with one float4 of
// cos and of sin either way. Consecutive groups of lanes take consecutive heads
// of a token, so a wave reads whole heads side by side. A group takes HPG heads
// of its token, all loaded before the first is used: the token's table row,
// position and page are then looked up once for them.
//
// Bound: HBM for prompts, the chain of dependent loads (sequence, length, table
// row) and the launch for single tokens.
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
};

struct RopeArgs {
  const char *q, *k, *v;
  char *qo, *ko, *vo;  // append: ko and vo are the pools
  const float *qw, *kw, *cos, *sin;
  const int32_t *pos;                       // qk_norm_rope: position of each token
  const int32_t *cu, *lens, *btab;          // append
  const float *ksc, *vsc;                   // E4M3 pools
  // byte strides (batch, head, token); of a pool (page, head, place)
  int64_t qs[3], ks[3], vs[3], qos[3], kos[3], vos[3];
  int32_t Hq, Hk, heads;                    // heads: all rows of a token
  int32_t S, tokens, runs;                  // runs: groups of lanes per token
  int32_t half, P, interleaved;             // pairs rotated, table rows
  int32_t B, ps, maxp, npages;
  float eps, inv_dim;
};

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

// four E4M3 codes of x / scale: nearest even, saturated (a NaN keeps its code;
// the instruction turns what passes 448 into NaN, so it is cut off first). A
// page of scale 0 holds zeros.
__device__ inline uint32_t codes4(f32x4 x, float scale) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = scale == 0.0f ? 0.0f : x[i] / scale;
    y[i] = y[i] > 448.0f ? 448.0f : y[i];
    y[i] = y[i] < -448.0f ? -448.0f : y[i];
  }
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}

template <class E, int D, bool APPEND, bool FP8, int HPG>
__global__ __launch_bounds__(NT) void norm_rope(RopeArgs a) {
  typedef typename E::raw raw;
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x & 63, l = threadIdx.x % LPR;
  const uint32_t gid = blockIdx.x * (NT / LPR) + threadIdx.x / LPR;
  const int at = (int)(gid / (uint32_t)a.runs), run = (int)(gid - (uint32_t)at * a.runs);
  const int tok = min(at, a.tokens - 1);
  bool live = at < a.tokens;

  // this lane's two runs of four elements, the rotated ones' pairs 4l ..
  const bool turns = 4 * l < a.half;
  const int offa = turns && !a.interleaved ? 4 * l : 8 * l;
  const int offb = turns && !a.interleaved ? 4 * l + a.half : 8 * l + 4;
  const int64_t t0 = APPEND ? 0 : tok / a.S, t1 = APPEND ? tok : tok - (int)t0 * a.S;
  auto source = [&](int h) {
    const char *base = h < a.Hq ? a.q : h < a.Hq + a.Hk ? a.k : a.v;
    const int64_t *st = h < a.Hq ? a.qs : h < a.Hq + a.Hk ? a.ks : a.vs;
    const int hh = h < a.Hq ? h : h < a.Hq + a.Hk ? h - a.Hq : h - a.Hq - a.Hk;
    return base + t0 * st[0] + hh * st[1] + t1 * st[2];
  };
  raw xa[HPG], xb[HPG];
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const char *p = source(min(run + i * a.runs, a.heads - 1));
    xa[i] = *(const raw *)(p + offa * E::SIZE);
    xb[i] = *(const raw *)(p + offb * E::SIZE);
  }

  // the token's position, and its slot in the cache
  int t, page = -1, place = 0;
  if constexpr (APPEND) {
    int b = tok, left = 1;
    if (a.cu) {
      // the sequence: as many ends lie at or before the row
      b = 0;
      for (int j = 0; j < a.B; j += 64) {
        const int end = j + lane < a.B ? a.cu[j + lane + 1] : 0x7fffffff;
#pragma unroll
        for (int g = 0; g < 64 / LPR; ++g) {
          const int other = __builtin_amdgcn_readlane(tok, g * LPR);
          const int n = __builtin_popcountll(__ballot(end <= other));
          if (lane / LPR == g) b += n;
        }
      }
      live = live && b < a.B && a.cu[0] <= tok;  // rows behind the last sequence stay as they were
      b = min(b, a.B - 1);
      left = a.cu[b + 1] - tok;
    }
    t = a.lens[b] - left;
    const int index = (int)((uint32_t)max(t, 0) / (uint32_t)a.ps);
    place = max(t, 0) - index * a.ps;
    if (t >= 0 && index < a.maxp) page = a.btab[(int64_t)b * a.maxp + index];
  } else {
    t = a.pos[tok];
  }
  f32x4 c = {1, 1, 1, 1}, s = {0, 0, 0, 0};
  if (turns) {
    const int64_t row = (int64_t)min(max(t, 0), a.P - 1) * a.half + 4 * l;
    c = *(const f32x4 *)(a.cos + row);
    s = *(const f32x4 *)(a.sin + row);
  }
  const bool stored = APPEND && page >= 0 && page < a.npages;

#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    const int h = run + i * a.runs;
    const bool is_q = h < a.Hq, is_v = APPEND && h >= a.Hq + a.Hk;
    f32x4 ya = E::load(xa[i]), yb = E::load(xb[i]);
    if (!is_v) {
      const float *w = is_q ? a.qw : a.kw;
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(ya[j], ya[j], fmaf(yb[j], yb[j], ss));
        const float r = 1.0f / sqrtf(fmaf(group_sum<LPR>(ss), a.inv_dim, a.eps));
        const f32x4 wa = *(const f32x4 *)(w + offa), wb = *(const f32x4 *)(w + offb);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ya[j] = ya[j] * r * wa[j];
          yb[j] = yb[j] * r * wb[j];
        }
      }
      if (turns) {
        f32x4 za, zb;
        if (a.interleaved) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            za[2 * j] = ya[2 * j] * c[j] - ya[2 * j + 1] * s[j];
            za[2 * j + 1] = ya[2 * j + 1] * c[j] + ya[2 * j] * s[j];
            zb[2 * j] = yb[2 * j] * c[2 + j] - yb[2 * j + 1] * s[2 + j];
            zb[2 * j + 1] = yb[2 * j + 1] * c[2 + j] + yb[2 * j] * s[2 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            za[j] = ya[j] * c[j] - yb[j] * s[j];
            zb[j] = yb[j] * c[j] + ya[j] * s[j];
          }
        }
        ya = za;
        yb = zb;
      }
    }
    if (!live || h >= a.heads) continue;
    if (APPEND && !is_q) {
      if (!stored) continue;
      const int hh = is_v ? h - a.Hq - a.Hk : h - a.Hq;
      const int64_t *st = is_v ? a.vos : a.kos;
      char *p = (is_v ? a.vo : a.ko) + page * st[0] + hh * st[1] + place * st[2];
      if constexpr (FP8) {
        const float scale = (is_v ? a.vsc : a.ksc)[(int64_t)page * a.Hk + hh];
        *(uint32_t *)(p + offa) = codes4(ya, scale);
        *(uint32_t *)(p + offb) = codes4(yb, scale);
      } else {
        *(raw *)(p + offa * E::SIZE) = E::store(ya);
        *(raw *)(p + offb * E::SIZE) = E::store(yb);
      }
    } else {
      const int hh = is_q ? h : h - a.Hq;
      const int64_t *st = is_q ? a.qos : a.kos;
      char *p = (is_q ? a.qo : a.ko) + t0 * st[0] + hh * st[1] + t1 * st[2];
      *(raw *)(p + offa * E::SIZE) = E::store(ya);
      *(raw *)(p + offb * E::SIZE) = E::store(yb);
    }
  }
}

template <class E, int D, bool APPEND, bool FP8>
hipError_t launch_hpg(RopeArgs a, hipStream_t s) {
  constexpr int GPB = NT / (D / 8);  // groups of lanes per work-group
  auto go = [&](auto H) {
    constexpr int HPG = decltype(H)::value;
    a.runs = (a.heads + HPG - 1) / HPG;
    const int64_t groups = (int64_t)a.tokens * a.runs;
    hipLaunchKernelGGL((norm_rope<E, D, APPEND, FP8, HPG>), dim3((unsigned)((groups + GPB - 1) / GPB)),
                       dim3(NT), 0, s, a);
  };
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
  return true;
}

hipError_t launch_rope(const RopeLaunch &L, hipStream_t s) {
  RopeArgs a;
  const int64_t size = L.dtype == 0 ? 4 : 2, kv = L.fp8 ? 1 : size;
  a.q = (const char *)L.q; a.k = (const char *)L.k; a.v = (const char *)L.v;
  a.qo = (char *)L.qo; a.ko = (char *)L.ko; a.vo = (char *)L.vo;
  a.qw = L.q_weight; a.kw = L.k_weight; a.cos = L.cos; a.sin = L.sin;
  a.pos = L.positions; a.cu = L.cu_seqlens; a.lens = L.seq_lens; a.btab = L.block_table;
  a.ksc = L.k_scales; a.vsc = L.v_scales;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = L.qs[i] * size; a.ks[i] = L.ks[i] * size; a.vs[i] = L.vs[i] * size;
    a.qos[i] = L.qos[i] * size;
    a.kos[i] = L.kos[i] * (L.append ? kv : size);
    a.vos[i] = L.vos[i] * kv;
  }
  a.Hq = (int32_t)L.heads_q;
  a.Hk = (int32_t)L.heads_kv;
  a.heads = a.Hq + (L.append ? 2 : 1) * a.Hk;
  a.S = (int32_t)L.seq;
  a.tokens = (int32_t)(L.batch * L.seq);
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
