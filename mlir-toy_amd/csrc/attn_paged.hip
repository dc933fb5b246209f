// attn_paged.hip — attention of a ragged batch of new tokens over a paged KV
// cache, for gfx950.
//
// Not in the reference; the recurrence is the HTile one
// (tests/data/flash_attention_htile.mlir:40-143) per query row:
//   O_r = sum_{j <= t} 2^(s_rj - m) v_j / l,   s_rj = q_r . k_j scale log2(e),
//   l = sum_j 2^(s_rj - m),   lse_r = (m + log2 l) ln 2,
// with t the row's place in its sequence. 16-bit pools, or E4M3 codes with a
// scale per page and KV head.
//
// Tiles and items. The rows of a KV head's whole group, token by token, form a
// sequence's run of rows (row r: token r / group, head r % group), cut into tiles
// of 128: K and V are then read once for the group, and the causal edge of a tile
// spans 128 / group tokens only. The lengths are on the device, so the launch
// has an upper bound of work-groups and each finds its item (sequence, tile,
// split of the keys) itself from cu_seqlens and seq_lens (Schedule).
//
// A work-group is that of attn_fwd_tile.hip: 4 waves of 32 rows, 64-key blocks,
// S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_32x32x16, two LDS slots per
// operand, block j+1's QK^T in the MFMA stream of block j's P.V. A block's 64
// keys are four runs of 16, one per wave, each within a page (the page size is a
// multiple of 16): the run's page comes by v_readlane from a window of 64
// block-table entries, so no load waits on a load. E4M3 codes pass through
// registers and are widened to bf16 (exact) on their way to LDS, once for the
// work-group's four waves; the K scale meets the scores, the V scale P before
// its rounding.
#include <algorithm>

#include "attn_tile.h"
#include "kernels.h"

namespace neptune {
namespace {

constexpr int64_t kSlots = 512;   // two work-groups on each of 256 CUs
constexpr int64_t kParts = 2 * kSlots;  // split items a launch makes at most (Schedule)

struct PagedArgs {
  const uint16_t *q;
  const char *k, *v;
  const float *ksc, *vsc;
  const int32_t *btab, *cu, *lens;
  uint16_t *o;
  float *lse, *po, *pml;
  int64_t qs0, qs1, os0, os1;     // (token, head), elements
  int64_t kps0, kps1, vps0, vps1; // (page, head), bytes
  int64_t ktok, vtok;             // place, bytes
  int32_t T, B, Hq, Hk, group, Lmax, maxp, npages;
  int32_t ps16;                   // page size in runs of 16 tokens
  uint32_t ps16_inv;              // floor((2^32 - 1) / ps16)
  int32_t parts;                  // 0: keys are never split
  int32_t prows;                  // rows of a split item's states
  float scale2;
};

// run / ps16 and the rest, exactly: the estimate is the quotient or one less
__device__ inline void page_of(const PagedArgs &a, int run, int *index, int *rest) {
  int q = (int)__umulhi((uint32_t)run, a.ps16_inv);
  int r = run - q * a.ps16;
  if (r >= a.ps16) {
    ++q;
    r -= a.ps16;
  }
  *index = q;
  *rest = r;
}

struct Item {
  int b, n, row0;   // sequence, its new tokens, its first row of q
  int len;          // tokens in its cache
  int tile, tiles;  // 128-row tile
  int split, splits;
  int part;         // first part of the tile (splits > 1)
};

// Sequence b's share of the launch. cu, lens and the table are the caller's
// device data: whatever they hold, rows stay within q and lengths within
// the table.
struct Seq {
  int n, row0, len, tiles, blocks;
};
__device__ inline Seq sequence(const PagedArgs &a, int b) {
  Seq s = {0, 0, 0, 0, 0};
  if (b < a.B) {
    const int lo = a.cu ? min(max(a.cu[b], 0), a.T) : b;
    const int hi = a.cu ? min(max(a.cu[b + 1], lo), a.T) : b + 1;
    s.n = hi - lo;
    s.row0 = lo;
    s.len = min(max(a.lens[b], 0), a.Lmax);
    s.tiles = (s.n * a.group + BM - 1) / BM;
    s.blocks = (s.len + BN - 1) / BN;
  }
  return s;
}

// Splits of a sequence's tiles. A work-group's time is its chain of key blocks,
// so chains longer than the launch's work over kSlots work-groups (work: tile
// blocks, a tile's taken as the mean of its sequence's first and last tile's)
// are cut into that many or longer. A split costs its states, written and read:
// worth at least 4 blocks, 12 for a full tile.
__device__ inline int splits_of(const Seq &s, int group, int chain) {
  const int least = 4 + min(s.n * group, BM) / 16;
  return max(s.blocks / max(chain, least), 1);
}

// Item idx of the launch (per_tile: tile idx) of one KV head, false if there is
// none. Sequences in order, a sequence's tiles from the last (under the causal
// mask the longest), a tile's splits together. Every wave works it out by
// itself, one sequence per lane.
__device__ inline bool find_item(const PagedArgs &a, int lane, int idx, bool per_tile, Item *it) {
  int chain = 0x7fffffff;
  if (a.parts) {
    uint64_t work = 0;  // in half blocks
    for (int b = lane; b < a.B; b += 64) {
      const Seq s = sequence(a, b);
      const int first = max(s.len - s.n + 1 + BN - 1, 0) / BN;
      work += (uint64_t)s.tiles * (uint32_t)(s.blocks + min(first, s.blocks));
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const uint32_t lo = __shfl_xor((int)(uint32_t)work, off, 64);
      const uint32_t hi = __shfl_xor((int)(uint32_t)(work >> 32), off, 64);
      work += ((uint64_t)hi << 32) | lo;
    }
    work = (work * (uint32_t)a.Hk + 2 * kSlots - 1) / (2 * kSlots);
    chain = work > 0x7fffffff ? 0x7fffffff : (int)work;
  }
  int base = 0, parts = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = sequence(a, b0 + lane);
    const int sp = a.parts ? splits_of(s, a.group, chain) : 1;
    const int mine = per_tile ? s.tiles : s.tiles * sp;
    const int mparts = sp > 1 ? s.tiles * sp : 0;
    int sum = mine, psum = mparts;  // inclusive sums over the lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int u = __shfl_up(sum, off, 64), v = __shfl_up(psum, off, 64);
      if (lane >= off) {
        sum += u;
        psum += v;
      }
    }
    const uint64_t past = __ballot(base + sum > idx);
    if (past) {
      const int at = __builtin_ctzll(past);
      auto take = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      it->b = b0 + at;
      it->n = take(s.n);
      it->row0 = take(s.row0);
      it->len = take(s.len);
      it->tiles = take(s.tiles);
      it->splits = take(sp);
      const int rest = idx - (base + take(sum) - take(mine));
      const int down = per_tile ? rest : rest / it->splits;
      it->tile = it->tiles - 1 - down;
      it->split = per_tile ? 0 : rest - down * it->splits;
      it->part = parts + take(psum) - take(mparts) + down * it->splits;
      return true;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
    parts += __builtin_amdgcn_readlane(psum, 63);
  }
  return false;
}

// bf16 bits of 4 E4M3 codes (exact)
__device__ inline u32x2 widen4(uint32_t c) {
  const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, false);
  const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.0f, true);
  return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

template <class E, int HD, bool FP8>
__global__ __launch_bounds__(NT, 2) void attn_paged(PagedArgs a) {
  typedef typename E::vec8 V8;
  typedef TileLoader<HD> TL;
  constexpr int TILE = TL::TILE_BYTES;
  constexpr int ROWB = HD * 2;   // bytes per LDS row
  constexpr int NST = HD / 16;   // QK^T k-steps
  constexpr int NB = HD / 32;    // 32-wide head_dim blocks of O^T
  constexpr int NQK = 2 * NST, NPV = 4 * NB;  // MFMAs per key block
  constexpr int CHUNKS = TL::CHUNKS, RPC = TL::RPC;
  // K slots 0 and 1, then V slots 0 and 1; block t uses slot t & 1
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * TILE];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 31, g = lane >> 5;
  auto kslot = [&](int t) { return smem + (t & 1) * TILE; };
  auto vslot = [&](int t) { return smem + (2 + (t & 1)) * TILE; };

  // kv heads fastest: with a multiple of 8 of them, id % 8 (the XCD) fixes the
  // head modulo 8 and the tiles of a head share an L2
  const int hk = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % (uint32_t)a.Hk));
  const int idx = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / (uint32_t)a.Hk));
  Item it;
  if (!find_item(a, lane, idx, false, &it)) return;
  const int rows = it.n * a.group;
  const int off = it.len - it.n;  // place of the sequence's first new token
  const int r0 = it.tile * BM + w * 32;

  // this lane's row: query head hk * group + hr of token tok, at place pos
  const int row = r0 + lq;
  const int tok = min(row, rows - 1) / a.group, hr = min(row, rows - 1) - tok * a.group;
  const int pos = off + tok;
  // blocks seen by rows up to r: through the place of its token
  auto blocks_to = [&](int r) {
    const int last = off + min(r, rows - 1) / a.group;
    return last < 0 ? 0 : last / BN + 1;
  };
  const int all = blocks_to(it.tile * BM + BM - 1);
  const int per = (all + it.splits - 1) / it.splits;
  const int kb0 = __builtin_amdgcn_readfirstlane(it.split * per);
  const int nv = __builtin_amdgcn_readfirstlane(min(max(all - kb0, 0), per));
  const int nkw = __builtin_amdgcn_readfirstlane(
      r0 < rows ? min(max(blocks_to(r0 + 31) - kb0, 0), nv) : 0);
  const int lo_w = __builtin_amdgcn_readfirstlane(off + min(r0, rows - 1) / a.group);

  const char *kp = a.k + hk * a.kps1, *vp = a.v + hk * a.vps1;
  const int32_t *tab = a.btab + (int64_t)it.b * a.maxp;
  const int last_key = it.len - 1;

  // the window of the block table: lane j holds entry tab0 + j. It starts at a
  // page of the block before the one being copied and moves when a copy passes it
  int tab0 = 0, tabv = 0;
  auto load_tab = [&](int first) {
    tab0 = first;
    const int j = first + lane;
    tabv = j < a.maxp ? tab[j] : 0;
    settle(tabv);
  };
  // the wave's run of block t: its page's byte offset in each pool, and the
  // tokens of it that exist less one (a run behind the end takes the last run)
  auto run_at = [&](int t, int64_t *ko, int64_t *vo, int *most) {
    int run = (kb0 + t) * (BN / 16) + w;
    const int key = min(run * 16, last_key & ~15);
    run = key >> 4;
    int index, rest;
    page_of(a, run, &index, &rest);
    if (index - tab0 >= 64) load_tab(max(index - 4, 0));
    int page = __builtin_amdgcn_readlane(tabv, index - tab0);
    page = min(max(page, 0), a.npages - 1);
    *ko = page * a.kps0 + (int64_t)(rest * 16) * a.ktok;
    *vo = page * a.vps0 + (int64_t)(rest * 16) * a.vtok;
    *most = last_key - key;
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
        dma16(base, offs[c], lds_offset(tile + (CHUNKS * w + c) * 1024));
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
  // E4M3 pools: 16 codes per lane and load, two rows' worth of units each
  constexpr int LPR8 = HD / 16, ROWS8 = 64 / LPR8, N8 = 16 / ROWS8;
  u32x4 k8[N8], v8[N8];
  auto load8 = [&](const char *base, int64_t tokb, int most, u32x4 *dst) {
#pragma unroll
    for (int c = 0; c < N8; ++c)
      dst[c] = *(const u32x4 *)(base + min(lane / LPR8 + ROWS8 * c, most) * tokb +
                                (lane % LPR8) * 16);
  };
  auto store8 = [&](const u32x4 *src, const uint8_t *tile, bool is_v) {
#pragma unroll
    for (int c = 0; c < N8; ++c) {
      const int r = 16 * w + lane / LPR8 + ROWS8 * c, u = 2 * (lane % LPR8);
      const int z = is_v ? tile_swizzle<HD, true>(r) : tile_swizzle<HD, false>(r);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x2 lo = widen4(src[c][2 * h]), hi = widen4(src[c][2 * h + 1]);
        *(u32x4 *)(uint8_t *)(tile + r * ROWB + (((u + h) ^ z) << 4)) =
            u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }
  };
  auto load_k = [&](int t) {
    int64_t ko, vo;
    int most;
    run_at(t, &ko, &vo, &most);
    if constexpr (FP8)
      load8(kp + ko, a.ktok, most, k8);
    else
      copy(kp + ko, koff, a.ktok, most, false, kslot(t));
  };
  auto load_v = [&](int t) {
    int64_t ko, vo;
    int most;
    run_at(t, &ko, &vo, &most);
    if constexpr (FP8)
      load8(vp + vo, a.vtok, most, v8);
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
  if (nv > 0) {
    int index, rest;
    page_of(a, kb0 * (BN / 16), &index, &rest);
    load_tab(index);
  }

  // Q^T operand: k-step st covers head_dim 16 st + 8 g .. +7 of the row
  u32x4 qf[NST];
  {
    const uint16_t *qp = a.q + (int64_t)(it.row0 + tok) * a.qs0 +
                         (int64_t)(hk * a.group + hr) * a.qs1 + 8 * g;
#pragma unroll
    for (int st = 0; st < NST; ++st)
      qf[st] = row < rows ? *(const u32x4 *)(qp + 16 * st) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < NST; ++st) settle(qf[st]);
  }
  if (nv > 0) {
    load_k(0);
    put_k(0);
    load_v(0);
    put_v(0);
  }
  if (nv > 1) {
    load_k(1);
    put_k(1);
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
      va[nb] = (4 * g + i) * ROWB + (((4 * nb + 2 * dh) ^ tile_swizzle<HD, true>(i)) << 4) + 8 * q;
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
    int index, rest;
    page_of(a, kb0 * (BN / 16), &index, &rest);
    if (nv > 0) load_scales(index);
  }

  f32x16 o[NB];
  f32x16 s[2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[nb][r] = 0.0f;
  float m = kNegFltMax, lsum = 0.0f;
  const f32x16 zero16 = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

  // The A operand of MFMA i = 2 st + kb of S^T = K.Q^T (32 keys x 16 head_dim)
  auto k_operand = [&](const uint8_t *kt, int i) {
    return *(const u32x4 *)(kt + (i & 1) * 32 * ROWB + ka[i >> 1]);
  };
  // S^T of one key block, its first two A operands already read (k0, k1)
  auto qk_from = [&](const uint8_t *kt, const u32x4 &k0, const u32x4 &k1) {
#pragma unroll
    for (int i = 0; i < NQK; ++i) {
      const u32x4 A = i == 0 ? k0 : i == 1 ? k1 : k_operand(kt, i);
      s[i & 1] = E::mfma32(as_vec8<V8>(A), as_vec8<V8>(qf[i >> 1]), i < 2 ? zero16 : s[i & 1]);
    }
    // the remaining operand reads run two MFMAs ahead
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
#pragma unroll
    for (int i = 0; i < NQK - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
  };
  // The A operand of P.V step st (V^T: head_dim rows 32 nb .., keys 16 c ..)
  auto v_operand = [&](const uint8_t *vt, int st) {
    const int c = st / NB, nb = st % NB;
    const u32x2 a0 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + 16 * c * ROWB + va[nb]));
    const u32x2 a1 = __builtin_bit_cast(u32x2, lds_read_tr16(vt + (16 * c + 8) * ROWB + va[nb]));
    return u32x4{a0[0], a0[1], a1[0], a1[1]};
  };

  wait_vmem();
  __syncthreads();
  if (nkw > 0) qk_from(kslot(0), k_operand(kslot(0), 0), k_operand(kslot(0), 1));
  __syncthreads();  // every wave is done with K slot 0 before it is refilled

  for (int jb = 0; jb < nv; ++jb) {
    // K of block jb + 2 goes to the slot block jb's K has left, V of block
    // jb + 1 to the slot of block jb - 1's V
    if (jb + 1 < nv) load_v(jb + 1);
    if (jb + 2 < nv) load_k(jb + 2);
    if (jb < nkw) {
      // the first two V^T operands of this block's P.V, read before the softmax
      const uint8_t *vt = vslot(jb);
      const u32x4 vp0 = v_operand(vt, 0), vp1 = v_operand(vt, 1);
      const int key0 = (kb0 + jb) * BN;
      float sc = a.scale2;
      float vs[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if constexpr (FP8) {
        // each run's scales: K's meets the scores here (before the mask: a zero
        // scale must not meet -inf), V's meets P
        int index, rest;
        page_of(a, key0 >> 4, &index, &rest);
        if (index + 3 - sc0 >= 64) load_scales(index);
        const int runs = last_key / 16 - (key0 >> 4);  // runs behind the end take the last one's
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float ks = sc * __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, kscv), index - sc0));
          vs[c] = __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vscv), index - sc0));
#pragma unroll
          for (int r = 0; r < 8; ++r) s[c >> 1][8 * (c & 1) + r] *= ks;
          if (c < runs && ++rest == a.ps16) {
            rest = 0;
            ++index;
          }
        }
        sc = 1.0f;
      }
      if (key0 + BN - 1 > lo_w) {
        // element (kb, r) holds key key0 + 4 g + c with c = 32 kb + 8 (r >> 2)
        // + (r & 3): it is masked when c passes the row's own place
        const int lim = pos - key0 - 4 * g;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * kb + 8 * (r >> 2) + (r & 3) > lim) s[kb][r] = -INFINITY;
      }
      // p = 2^(s sc - m) for the block, packed for P.V, and the lane's sum
      float rs;
      u32x4 pf[4];
      auto expo = [&]() {
        const float nm = -m;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int kb = c >> 1, hh = c & 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p0 = fast_exp2(fmaf(s[kb][8 * hh + 2 * i], sc, nm));
            const float p1 = fast_exp2(fmaf(s[kb][8 * hh + 2 * i + 1], sc, nm));
            rs = c + i == 0 ? p0 : rs + p0;
            rs += p1;
            pf[c][i] = FP8 ? E::pack2(p0 * vs[c], p1 * vs[c]) : E::pack2(p0, p1);
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
        }
      };
      if constexpr (HD == 64) {
        raise_max(0.0f);
        expo();
      } else {
        // the block max is only formed when it can matter: past the first block,
        // a lane sum of at most 2^kSlack bounds every p by it, and m keeps
        bool full = jb == 0;
        if (!full) {
          expo();
          full = __any(!(rs <= kSumCap));
        }
        if (full) {
          raise_max(kSlack);
          expo();
        }
      }
      lsum += rs;

      // O^T += V^T P^T, then the next block's S^T, at raised issue priority
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int st = 0; st < NPV; ++st) {
        const u32x4 A = st == 0 ? vp0 : st == 1 ? vp1 : v_operand(vt, st);
        o[st % NB] = E::mfma32(as_vec8<V8>(A), as_vec8<V8>(pf[st / NB]), o[st % NB]);
      }
      // the next block's first two K operands (past the last block they are stale
      // and dropped)
      const u32x4 kn0 = k_operand(kslot(jb + 1), 0), kn1 = k_operand(kslot(jb + 1), 1);
      // reads run two MFMAs ahead
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < NPV - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      if (jb + 1 < nkw) qk_from(kslot(jb + 1), kn0, kn1);
      __builtin_amdgcn_s_setprio(0);
    }
    if (jb + 1 < nv) put_v(jb + 1);
    if (jb + 2 < nv) put_k(jb + 2);
    wait_vmem();
    __syncthreads();
  }

  const float ltot = pair_sum(lsum);
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
  // O = acc / l, the correctly rounded fp32 quotient, rounded to the input type
  const float inv = ltot > 0.0f ? 1.0f / ltot : 0.0f;
  auto quot = [&](float v) {
    const float q0 = v * inv;
    return __builtin_fmaf(__builtin_fmaf(-q0, ltot, v), inv, q0);
  };
  const int64_t t = it.row0 + tok;
  uint16_t *op = a.o + t * a.os0 + (int64_t)(hk * a.group + hr) * a.os1 + 4 * g;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      const u32x2 pk = {E::pack2(quot(o[nb][4 * rq]), quot(o[nb][4 * rq + 1])),
                        E::pack2(quot(o[nb][4 * rq + 2]), quot(o[nb][4 * rq + 3]))};
      *(u32x2 *)(op + 32 * nb + 8 * rq) = pk;
    }
  if (g == 0 && a.lse)
    a.lse[t * a.Hq + hk * a.group + hr] = ltot > 0.0f ? row_lse(m, ltot) : -INFINITY;
}

// Combine of a split tile's states, one work-group per (tile, kv head) and 8 (16
// at head_dim 64) of its rows: HD / 4 lanes per row, four elements each.
// M = max m_s, l = sum 2^(m_s - M) l_s, O = sum 2^(m_s - M) O_s / l. A split with
// l_s = 0 (no visible key) may have left no O_s and is passed over.
template <class E, int HD>
__global__ __launch_bounds__(NT) void attn_paged_combine(PagedArgs a) {
  constexpr int LPR = HD / 4, ROWS = NT / LPR;
  const int lane = threadIdx.x & 63;
  const int hk = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % (uint32_t)a.Hk));
  const int idx = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / (uint32_t)a.Hk));
  Item it;
  if (!find_item(a, lane, idx, true, &it) || it.splits <= 1) return;
  const int r = blockIdx.y * ROWS + threadIdx.x / LPR, row = it.tile * BM + r;
  if (r >= BM || row >= it.n * a.group) return;
  const int d = 4 * (threadIdx.x % LPR);
  const int64_t part = ((int64_t)it.part * a.Hk + hk) * a.prows + r;
  const int64_t step = (int64_t)a.Hk * a.prows;
  float M = kNegFltMax;
  for (int s = 0; s < it.splits; ++s) M = fmaxf(M, a.pml[(part + s * step) * 2]);
  float l = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = 0; s < it.splits; ++s) {
    const f32x2 ml = *(const f32x2 *)(a.pml + (part + s * step) * 2);
    if (ml[1] == 0.0f) continue;
    const float wgt = fast_exp2(ml[0] - M);
    l = fmaf(wgt, ml[1], l);
    const f32x4 os = *(const f32x4 *)(a.po + (part + s * step) * HD + d);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = fmaf(wgt, os[k], acc[k]);
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  auto quot = [&](float v) {
    const float q0 = v * inv;
    return __builtin_fmaf(__builtin_fmaf(-q0, l, v), inv, q0);
  };
  const int tok = row / a.group, h = hk * a.group + row - tok * a.group;
  const int64_t t = it.row0 + tok;
  *(u32x2 *)(a.o + t * a.os0 + h * a.os1 + d) =
      u32x2{E::pack2(quot(acc[0]), quot(acc[1])), E::pack2(quot(acc[2]), quot(acc[3]))};
  if (d == 0 && a.lse) a.lse[t * a.Hq + h] = l > 0.0f ? row_lse(M, l) : -INFINITY;
}

// Tiles of one KV head at most: every sequence ends a tile of its own
int64_t most_tiles(const PagedAttnLaunch &L) {
  const int64_t rows = L.tokens * (L.heads_q / L.heads_kv);
  return std::min((rows + (BM - 1) * L.batch) / BM, rows);
}

bool may_split(const PagedAttnLaunch &L) {
  // a split is worth 4 blocks at least, so two need 8; one sequence of at least
  // 2 kSlots items is never cut (its mean chain is at least half its longest)
  if ((L.seq_kv + BN - 1) / BN < 8) return false;
  const int64_t tiles = L.tokens * (L.heads_q / L.heads_kv) / BM;
  return !(L.batch == 1 && tiles * L.heads_kv >= 2 * kSlots);
}

int64_t part_rows(const PagedAttnLaunch &L) {
  return std::min<int64_t>(BM, L.tokens * (L.heads_q / L.heads_kv));
}

template <class E, int HD, bool FP8>
hipError_t launch_t(const PagedArgs &a, const PagedAttnLaunch &L, hipStream_t s) {
  const int64_t tiles = most_tiles(L);
  const int64_t items = (tiles + (a.parts ? kParts / L.heads_kv : 0)) * L.heads_kv;
  hipLaunchKernelGGL((attn_paged<E, HD, FP8>), dim3((unsigned)items), dim3(NT), 0, s, a);
  if (a.parts) {
    constexpr int ROWS = NT / (HD / 4);
    const dim3 grid((unsigned)(tiles * L.heads_kv), (unsigned)((a.prows + ROWS - 1) / ROWS));
    hipLaunchKernelGGL((attn_paged_combine<E, HD>), grid, dim3(NT), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

bool attn_paged_supported(const PagedAttnLaunch &L, const char **why) {
  if (L.head_dim != 64 && L.head_dim != 128) {
    *why = "head_dim must be 64 or 128";
    return false;
  }
  if (L.fp8 && L.dtype != 2) {
    *why = "E4M3 pools take BF16 queries";
    return false;
  }
  if (L.page_size % 16) {
    *why = "the page size must be a multiple of 16 tokens";
    return false;
  }
  const int64_t size = L.fp8 ? 1 : 2;
  // a run's 16 rows lie within 32-bit offsets of its first
  if (15 * L.kps[2] * size + 256 > INT32_MAX || 15 * L.vps[2] * size + 256 > INT32_MAX) {
    *why = "token strides must be below 2^31 / 15 bytes";
    return false;
  }
  if (L.seq_kv > (int64_t)1 << 30 || L.num_pages > INT32_MAX || L.max_pages > INT32_MAX - 64 ||
      L.page_size > (int64_t)1 << 30 || L.batch > (int64_t)1 << 24 || L.tokens > (int64_t)1 << 30 ||
      L.heads_q > 1 << 20 || L.tokens * (L.heads_q / L.heads_kv) > (int64_t)1 << 30 ||
      (most_tiles(L) + kParts) * L.heads_kv * NT > (int64_t)0xffffffff) {
    *why = "shape too large for one launch";
    return false;
  }
  return true;
}

size_t attn_paged_bytes(const PagedAttnLaunch &L) {
  if (!may_split(L)) return 0;
  const size_t parts = (size_t)(kParts / L.heads_kv + 1) * L.heads_kv;
  return parts * part_rows(L) * (L.head_dim + 2) * 4;
}

hipError_t launch_attn_paged(const PagedAttnLaunch &L, hipStream_t s) {
  PagedArgs a;
  const int64_t size = L.fp8 ? 1 : 2;
  a.q = (const uint16_t *)L.q;
  a.k = (const char *)L.k;
  a.v = (const char *)L.v;
  a.ksc = L.k_scales;
  a.vsc = L.v_scales;
  a.btab = L.block_table;
  a.cu = L.cu_seqlens;
  a.lens = L.seq_lens;
  a.o = (uint16_t *)L.o;
  a.lse = L.lse;
  a.qs0 = L.qs[0]; a.qs1 = L.qs[1];
  a.os0 = L.os[0]; a.os1 = L.os[1];
  a.kps0 = L.kps[0] * size; a.kps1 = L.kps[1] * size; a.ktok = L.kps[2] * size;
  a.vps0 = L.vps[0] * size; a.vps1 = L.vps[1] * size; a.vtok = L.vps[2] * size;
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
  a.parts = may_split(L) ? 1 : 0;
  a.prows = (int32_t)part_rows(L);
  a.po = (float *)L.workspace;
  a.pml = a.po + (size_t)(kParts / L.heads_kv + 1) * L.heads_kv * a.prows * L.head_dim;
  a.scale2 = L.scale_log2;
  if (L.fp8)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, true>(a, L, s)
                            : launch_t<Bf16Tag, 128, true>(a, L, s);
  if (L.dtype == 2)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, false>(a, L, s)
                            : launch_t<Bf16Tag, 128, false>(a, L, s);
  return L.head_dim == 64 ? launch_t<F16Tag, 64, false>(a, L, s)
                          : launch_t<F16Tag, 128, false>(a, L, s);
}

}  // namespace neptune
