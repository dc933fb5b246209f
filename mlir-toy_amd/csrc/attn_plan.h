// attn_plan.h — how a launch of attn_paged.hip is cut into work-groups' items: the
// plan that every wave works out from cu_seqlens and seq_lens, and the bounds the
// host sets for it (the grid, the room for states). It stands apart from the kernels
// so that a test can run the same code on the CPU, lane by lane: what it takes of
// the wave are wave_scan, wave_total and together, given by its includer, and the
// builtins for ballots, lane reads, products, roots and reciprocals. PagedAttnLaunch
// is kernels.h's; BM and BN are attn_tile.h's.
#pragma once

#include <algorithm>

namespace neptune {
namespace {

constexpr int kSlots = 512;         // two work-groups on each of 256 CUs
constexpr int kParts = 2 * kSlots;  // items of cut tiles in a launch at most (make_plan)
// Rows up to which a tile takes the narrow form. Measured (us, narrow / wide for such
// tiles): 32 x 1 over 8000 164 / 182, E4M3 95 / 154, 16 x 1-4 over 8000 69 / 79, 1 over
// 2000 12.6 / 13.7; a tile of more rows than one wave's 32 needs the wide one's waves.
constexpr int NARROW = 32;

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
  uint32_t ps16_inv, group_inv, Hk_inv;  // floor((2^32 - 1) / ..), for quotient()
  int32_t items, slots, parts;    // per KV head: work-groups, those of one round, items of
                                  // cut tiles at most (0: no keys are cut)
  int32_t prows;                  // rows of a split item's states
  float scale2;
};

// floor(x / d), inv = floor((2^32 - 1) / d): the estimate is that or one less
__device__ inline int quotient(int x, int d, uint32_t inv) {
  const uint32_t q = __umulhi((uint32_t)x, inv);
  return (int)((uint32_t)x - q * (uint32_t)d >= (uint32_t)d ? q + 1 : q);
}

// run / ps16 and the rest
__device__ inline void page_of(const PagedArgs &a, int run, int *index, int *rest) {
  *index = quotient(run, a.ps16, a.ps16_inv);
  *rest = run - *index * a.ps16;
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
  const int i = min(b, a.B - 1);
  int len = a.lens[i], lo = i, hi = i + 1;
  if (a.cu) {
    lo = a.cu[i];
    hi = a.cu[i + 1];
  }
  together(len, lo, hi);
  lo = min(max(lo, 0), a.T);
  hi = min(max(hi, lo), a.T);
  Seq s;
  s.n = b < a.B ? hi - lo : 0;
  s.row0 = lo;
  s.len = b < a.B ? min(max(len, 0), a.Lmax) : 0;
  s.tiles = (s.n * a.group + BM - 1) / BM;
  s.blocks = (s.len + BN - 1) / BN;
  return s;
}

// The cut of the keys. A work-group's time is its chain of key blocks, and a
// launch's at least its blocks over kSlots work-groups, so chains longer than
// that (make_plan) are cut. A tile of n splits takes blocks / n + 3 + n rows / 62
// blocks of time, the latter two for the combine's launch and for writing and
// reading the states of all rows (rows: full tiles of the launch; 128 rows of
// states are 133 KB, a block some 1.65 us, memory 5 TB/s): least at n =
// sqrt(62 blocks / rows), and no cut where that takes longer than the whole.
// rows_inv: 62 / rows. The quotient blocks / chain is cut to a whole number (a
// quarter block keeps whole ones whole), but for a tile of few rows rounded to
// one: those wait for memory, and more of them side by side help (24 x 12 heads,
// 1 over 7300: 185 / 214 us). Few rows' states are small, but the combine still joins
// them one after the other: kFewRows more rows of them (3 x 1 over 20000, one KV head
// 16.8 / 19.6 us).
// (Uncontracted, so that every wave of both kernels rounds alike.)
__device__ inline int splits_of(int blocks, bool few, float chain_inv, float rows, float rows_inv) {
#pragma clang fp contract(off)
  const float x = (float)blocks;
  const float most = __builtin_amdgcn_sqrtf(x * rows_inv);
  const float quot = (x + 0.25f) * chain_inv;
  const float n = floorf(fminf(few && quot >= 1.5f ? quot + 0.5f : quot, most));
  const float per = ceilf(x * __builtin_amdgcn_rcpf(n));
  return n >= 2.0f && (x - per - 3.0f) * 62.0f > n * rows ? (int)n : 1;
}

struct Plan {
  float chain_inv, rows[2], rows_inv[2];  // of splits_of; [1]: tiles of few rows
  Seq first;                              // of the wave's lane as sequence 0 .. 63
};
constexpr float kFewRows = 1.5f;

__device__ inline int splits_of(const PagedArgs &a, const Plan &p, const Seq &s) {
  const bool few = s.n * a.group <= NARROW;
  return splits_of(s.blocks, few, p.chain_inv, few ? p.rows[1] : p.rows[0],
                   few ? p.rows_inv[1] : p.rows_inv[0]);
}

// The plan of a launch, by every wave for itself, one sequence per lane. The chain
// starts at the launch's blocks (a tile's taken as the mean of its sequence's first
// and last tile's) over kSlots work-groups, two blocks at least (of four: 1 over 3000
// 11.8 / 13.0 us, 100 over 600 15.3 / 17.5), and grows until the items fit: into one
// round of the GPU where the tiles themselves do, else into the launch's
// work-groups, and in any case into the room for states. One round of items that
// differ by up to a factor of two in length did better than two of half as long
// ones wherever tried (8 mixed E4M3 sequences 97 / 120 us, 1 over 32768 28.8 / 31.7,
// 500 over 7000 71 / 98), and a few items more than one round cost nearly a second
// (16 x 1-4 over 8000, 520 items 77, 512 at most 68). Where growing would leave a
// quarter of the GPU idle, the first chain stands if its items are at most 4/3 of a
// round (24 x 12 heads: 576 items 185, 288 items 214).
__device__ inline Plan make_plan(const PagedArgs &a, int lane) {
#pragma clang fp contract(off)
  Plan p;
  p.first = sequence(a, lane);
  p.chain_inv = p.rows[0] = p.rows[1] = p.rows_inv[0] = p.rows_inv[1] = 0.0f;
  if (!a.parts) return p;
  uint64_t work = 0;  // half blocks
  // Sequences that overlap (65536 of them at most, of 2^23 tiles each) may sum to more
  // than 32 bits hold: a lane's tiles stop at MANY, more than any launch has items
  // (attn_paged_supported), and 64 lanes' still fit; rows may wrap, and count only
  // where the tiles fit, at most 2^31 - 128 of them then.
  constexpr int MANY = 1 << 24;
  uint32_t rows = 0;
  int tiles = 0;
  auto add = [&](const Seq &s) {
    const int first = max(s.len - s.n + BN, 0) / BN;
    work += (uint64_t)s.tiles * (uint32_t)(s.blocks + min(first, s.blocks));
    rows += (uint32_t)(s.n * a.group);
    tiles = min(tiles + s.tiles, MANY);
  };
  add(p.first);
  for (int b0 = 64; b0 < a.B; b0 += 64) add(sequence(a, b0 + lane));
  // (exactly, by 21 bits)
  const uint64_t total = (uint64_t)wave_total((int)(work & 0x1fffff)) +
                         ((uint64_t)wave_total((int)((work >> 21) & 0x1fffff)) << 21) +
                         ((uint64_t)wave_total((int)(work >> 42)) << 42);
  tiles = wave_total(tiles);
  if (tiles > a.items) return p;  // sequences that overlap: not all of it is done, nothing is cut
  p.rows[0] = (float)wave_total((int)rows) * (float)a.Hk * (1.0f / BM);
  p.rows[1] = p.rows[0] + kFewRows;
  for (int i = 0; i < 2; ++i) p.rows_inv[i] = 62.0f * __builtin_amdgcn_rcpf(p.rows[i]);
  const uint64_t even = (total * (uint32_t)a.Hk + 2 * kSlots - 1) / (2 * kSlots);
  const int chain0 = (int)min(max(even, (uint64_t)2), (uint64_t)1 << 25);
  int chain = chain0;
  bool fits = false, first_fits = false;
  while (true) {
    p.chain_inv = __builtin_amdgcn_rcpf((float)chain);
    int items = 0, parts = 0;
    auto count = [&](const Seq &s) {
      const int sp = splits_of(a, p, s);
      items += s.tiles * sp;
      parts += sp > 1 ? s.tiles * sp : 0;
    };
    count(p.first);
    for (int b0 = 64; b0 < a.B; b0 += 64) count(sequence(a, b0 + lane));
    items = wave_total(items);
    const bool room = items <= a.items && wave_total(parts) <= a.parts;
    if (fits) return p;  // back at the first chain
    if (chain == chain0) first_fits = room;
    // past 2^25 blocks, longer than any sequence, nothing is cut
    fits = chain >= 1 << 25 || (room && (tiles >= a.slots || items <= a.slots));
    if (fits) {
      if (chain == chain0 || !first_fits || 4 * items >= 3 * a.slots) return p;
      chain = chain0;
    } else {
      chain += max(chain >> 4, 1);  // (by eighths: 16 mixed sequences 79 us, so 76)
    }
  }
}

// Item idx of one KV head, false if there is none. Sequences in order, a
// sequence's tiles from the last (under the causal mask the longest), a tile's
// splits together. take > 0 (it divides BM): instead the idx-th run of `take` rows
// in a cut tile, split the run's first row in its tile.
__device__ inline bool find_item(const PagedArgs &a, const Plan &p, int lane, int idx, int take,
                                 Item *it) {
  int base = 0, parts = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 ? sequence(a, b0 + lane) : p.first;
    const int sp = a.parts ? splits_of(a, p, s) : 1;
    const int mparts = sp > 1 ? s.tiles * sp : 0;
    const int mine = take ? (sp > 1 ? (s.n * a.group + take - 1) / take : 0) : s.tiles * sp;
    const int sum = wave_scan(mine), psum = a.parts ? wave_scan(mparts) : 0;
    const uint64_t past = __ballot(base + sum > idx);
    if (past) {
      const int at = __builtin_ctzll(past);
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      it->b = b0 + at;
      it->n = of(s.n);
      it->row0 = of(s.row0);
      it->len = of(s.len);
      it->tiles = of(s.tiles);
      it->splits = of(sp);
      const int rest = idx - (base + of(sum) - of(mine));
      // tiles before this one in the items' order
      const int down = take             ? it->tiles - 1 - rest * take / BM
                       : it->splits > 1 ? rest / it->splits
                                        : rest;
      it->tile = it->tiles - 1 - down;
      it->split = take ? rest * take % BM : rest - down * it->splits;
      it->part = parts + of(psum) - of(mparts) + down * it->splits;
      return true;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
    parts += __builtin_amdgcn_readlane(psum, 63);
  }
  return false;
}

// Tiles of one KV head at most: every sequence ends a tile of its own
int64_t most_tiles(const PagedAttnLaunch &L) {
  const int64_t rows = L.tokens * (L.heads_q / L.heads_kv);
  return std::min((rows + (BM - 1) * L.batch) / BM, rows);
}

// Whether the device may cut keys: not those of fewer than eight blocks, and one
// sequence of at least 2 kSlots tiles is not cut (its mean chain is at least half
// its longest).
bool may_split(const PagedAttnLaunch &L) {
  if ((L.seq_kv + BN - 1) / BN < 8) return false;
  const int64_t tiles = L.tokens * (L.heads_q / L.heads_kv) / BM;
  return !(L.batch == 1 && tiles * L.heads_kv >= 2 * kSlots);
}

int64_t part_rows(const PagedAttnLaunch &L) {
  return std::min<int64_t>(BM, L.tokens * (L.heads_q / L.heads_kv));
}

// What a launch has room for, per KV head (PagedArgs)
struct Room {
  int64_t items, slots, parts;
};
Room room_of(const PagedAttnLaunch &L) {
  Room r;
  const int64_t tiles = most_tiles(L);
  r.slots = (kSlots + L.heads_kv - 1) / L.heads_kv;
  r.items = tiles;
  r.parts = 0;
  if (may_split(L)) {
    const int64_t splits = ((L.seq_kv + BN - 1) / BN + 2) / 2 + 1;  // splits_of at most
    r.parts = std::min(tiles * splits, (int64_t)kParts / L.heads_kv);
    if (r.parts < 2) r.parts = 0;  // heads enough without
    // work-groups without an item cost some 10 us a thousand
    if (r.parts)
      r.items = std::min(tiles * splits, std::max(tiles + r.slots / 4, r.slots * 4 / 3 + 1));
  }
  return r;
}

// Groups of lanes that join a row's states in the combine: eight where the rows are few
// and a tile may have that many splits (1 over 32768 29.4 us, one group 38.6), else one
// (16 x 8 over 8000 90, eight 96; 6 x 32-130 head_dim-64 tokens over 1500 20, 26; 200
// over 8000 45, 53)
int combine_groups(const PagedAttnLaunch &L, const Room &r) {
  return L.tokens * L.heads_q <= 512 && r.items >= 8 * most_tiles(L) ? 8 : 1;
}

}  // namespace
}  // namespace neptune
