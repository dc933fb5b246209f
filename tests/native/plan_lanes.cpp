// Runs attn_plan.h on the CPU: 64 lanes as coroutines that meet at every ballot,
// lane read and sum, as a wave does. stdin: tokens batch heads_q heads_kv head_dim
// seq_kv, whether cu_seqlens follows, its batch + 1 numbers, batch lengths, then the
// asked items as "count index..". stdout: "items slots parts part_rows combine_groups",
// then for each asked index "-" or "b n row0 len tile tiles split splits part".
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <ucontext.h>

#include <algorithm>
#include <vector>

namespace neptune {
struct PagedAttnLaunch {
  int64_t tokens, batch, heads_q, heads_kv, head_dim, seq_kv;
};
constexpr int BM = 128, BN = 64;
using std::max;
using std::min;
}  // namespace neptune

namespace {
constexpr int WAVE = 64;
ucontext_t scheduler, context[WAVE];
int current;
int64_t box[2][WAVE];
int turn[WAVE];

// x of every lane, once all have come here
const int64_t *meet(int64_t x) {
  const int lane = current, side = turn[lane]++ & 1;
  box[side][lane] = x;
  swapcontext(&context[lane], &scheduler);
  return box[side];
}
uint64_t host_ballot(bool x) {
  const int64_t *v = meet(x);
  uint64_t r = 0;
  for (int i = 0; i < WAVE; ++i) r |= (uint64_t)(v[i] != 0) << i;
  return r;
}
int host_readlane(int x, int at) { return (int)meet(x)[at]; }
uint32_t host_umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }
// (wraps, as the device's sums do)
int wave_scan(int x) {
  const int lane = current;
  const int64_t *v = meet(x);
  uint32_t sum = 0;
  for (int i = 0; i <= lane; ++i) sum += (uint32_t)v[i];
  return (int)sum;
}
int wave_total(int x) {
  const int64_t *v = meet(x);
  uint32_t sum = 0;
  for (int i = 0; i < WAVE; ++i) sum += (uint32_t)v[i];
  return (int)sum;
}
void together(int &, int &, int &) {}
}  // namespace

#define __device__
#define __umulhi host_umulhi
#define __ballot host_ballot
#define __builtin_amdgcn_readlane host_readlane
#define __builtin_amdgcn_sqrtf sqrtf
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#include "attn_plan.h"

using namespace neptune;

static PagedArgs args;
static std::vector<int> asked;
static std::vector<Item> found;
static std::vector<char> there;

static void lane_main() {
  const int lane = current;
  const Plan p = make_plan(args, lane);
  for (size_t i = 0; i < asked.size(); ++i) {
    Item it = {};
    const bool yes = find_item(args, p, lane, asked[i], 0, &it);
    if (lane == 0) {
      there[i] = yes;
      found[i] = it;
    }
  }
}

int main() {
  PagedAttnLaunch L;
  int cu = 0;
  if (scanf("%ld %ld %ld %ld %ld %ld %d", &L.tokens, &L.batch, &L.heads_q, &L.heads_kv,
            &L.head_dim, &L.seq_kv, &cu) != 7)
    return 2;
  auto read = [](std::vector<int> &v, size_t n) {
    v.resize(n);
    for (size_t i = 0; i < n; ++i)
      if (scanf("%d", &v[i]) != 1) return false;
    return true;
  };
  std::vector<int> cus, lens, count;
  if (cu && !read(cus, L.batch + 1)) return 2;
  if (!read(lens, L.batch) || !read(count, 1) || !read(asked, count[0])) return 2;
  found.resize(asked.size());
  there.resize(asked.size());
  const Room room = room_of(L);
  args = PagedArgs();
  args.cu = cu ? cus.data() : nullptr;
  args.lens = lens.data();
  args.T = (int)L.tokens;
  args.B = (int)L.batch;
  args.Hq = (int)L.heads_q;
  args.Hk = (int)L.heads_kv;
  args.group = (int)(L.heads_q / L.heads_kv);
  args.Lmax = (int)L.seq_kv;
  args.items = (int)room.items;
  args.slots = (int)room.slots;
  args.parts = (int)room.parts;
  std::vector<char> stacks(WAVE * 65536);
  for (int i = 0; i < WAVE; ++i) {
    getcontext(&context[i]);
    context[i].uc_stack.ss_sp = &stacks[i * 65536];
    context[i].uc_stack.ss_size = 65536;
    context[i].uc_link = nullptr;
    makecontext(&context[i], +[]() {
      lane_main();
      turn[current] = -1;  // done
      swapcontext(&context[current], &scheduler);
    }, 0);
  }
  for (bool live = true; live;) {
    live = false;
    for (int i = 0; i < WAVE; ++i) {
      if (turn[i] < 0) continue;
      current = i;
      swapcontext(&scheduler, &context[i]);
      live = live || turn[i] >= 0;
    }
  }
  printf("%ld %ld %ld %ld %d\n", room.items, room.slots, room.parts, part_rows(L),
         combine_groups(L, room));
  for (size_t i = 0; i < asked.size(); ++i) {
    const Item &t = found[i];
    if (!there[i])
      printf("-\n");
    else
      printf("%d %d %d %d %d %d %d %d %d\n", t.b, t.n, t.row0, t.len, t.tile, t.tiles, t.split,
             t.splits, t.part);
  }
  return 0;
}
