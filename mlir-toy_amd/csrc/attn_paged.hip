// attn_paged.hip — attention over a paged cache: what is covered, the launch, and
// the kernels of plain scores over 16-bit and E4M3 pools (attn_paged_kernel.h).
#include "attn_paged_kernel.h"

namespace neptune {

bool attn_paged_supported(const PagedAttnLaunch &L, const char **why) {
  if (L.head_dim != 64 && L.head_dim != 128) {
    *why = "head_dim must be 64 or 128";
    return false;
  }
  if (L.pool == E4M3 && L.dtype != 2) {
    *why = "E4M3 pools take BF16 queries";
    return false;
  }
  if (L.page_size % 16) {
    *why = "the page size must be a multiple of 16 tokens";
    return false;
  }
  const int64_t size = L.pool == WIDE ? 2 : 1;
  // a run's 16 rows lie within 32-bit offsets of its first
  const int64_t most = (INT32_MAX - 256) / 15 / size;
  if (L.kps[2] > most || L.vps[2] > most || L.kss[2] > most || L.vss[2] > most) {
    *why = "token strides must be below 2^31 / 15 bytes";
    return false;
  }
  if (L.pool == MXFP4)
    // a page's offset is a product of 32-bit factors, and 32 bits hold a place's within it
    for (const int64_t *t : {L.kps, L.vps, L.kss, L.vss})
      if (t[0] > INT32_MAX || t[2] > INT32_MAX / std::max<int64_t>(L.page_size, 1)) {
        *why = "MXFP4 pools' pages must lie less than 2 GiB apart, and their tokens within as much";
        return false;
      }
  if (L.seq_kv > (int64_t)1 << 30 || L.num_pages > INT32_MAX || L.max_pages > INT32_MAX - 64 ||
      L.page_size > (int64_t)1 << 30 || L.batch > 1 << 16 || L.tokens > (int64_t)1 << 30 ||
      L.heads_q > 1 << 20 || L.tokens * (L.heads_q / L.heads_kv) > (int64_t)1 << 30 ||
      (most_tiles(L) + kParts) * L.heads_kv * NT > (int64_t)0xffffffff) {
    *why = "shape too large for one launch";
    return false;
  }
  return true;
}

size_t attn_paged_bytes(const PagedAttnLaunch &L) {
  const size_t parts = (size_t)room_of(L).parts * L.heads_kv;
  return parts * part_rows(L) * (L.head_dim + 2) * 4;
}

hipError_t launch_attn_paged(const PagedAttnLaunch &L, hipStream_t s) {
  if (L.pool == MXFP4) return launch_attn_paged_mx(L, s);
  if (shaped(L)) return launch_attn_paged_shaped(L, s);
  const PagedArgs a = paged_args(L);
  if (L.pool == E4M3)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, E4M3, false>(a, L, s)
                            : launch_t<Bf16Tag, 128, E4M3, false>(a, L, s);
  if (L.dtype == 2)
    return L.head_dim == 64 ? launch_t<Bf16Tag, 64, WIDE, false>(a, L, s)
                            : launch_t<Bf16Tag, 128, WIDE, false>(a, L, s);
  return L.head_dim == 64 ? launch_t<F16Tag, 64, WIDE, false>(a, L, s)
                          : launch_t<F16Tag, 128, WIDE, false>(a, L, s);
}

}  // namespace neptune
