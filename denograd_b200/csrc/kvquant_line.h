// How attention over the 8-bit cache is cut over CTAs, as plain C++: the kernels work it out on the GPU, and a test walks it on the host.
//
// The units of work of all items (a (sequence, kv head), or some rows of one) are one line, with some more for what each item costs by itself,
// and the line is cut evenly over the CTAs.  An item on several CTAs is made in pieces, which are left in a workspace and put together.
//
// Nothing that a launch shares is shared by two items, because a cut of the line lies in one item at most:
//   slots    2 c for the piece of CTA c that the cut in front of its stretch lies in, 2 c + 1 for one that only the cut behind it lies in
//   tickets  every count of arrivals is named by the CTA ahead of a cut that lies in its item: the first of the item's CTAs, or of a group of at
//            least two of them.  (A group of one has nothing to add up and counts nothing: its CTA may be the first one of the next item.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define KVQ_LINE __host__ __device__ __forceinline__
#else
#define KVQ_LINE static inline
#endif

// Where CTA c's stretch of a line of `total` units begins, and CTA c - 1's ends.  In 32 bits as long as c * total fits: up to 2^(32 - BITS) CTAs.
template <int BITS>
KVQ_LINE long long kvq_cut(long long total, long long ctas, unsigned c) {
  if (total < (1ll << BITS)) return c * (uint32_t)total / (uint32_t)ctas;
  return c * total / ctas;
}
// The CTA whose stretch holds a unit.
KVQ_LINE int kvq_owner(long long total, long long ctas, long long at) { return (int)(((at + 1) * ctas - 1) / total); }
// The place in the workspace of a CTA's piece of an item that others have pieces of: `first` of them or not.
KVQ_LINE int kvq_slot(int cta, bool first) { return 2 * cta + (first ? 1 : 0); }

// Few queries (kvquant_split.cuh): units of 64 positions; pieces that are added up ahead of the others, where there are many.
constexpr int KS_WARPS = 4, KS_UNIT = 16 * KS_WARPS, KS_GROUP = 8, KS_BITS = 20;
// Units that a (sequence, kv head) costs beside its own, by column groups.  One: 1, 3 and 6 within 1 %; more: 8 sequences of 5 positions behind 3001 of
// the 8B, in L2, 30.9 us with 3, 29.5 with 5, 29.8 with 7 (30 ragged ones 25.5, 25.3, 27.1).
constexpr int ks_fixed(int groups) { return groups == 1 ? 3 : 5; }
// A piece's group: pieces from .. to - 1 of the item, added up first and counted at `ticket` (-1: there is none).  Not grouped: the piece itself.
struct KsGroup {
  int from, to, step, ticket;  // step: pieces to a group
};
KVQ_LINE KsGroup ks_group(int piece, int pieces, int c_lo) {
  KsGroup g;
  g.step = pieces > KS_GROUP + KS_GROUP / 2 ? KS_GROUP : 1;
  g.from = piece / g.step * g.step;
  g.to = g.from + g.step < pieces ? g.from + g.step : pieces;
  g.ticket = g.to - g.from > 1 ? c_lo + g.from : -1;
  return g;
}
// Groups of an item, and where they are counted as they are done.
KVQ_LINE int ks_groups(int pieces, int step) { return (pieces + step - 1) / step; }
KVQ_LINE int ks_last_ticket(int grid, int c_lo) { return grid + c_lo; }

// Chunks (kvquant_chunk.cu): query rows of an item, keys of a tile; tiles: see the line of tiles there.
constexpr int KC_ROWS = 256, KC_KEYS = 128, KC_WHOLE = 8, KC_SINGLE = 12, KC_GRAIN = 2, KC_FIXED = 2, KC_BITS = 23;
// Pieces of an item that have arrived, and CTAs that are done with waiting for them.
KVQ_LINE int kc_ticket(int c_lo) { return c_lo; }
KVQ_LINE int kc_done_ticket(int grid, int c_lo) { return grid + c_lo; }
