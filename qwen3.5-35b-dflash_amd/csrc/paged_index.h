// Index arithmetic of the paged-cache kernels, shared by the kernels and the host (plain C++: it also compiles without a
// GPU compiler, so that a host test can run it over every size).
//
// Attention work is cut in two directions.  A sequence's block gives ceil(tokens * group / R) row tiles of R rows (row =
// token * group + head in group) per KV head.  A tile's keys are cut into chunks of `c` units of `unit` keys, with one c
// for the whole batch: c = max(c_min, U * kv / slots rounded up), U = sum over sequences of tiles * ceil(keys / unit).  Equal
// chunks keep the workgroups alike whatever the lengths are, and there are at most slots / kv + tiles of them per KV
// head, which bounds the grid without knowing a length on the host.
#pragma once

#include <math.h>
#include <stdint.h>

#if defined(__HIPCC__)
#define DFLASH_HD __host__ __device__ __forceinline__
#else
#define DFLASH_HD inline
#endif

namespace dflash {

// Division of x < 2^31 by a fixed d >= 1: (mulhi(x, mul) + x) >> shift, with 2^shift >= d.
struct FastDiv {
  uint32_t mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t s = 0;
  while (s < 31 && (1u << s) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1), s};
}
DFLASH_HD uint32_t divide(uint32_t x, FastDiv d) {
  return (static_cast<uint32_t>((static_cast<uint64_t>(x) * d.mul) >> 32) + x) >> d.shift;
}

DFLASH_HD int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
DFLASH_HD int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Block and keys of one sequence, from device memory: whatever it holds, tokens lie in [0, T) and keys in [0, capacity].
struct SeqSpan {
  int start, tokens, keys;
};
DFLASH_HD SeqSpan seq_span(int start, int end, int length, int T, int capacity) {
  SeqSpan s;
  s.start = clampi(start, 0, T);
  s.tokens = clampi(end, s.start, T) - s.start;
  s.keys = clampi(length, 0, capacity);
  return s;
}

// Row tiles of a sequence (tokens * group <= 2^22), and units of its keys.
DFLASH_HD int seq_tiles(int tokens, int group, int tile_rows) { return (tokens * group + tile_rows - 1) / tile_rows; }
DFLASH_HD int seq_units(int keys, int unit) { return (keys + unit - 1) / unit; }

// Units a chunk, for `total` (tile, unit) pairs of all sequences per KV head: at least total * kv / slots, whatever the
// product's rounding (a 64-bit division would take longer than the rest of the search).
DFLASH_HD int chunk_units(double total, int kv, double per_slot, int least) {
  const double c = total * kv * per_slot;
  const int up = c < 1e9 ? static_cast<int>(c) + 1 : 1000000001;
  return up < least ? least : up;
}
// A prefix that all sequences share and their own keys, in one launch: of `slots` places the own keys get for_own, in [1, slots - 1]
// whatever the work is, by what the two sides' units take (kUnitCost, kStartCost a row tile, in units of the prefix), and the
// prefix the others.  Each side's chunks are cut for its places: c >= units * kv / places on either side, so together
// there are at most slots / kv + tiles of both, as many as the grid has.
DFLASH_HD float own_places(double own_units, int own_tiles, double front_units, int kv, int slots, float unit_cost, float start_cost) {
  const float own_cost = static_cast<float>(own_units) * unit_cost + static_cast<float>(own_tiles) * start_cost;
  const float places = static_cast<float>(slots), tiles = static_cast<float>(own_tiles * kv);
  float for_own = places * own_cost / (own_cost + static_cast<float>(front_units) + 1.f);
  if (for_own < tiles) for_own = tiles / rintf(tiles / for_own);  // as many row tiles to each place
  return fminf(fmaxf(for_own, 1.f), places - 1.f);
}
constexpr float kAbove = 1.000001f;  // more than the quotients' roundings take off
DFLASH_HD int front_chunk(double units, int kv, int slots, float for_own, int least) {
  return chunk_units(units, kv, kAbove / (static_cast<float>(slots) - for_own), least);
}
DFLASH_HD int own_chunk(double units, int kv, float for_own, int least) { return chunk_units(units, kv, kAbove / for_own, least); }

// Chunks a tile: one at least, which writes the rows of a sequence without keys.
DFLASH_HD int tile_chunks(int units, int c) {
  const int k = static_cast<int>(static_cast<uint32_t>(units + c - 1) / static_cast<uint32_t>(c));
  return k < 1 ? 1 : k;
}
// End of the chunk of c units that starts at key k0, among n keys (c may be far more than they have).
DFLASH_HD int chunk_end(int k0, int c, int unit, int n) {
  const int64_t end = k0 + static_cast<int64_t>(c) * unit;
  return end < n ? static_cast<int>(end) : n;
}

// Keys that token i of a block of `tokens` sees (causal: itself and what lies before it).
DFLASH_HD int visible_keys(int keys, int tokens, int i, bool causal) {
  const int v = causal ? keys - tokens + i + 1 : keys;
  return v < 0 ? 0 : v;
}

// Bounds without knowing any length: tiles of T tokens in B sequences, chunks of one KV head, and partial tiles of all
// KV heads.  Tiles of a single chunk keep no partial result unless another stage's are merged with it (`always`).
inline int64_t max_tiles(int64_t T, int64_t B, int64_t group, int64_t tile_rows) {
  return T * group / tile_rows + (B < T ? B : T);
}
inline int64_t max_chunks(int64_t tiles, int64_t kv, int64_t slots) { return tiles + slots / kv; }
inline int64_t max_partial_tiles(int64_t tiles, int64_t kv, int64_t slots, bool always) {
  const int64_t all = max_chunks(tiles, kv, slots) * kv;
  // a tile in two chunks or more has more than c units, so there are at most slots / kv of them, of twice as many chunks
  return always || all < 2 * slots ? all : 2 * slots;
}

}  // namespace dflash
