// The plan of a step's rows by adapter: one int32 buffer that moe_mi355x_lora_plan (lora_plan.hip) fills from the
// adapters' numbers and that moe_mi355x_lora_add (lora.hip) reads.  Sections, the tiles from a multiple of 4 ints:
//   head    [16]      counts (LH_*)
//   offsets [L + 2]   first entry in `rows` of each adapter, of the rows without one, and T
//   rows    [T]       the rows in the order of their adapter, those of one adapter in theirs; without one: last
//   tiles   [N][4]    {adapter, first entry in `rows`, rows, 0}: up to tile_rows rows of one adapter
#pragma once

#include "common.h"

constexpr int kLoraMaxRows = 1 << 18;
constexpr int kLoraMaxAdapters = 256;
constexpr int kLoraMaxSeqs = 4096;  // a workgroup holds their offsets in LDS

enum { LH_TILES, LH_INTS = 16 };

struct LoraLayout {
  int T, L;
  int tile_rows;
  int N;  // capacity of the tile list
  long offsets, rows, tiles, ints;
};

static inline bool lora_plan_ok(int T, int L) { return T >= 0 && T <= kLoraMaxRows && L >= 1 && L <= kLoraMaxAdapters; }

// Rows of a tile: few, where each may have an adapter of its own, or many, which share the reading of theirs.
constexpr int kLoraFewRows = 2;
static inline int lora_tile_rows(int T) { return T <= 256 ? kLoraFewRows : 64; }

static inline LoraLayout lora_layout(int T, int L) {
  LoraLayout p{};
  p.T = T, p.L = L, p.tile_rows = lora_tile_rows(T);
  p.N = T / p.tile_rows + (T < L ? T : L);
  p.offsets = LH_INTS;
  p.rows = p.offsets + L + 2;
  p.tiles = (p.rows + T + 3) / 4 * 4;
  p.ints = p.tiles + 4L * p.N;
  return p;
}
