// The plan of a step's rows by adapter: one int32 buffer that moe_mi355x_lora_plan (lora_plan.hip) fills from the
// adapters' numbers and that moe_mi355x_lora_add (lora.hip) reads.  Sections, the tiles from a multiple of 4 ints:
//   head    [16]      counts (LH_*)
//   offsets [L + 2]   first entry in `rows` of each adapter, of the rows without one, and T
//   rows    [T]       the rows in the order of their adapter, those of one adapter in theirs; without one: last
//   tiles   [N][4]    {adapter, first entry in `rows`, rows, 0}: up to kLoraRows rows of one adapter
//   pairs   [M][4]    the same, up to kLoraPair rows (steps of up to kLoraFewT rows)
#pragma once

#include "common.h"

constexpr int kLoraMaxRows = 1 << 18;
constexpr int kLoraMaxAdapters = 256;
constexpr int kLoraMaxSeqs = 4096;  // a workgroup holds their offsets in LDS

constexpr int kLoraRows = 64;   // rows of a tile, which share the reading of their adapter
constexpr int kLoraPair = 2;    // of a small one, where each row may have an adapter of its own
constexpr int kLoraFewT = 256;  // rows of a step that is cut into small ones too

enum { LH_TILES, LH_PAIRS, LH_INTS = 16 };

struct LoraLayout {
  int T, L;
  int N, M;  // capacities of the lists
  long offsets, rows, tiles, pairs, ints;
};

static inline bool lora_plan_ok(int T, int L) { return T >= 0 && T <= kLoraMaxRows && L >= 1 && L <= kLoraMaxAdapters; }

static inline LoraLayout lora_layout(int T, int L) {
  LoraLayout p{};
  p.T = T, p.L = L;
  const int some = T < L ? T : L;  // adapters that may have rows
  p.N = T / kLoraRows + some;
  p.M = T <= kLoraFewT ? T / kLoraPair + some : 0;
  p.offsets = LH_INTS;
  p.rows = p.offsets + L + 2;
  p.tiles = (p.rows + T + 3) / 4 * 4;
  p.pairs = p.tiles + 4L * p.N;
  p.ints = p.pairs + 4L * p.M;
  return p;
}
