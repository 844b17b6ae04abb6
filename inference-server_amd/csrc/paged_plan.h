// The plan of a step over the 8-bit paged KV cache: one int32 buffer that moe_mi355x_paged_plan
// (paged_plan.hip) fills from the sequences' lengths and that the cache writers (kv_fp8.hip) and the
// attention (attn_fp8.hip) read.  Sections, the lists from a multiple of 16 ints:
//   head    [16]         counts (PH_*)
//   cu      [B + 1]      first token of each sequence in the step's T rows
//   context [B]          tokens of each sequence with this step's
//   pos     [T]          position of each token in its sequence (-1: a row behind the last sequence)
//   slot    [T]          16 * page + slot of each token (-1: none)
//   writes  [W][4]       pages that get tokens: {page or -1, first token, its slot, tokens}
//   shorts  [S][8]       attention items of sequences with few query rows (PI_*)
//   tiles   [N][8]       attention items of the others: 128 or 256 query rows (PI_*)
//   short_merges [..][4] sequences, resp. tiles, whose keys are split over items: {items, first item, first
//   tile_merges  [..][4] token, tokens}
#pragma once

#include "common.h"

constexpr int kPlanPage = 16;        // tokens per page
constexpr int kPlanMaxSeqs = 4096;   // a workgroup holds every sequence's offsets in LDS
constexpr int kPlanMaxTokens = 1 << 18;
constexpr int kPlanMaxPages = 1 << 22;  // per sequence

constexpr int kShortRows = 16;       // query rows (tokens x heads of the group) of a short item
constexpr int kTileRows = 128;       // and of a tile, or, where rows fill so many of them,
constexpr int kTileRowsMany = 256;   // of these: the cache is widened and staged half as often (a prompt of 4096
constexpr int kManyTiles = 512;      // tokens, 32 / 4 heads: 154 -> 139 us; at 2500, half as many: 73 -> 120)
constexpr int kShortStep = 8;        // pages that a short item's workgroup takes at once
// Items that short sequences are split into, over all kv heads: three for each CU.  (128 sequences of 512 to 8192
// tokens, 32 / 4 heads, in us, for 512 / 768 / 1024 / 2048: 95.7 / 94.8 / 98.2 / 101.7; two of 100000 and more:
// 45.8 / 47.6 / 49.4 / 58.0; 64 of up to 8192, 32 / 8 heads: 90.7 / 89.0 / 89.1 / 92.4.)
constexpr int kShortTarget = 768;
// Tables of up to so many pages, for many (sequence, kv head) pairs and for few: a short sequence is one item and there
// is nothing to join, which saves the merge's launch.  (us in a graph, whole against split: one sequence of 1000
// tokens and 4 kv heads 7.5 / 7.4, of 1400 8.9 / 6.9; 16 of 700..1400 10.1 / 10.7, of 1000..2000 13.6 / 12.2; 100 of
// 500..2000 27.0 / 29.9.  Without a graph a launch is 2.7 us of the host's time besides.)
constexpr int kShortWhole = 128;
constexpr int kShortWholeFew = 80;
constexpr int kFewPairs = 64;
// Fewer tiles than this, one per CU, are split along their keys, for twice as many workgroups in all and
// kTileMinKeys at least.  (8000 cached tokens and n new ones, 32 / 4 heads, split against whole: n = 100 47 us / 61,
// 200 79 / 86, 700 169 / 174; one more would not pay, n = 1024 228 / 180.)
constexpr int kTileFew = 256;
constexpr int kTileTarget = 512;
constexpr int kTileMinKeys = 512;
constexpr int kTileKeys = 64;        // keys and pages per step of a tile
constexpr int kTilePages = kTileKeys / kPlanPage;

enum { PH_TOKENS, PH_WRITES, PH_SHORTS, PH_TILES, PH_SHORT_MERGES, PH_TILE_MERGES, PH_PAGES = 15, PH_INTS };
// page_begin .. page_end: the item's keys; parts: items that share the rows (1: none other)
enum { PI_SEQ, PI_TOK, PI_NTOK, PI_POS, PI_PAGE0, PI_PAGE1, PI_PARTS, PI_INTS = 8 };

struct PlanLayout {
  int B, T, max_new, max_pages, Hq, Hkv, G;
  int tile_rows, tile_tok;    // rows and tokens of a tile
  int short_rows;             // query rows that a short item may have
  bool short_whole;           // short sequences are not split
  int W, S, N, SM, TM;        // list capacities
  int split_tiles;            // tiles, and items of tiles, that may hold partial results
  long cu, ctx, pos, slot, writes, shorts, tiles, short_merges, tile_merges, ints;  // offsets
};

static inline bool plan_shape_ok(const moe_mi355x_plan_shape* s) {
  return s && s->seqs >= 0 && s->seqs <= kPlanMaxSeqs && s->tokens >= 0 && s->tokens <= kPlanMaxTokens &&
         s->max_new >= 1 && s->max_pages >= 1 && s->max_pages <= kPlanMaxPages && s->heads >= 1 && s->kv_heads >= 1 &&
         s->kv_heads <= 1024 && s->heads % s->kv_heads == 0 && s->heads / s->kv_heads <= kShortRows;
}

static inline PlanLayout plan_layout(const moe_mi355x_plan_shape* s) {
  PlanLayout p{};
  p.B = s->seqs, p.T = s->tokens, p.max_pages = s->max_pages, p.Hq = s->heads, p.Hkv = s->kv_heads;
  p.max_new = s->max_new < p.T ? s->max_new : p.T;
  p.G = p.Hq / p.Hkv;
  p.tile_rows = (long)p.T * p.Hq / kTileRowsMany >= kManyTiles ? kTileRowsMany : kTileRows;
  p.tile_tok = p.tile_rows / p.G;
  const long B = p.B, T = p.T;
  // a sequence with n new tokens touches at most (n + 30) / 16 pages, and at most n
  p.W = (int)(T < (T + 30 * B) / 16 ? T : (T + 30 * B) / 16);
  const long seqs = B < T ? B : T;  // with new tokens
  const long per = (s->max_pages + kShortStep - 1) / kShortStep;
  p.short_rows = (long)p.max_new * p.G < kShortRows ? p.max_new * p.G : kShortRows;
  p.short_whole = p.max_pages <= (seqs * p.Hkv <= kFewPairs ? kShortWholeFew : kShortWhole);
  const long by_target = seqs + (kShortTarget + p.Hkv - 1) / p.Hkv, by_pages = p.short_whole ? seqs : seqs * per;
  p.S = (int)(by_target < by_pages ? by_target : by_pages);
  // no sequence is long enough for tiles: none
  const bool tiles = (long)p.max_new * p.G > kShortRows;
  const long nt = tiles ? T / p.tile_tok + seqs : 0;
  const long few = (kTileFew + p.Hkv - 1) / p.Hkv, whole = nt < few ? nt : few;
  p.split_tiles = (int)(tiles ? whole + (kTileTarget + p.Hkv - 1) / p.Hkv : 0);
  p.N = (int)(nt > p.split_tiles ? nt : p.split_tiles);
  p.SM = (int)seqs;
  p.TM = (int)whole;
  p.cu = PH_INTS;
  p.ctx = p.cu + B + 1;
  p.pos = p.ctx + B;
  p.slot = p.pos + T;
  p.ints = (p.slot + T + 15) / 16 * 16;
  auto at = [&](long ints) {
    const long here = p.ints;
    p.ints += (ints + 15) / 16 * 16;
    return here;
  };
  p.writes = at(4L * p.W);
  p.shorts = at((long)PI_INTS * p.S);
  p.tiles = at((long)PI_INTS * p.N);
  p.short_merges = at(4L * p.SM);
  p.tile_merges = at(4L * p.TM);
  return p;
}
