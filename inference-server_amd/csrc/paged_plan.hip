// Block tables, slots and work lists of a step over the 8-bit paged KV cache, from the sequences' lengths
// alone and without the host: the lengths live on the GPU, so a captured step plans itself.
//
// With c_b = clamp(cached_b, 0, 16 max_pages) and the step's T rows filled in sequence order,
//   cu[b+1] = min(T, sum_{i <= b} clamp(new_i, 0, max_new)),   n_b = cu[b+1] - cu[b]
//   have_b = ceil(c_b / 16),  all_b = min(max_pages, ceil((c_b + n_b) / 16)),  first_b = sum_{i < b} (all_i - have_i)
//   block_tables[b][have_b + i] = free_pages[first_b + i]   (-1 past the list's end)
//   pos[t] = c_b + t - cu[b],  slot[t] = 16 block_tables[b][pos / 16] + pos % 16
// The lists of pages to write and of attention items follow from the same sums.
//
// One launch.  Every workgroup forms the prefix sums over the sequences by itself (4 B of two arrays
// each, in LDS afterwards): cheaper than a launch of its own for them.  Workgroup 0 then builds the attention
// lists, the others take 1024 tokens each.  A new page's table entry and write record come from its first
// token's thread, so nothing waits for anything and every list has one order.
#include "paged_plan.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / MOE_WAVE;

struct PlanArgs {
  const int32_t *cached, *fresh;  // tokens of each sequence: in the cache, new
  int32_t* tables;
  const int32_t* free_pages;
  int n_free;
  int32_t* plan;
  PlanLayout p;
};

// Exclusive prefix sum over the workgroup; *total gets the sum.  Every thread calls it.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* total, T* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T t = __shfl_up(incl, d);
    if (lane >= d) incl += t;
  }
  __syncthreads();  // the last call's sums are read
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? s_wave[w] : 0;
    all += s_wave[w];
  }
  *total = all;
  return before + incl - v;
}

// The last index i < n with s[i] <= x, for s ascending from s[0] <= x.
__device__ __forceinline__ int last_le(const int* s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPlanPage - 1) / kPlanPage; }

__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a) {
  const PlanLayout& p = a.p;
  __shared__ int s_cu[kPlanMaxSeqs + 1], s_a[kPlanMaxSeqs + 1], s_b[kPlanMaxSeqs + 1];
  __shared__ long s_sum[kWaves];
  int* s_isum = (int*)s_sum;
  const int tid = threadIdx.x;
  const int per = (p.B + kThreads - 1) / kThreads;  // sequences per thread, 4 at most
  const int b0 = tid * per;
  const int room = p.max_pages * kPlanPage;
  int32_t* plan = a.plan;

  int c[4], n[4];
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool live = i < per && b0 + i < p.B;
    c[i] = live ? min(max(a.cached[b0 + i], 0), room) : 0;
    n[i] = live ? min(max(a.fresh[b0 + i], 0), p.max_new) : 0;
    sum += n[i];  // <= 4096 * 2^18
  }
  int total;
  int at = block_scan(sum, &total, s_isum);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int first = min(at, p.T);
    at += n[i];
    n[i] = min(at, p.T) - first;
    if (i < per && b0 + i < p.B) s_cu[b0 + i] = first;
  }
  total = min(total, p.T);
  if (tid == 0) s_cu[p.B] = total;

  if (blockIdx.x > 0) {  // tokens: page records and slots
    int need = 0, touched = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      need += pages_of(min(c[i] + n[i], room)) - pages_of(c[i]);
      touched += n[i] > 0 ? (c[i] + n[i] - 1) / kPlanPage - c[i] / kPlanPage + 1 : 0;
    }
    int all_need, all_touched;
    int need_at = block_scan(need, &all_need, s_isum);
    int touched_at = block_scan(touched, &all_touched, s_isum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < per && b0 + i < p.B) {
        s_a[b0 + i] = need_at;
        s_b[b0 + i] = touched_at;
        need_at += pages_of(min(c[i] + n[i], room)) - pages_of(c[i]);
        touched_at += n[i] > 0 ? (c[i] + n[i] - 1) / kPlanPage - c[i] / kPlanPage + 1 : 0;
      }
    }
    __syncthreads();
    if (blockIdx.x == 1 && tid == 0) {
      plan[PH_WRITES] = all_touched;
      plan[PH_PAGES] = all_need;
    }
    const int t = (blockIdx.x - 1) * kThreads + tid;
    if (t >= p.T) return;
    if (t >= total) {
      plan[p.pos + t] = -1;
      plan[p.slot + t] = -1;
      return;
    }
    const int b = last_le(s_cu, p.B, t);  // the last of those that begin at or before t: the one that has tokens
    const int first = s_cu[b], count = s_cu[b + 1] - first;
    const int cached = min(max(a.cached[b], 0), room);
    const int pos = cached + (t - first);
    const int j = pos / kPlanPage, have = pages_of(cached);
    int page = -1;
    if (j < p.max_pages) {
      if (j < have) {
        page = a.tables[(long)b * p.max_pages + j];
      } else {
        const int f = s_a[b] + j - have;
        page = f < a.n_free ? a.free_pages[f] : -1;
        if (pos % kPlanPage == 0) a.tables[(long)b * p.max_pages + j] = page;
      }
      if (page < 0 || page >= (1 << 27)) page = -1;  // no pool has so many pages
    }
    plan[p.pos + t] = pos;
    plan[p.slot + t] = page < 0 ? -1 : page * kPlanPage + pos % kPlanPage;
    if (t == first || pos % kPlanPage == 0) {
      const int w = s_b[b] + j - cached / kPlanPage;
      const int some = min(kPlanPage - pos % kPlanPage, first + count - t);
      *(int4*)(plan + p.writes + 4L * w) = make_int4(page, t, pos % kPlanPage, some);
    }
    return;
  }

  // workgroup 0: offsets, contexts and the attention's lists
  long short_pages = 0, tile_keys = 0;
  int tiles = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < per && b0 + i < p.B) {
      plan[p.cu + b0 + i] = s_cu[b0 + i];
      plan[p.ctx + b0 + i] = min(c[i] + n[i], room);
      if (n[i] > 0 && n[i] * p.G <= kShortRows) short_pages += pages_of(min(c[i] + n[i], room));
      if (n[i] * p.G > kShortRows) {
        const long nt = (n[i] + p.tile_tok - 1) / p.tile_tok;
        tiles += (int)nt;
        tile_keys += nt * c[i] + p.tile_tok * (nt * (nt - 1) / 2) + n[i];
      }
    }
  }
  if (tid == 0) plan[p.cu + p.B] = total;
  long all_pages, all_keys;
  int all_tiles;
  block_scan(short_pages, &all_pages, s_sum);
  block_scan(tile_keys, &all_keys, s_sum);
  int tile_at = block_scan(tiles, &all_tiles, s_isum);
  // pages per short item
  long pps = (all_pages * p.Hkv + kShortTarget - 1) / kShortTarget;
  pps = max(pps, 1L) + kShortStep - 1;
  pps = pps / kShortStep * kShortStep;
  // keys per item of a tile; with enough tiles to fill the GPU they are not split
  long chunk = (all_keys * p.Hkv + kTileTarget - 1) / kTileTarget;
  chunk = (max(chunk, (long)kTileMinKeys) + kTileKeys - 1) / kTileKeys * kTileKeys;
  if ((long)all_tiles * p.Hkv >= kTileTarget) chunk = 1L << 40;

  int items = 0, merged = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pages = pages_of(min(c[i] + n[i], room));
    const int ns = n[i] > 0 && n[i] * p.G <= kShortRows ? (int)((pages + pps - 1) / pps) : 0;
    items += ns;
    merged += ns > 1;
  }
  int n_items, n_merged;
  int item_at = block_scan(items, &n_items, s_isum);
  int merge_at = block_scan(merged, &n_merged, s_isum);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(i < per && b0 + i < p.B)) continue;
    const int b = b0 + i, pages = pages_of(min(c[i] + n[i], room));
    const int ns = n[i] > 0 && n[i] * p.G <= kShortRows ? (int)((pages + pps - 1) / pps) : 0;
    s_a[b] = item_at;
    s_b[b] = tile_at;
    if (ns > 1) {
      *(int4*)(plan + p.merges + 4L * merge_at) = make_int4(ns, item_at, s_cu[b], n[i]);
      ++merge_at;
    }
    item_at += ns;
    if (n[i] * p.G > kShortRows) tile_at += (n[i] + p.tile_tok - 1) / p.tile_tok;
  }
  if (tid == 0) {
    s_a[p.B] = n_items;
    s_b[p.B] = all_tiles;
  }
  __syncthreads();

  for (int k = tid; k < n_items; k += kThreads) {
    const int b = last_le(s_a, p.B, k);
    const int first = s_cu[b], count = s_cu[b + 1] - first;
    const int cached = min(max(a.cached[b], 0), room);
    const int pages = pages_of(min(cached + count, room)), ns = s_a[b + 1] - s_a[b];
    // equal shares, each a multiple of what a workgroup takes at once
    const int share = (pages + ns * kShortStep - 1) / (ns * kShortStep) * kShortStep;
    const int page0 = (k - s_a[b]) * share;
    int4* dst = (int4*)(plan + p.shorts + (long)PI_INTS * k);
    dst[0] = make_int4(b, first, count, cached);
    dst[1] = make_int4(page0, min(page0 + share, pages), ns, 0);
  }

  int n_tile_items = 0;
  for (int k0 = 0; k0 < all_tiles; k0 += kThreads) {  // workgroup-uniform
    const int k = k0 + tid;
    int ns = 0, b = 0, tok = 0, count = 0, pos = 0, keys = 0;
    if (k < all_tiles) {
      b = last_le(s_b, p.B, k);
      const int first = s_cu[b], n_b = s_cu[b + 1] - first;
      // a sequence's last tiles, which have the most keys, first
      const int i = s_b[b + 1] - 1 - k;
      tok = first + i * p.tile_tok;
      count = min(p.tile_tok, n_b - i * p.tile_tok);
      pos = min(max(a.cached[b], 0), room) + i * p.tile_tok;
      keys = min(pos + count, room);
      ns = (int)((keys + chunk - 1) / chunk);
    }
    int round, round_merged;
    const int item = n_tile_items + block_scan(ns, &round, s_isum);
    const int merge = n_merged + block_scan(ns > 1 ? 1 : 0, &round_merged, s_isum);
    if (ns > 1) *(int4*)(plan + p.merges + 4L * merge) = make_int4(-ns, item, tok, count);
    for (int s = 0; s < ns; ++s) {
      const int pages = pages_of(keys), step = ns > 1 ? (int)(chunk / kPlanPage) : pages;
      int4* dst = (int4*)(plan + p.tiles + (long)PI_INTS * (item + s));
      dst[0] = make_int4(b, tok, count, pos);
      dst[1] = make_int4(s * step, min((s + 1) * step, pages), ns, 0);
    }
    n_tile_items += round;
    n_merged += round_merged;
  }
  if (tid == 0) {
    plan[PH_TOKENS] = total;
    plan[PH_SHORTS] = n_items;
    plan[PH_TILES] = n_tile_items;
    plan[PH_MERGES] = n_merged;
  }
}

}  // namespace

extern "C" size_t moe_mi355x_paged_plan_bytes(const moe_mi355x_plan_shape* shape, int32_t* offsets) {
  if (!plan_shape_ok(shape)) return 0;
  const PlanLayout p = plan_layout(shape);
  if (offsets) {
    const long at[MOE_PLAN_SECTIONS] = {PH_PAGES, p.cu, p.ctx, p.pos, p.slot};
    for (int i = 0; i < MOE_PLAN_SECTIONS; ++i) offsets[i] = (int32_t)at[i];
  }
  return (size_t)p.ints * sizeof(int32_t);
}

extern "C" int moe_mi355x_paged_plan(const int32_t* cached_lens, const int32_t* new_lens, int32_t* block_tables,
                                     const int32_t* free_pages, int n_free, const moe_mi355x_plan_shape* shape,
                                     void* plan, size_t plan_bytes, void* stream) {
  MOE_RETURN_IF(!plan_shape_ok(shape) || n_free < 0, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(shape->seqs > 0 && (!cached_lens || !new_lens || !block_tables), MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(n_free > 0 && !free_pages, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(!plan || plan_bytes < moe_mi355x_paged_plan_bytes(shape, nullptr), MOE_ERR_WORKSPACE);
  MOE_RETURN_IF(!moe_aligned16(plan), MOE_ERR_ALIGNMENT);
  const PlanArgs a{cached_lens, new_lens, block_tables, free_pages, n_free, (int32_t*)plan, plan_layout(shape)};
  const int blocks = 1 + (a.p.T + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(blocks < 2 ? 2 : blocks), dim3(kThreads), 0, (hipStream_t)stream, a);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
