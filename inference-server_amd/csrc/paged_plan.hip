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
// each, in LDS afterwards): cheaper than a launch of its own for them.  Workgroups 0 and 1 then build the
// attention's two lists, the others take 256 tokens each.  A new page's table entry and write record come from its first
// token's thread, so nothing waits for anything and every list has one order.
#include "paged_plan.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / MOE_WAVE;
constexpr int kClasses = kThreads;  // of a tile's keys

struct PlanArgs {
  const int32_t *cached, *fresh;  // tokens of each sequence: in the cache, new
  int32_t* tables;
  const int32_t* free_pages;
  int n_free;
  int32_t* plan;
  PlanLayout p;
};

// Exclusive prefix sums of N values over the workgroup; v becomes them, total the sums.  Every thread calls it.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*s_wave)[kWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl[N];
#pragma unroll
  for (int k = 0; k < N; ++k) incl[k] = v[k];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int t = __shfl_up(incl[k], d);
      if (lane >= d) incl[k] += t;
    }
  __syncthreads();  // the last call's sums are read
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < N; ++k) s_wave[k][wave] = incl[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? s_wave[k][w] : 0;
      all += s_wave[k][w];
    }
    total[k] = all;
    v[k] = before + incl[k] - v[k];
  }
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
  // per sequence: tokens cached, first row, and two prefix sums that the workgroup needs
  __shared__ int s_cached[kPlanMaxSeqs], s_cu[kPlanMaxSeqs + 1], s_a[kPlanMaxSeqs + 1], s_b[kPlanMaxSeqs + 1];
  __shared__ int s_wave[3][kWaves];
  __shared__ unsigned long long s_sum;
  __shared__ int s_most, s_merged, s_class[kClasses];
  const int tid = threadIdx.x;
  const int per = (p.B + kThreads - 1) / kThreads;  // sequences per thread: b0 .. b1
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  const int room = p.max_pages * kPlanPage;
  int32_t* plan = a.plan;

  int row[1] = {0}, total[1];
  for (int b = b0; b < b1; ++b) {
    s_cached[b] = min(max(a.cached[b], 0), room);
    s_b[b] = min(max(a.fresh[b], 0), p.max_new);
    row[0] += s_b[b];  // <= 4096 * 2^18
  }
  if (tid == 0) s_sum = s_most = s_merged = 0;
  block_scan(row, total, s_wave);
  total[0] = min(total[0], p.T);
  for (int b = b0; b < b1; ++b) {
    s_cu[b] = min(row[0], p.T);
    row[0] += s_b[b];
  }
  if (tid == 0) s_cu[p.B] = total[0];
  const int end = min(row[0], p.T);  // of this thread's last sequence
  // a thread knows its own sequences' new tokens without waiting for the others
  auto new_of = [&](int b) __attribute__((always_inline)) { return (b + 1 < b1 ? s_cu[b + 1] : end) - s_cu[b]; };

  if (blockIdx.x > 1) {  // tokens: page records and slots
    int at[2] = {0, 0}, all[2];  // new pages, pages that get tokens
    auto count = [&](int b) __attribute__((always_inline)) {
      const int c = s_cached[b], n = new_of(b);
      at[0] += pages_of(min(c + n, room)) - pages_of(c);
      at[1] += n > 0 ? (c + n - 1) / kPlanPage - c / kPlanPage + 1 : 0;
    };
    for (int b = b0; b < b1; ++b) count(b);
    block_scan(at, all, s_wave);
    for (int b = b0; b < b1; ++b) {
      s_a[b] = at[0];
      s_b[b] = at[1];
      count(b);
    }
    __syncthreads();
    if (blockIdx.x == 2 && tid == 0) {
      plan[PH_PAGES] = all[0];
      plan[PH_WRITES] = all[1];
    }
    const int t = (blockIdx.x - 2) * kThreads + tid;
    if (t >= p.T) return;
    if (t >= total[0]) {
      plan[p.pos + t] = -1;
      plan[p.slot + t] = -1;
      return;
    }
    const int b = last_le(s_cu, p.B, t);  // the last of those that begin at or before t: the one that has tokens
    const int row0 = s_cu[b], cached = s_cached[b];
    const int pos = cached + (t - row0);
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
    if (t == row0 || pos % kPlanPage == 0) {
      const int w = s_b[b] + j - cached / kPlanPage;
      const int some = min(kPlanPage - pos % kPlanPage, s_cu[b + 1] - t);
      *(int4*)(plan + p.writes + 4L * w) = make_int4(page, t, pos % kPlanPage, some);
    }
    return;
  }

  if (blockIdx.x == 0) {  // offsets, contexts and the short sequences' items
    unsigned long long pages = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = new_of(b), ctx = min(s_cached[b] + n, room);
      plan[p.cu + b] = s_cu[b];
      plan[p.ctx + b] = ctx;
      if (n > 0 && n * p.G <= kShortRows) pages += pages_of(ctx);
    }
    if (tid == 0) plan[p.cu + p.B] = total[0];
    if (pages) atomicAdd(&s_sum, pages);
    __syncthreads();
    // pages per item
    long pps = ((long)s_sum * p.Hkv + kShortTarget - 1) / kShortTarget;
    pps = max(pps, 1L) + kShortStep - 1;
    pps = p.short_whole ? kShortWhole : pps / kShortStep * kShortStep;
    auto splits = [&](int b) __attribute__((always_inline)) {
      const int n = new_of(b);
      return n > 0 && n * p.G <= kShortRows ? (int)((pages_of(min(s_cached[b] + n, room)) + pps - 1) / pps) : 0;
    };
    // Equal shares of a sequence's pages, each a multiple of what a workgroup takes at once; the sequences with the
    // largest ones first (94.8 against 98.5 us for 128 sequences of 512 to 8192 tokens in their own order).
    auto share = [&](int pages_b, int ns) __attribute__((always_inline)) {
      return (pages_b + ns * kShortStep - 1) / (ns * kShortStep) * kShortStep;
    };
    auto class_of = [&](int b, int ns) __attribute__((always_inline)) {
      return kClasses - 1 - (int)((long)share(pages_of(min(s_cached[b] + new_of(b), room)), ns) * kClasses / (pps + 1));
    };
    int at[2] = {0, 0}, all[2];  // items, sequences that are split
    s_class[tid] = 0;
    __syncthreads();
    for (int b = b0; b < b1; ++b) {
      const int ns = splits(b);
      at[0] += ns;
      at[1] += ns > 1;
      if (ns > 0) atomicAdd(&s_class[class_of(b, ns)], ns);
    }
    block_scan(at, all, s_wave);
    int items[1] = {s_class[tid]}, all_items[1];
    block_scan(items, all_items, s_wave);
    s_class[tid] = items[0];
    __syncthreads();
    for (int b = b0; b < b1; ++b) {
      const int ns = splits(b);
      s_a[b] = at[0];
      s_b[b] = ns > 0 ? atomicAdd(&s_class[class_of(b, ns)], ns) : 0;
      if (ns > 1) *(int4*)(plan + p.short_merges + 4L * at[1]) = make_int4(ns, s_b[b], s_cu[b], new_of(b));
      at[0] += ns;
      at[1] += ns > 1;
    }
    if (tid == 0) {
      s_a[p.B] = all[0];
      plan[PH_TOKENS] = total[0];
      plan[PH_SHORTS] = all[0];
      plan[PH_SHORT_MERGES] = all[1];
    }
    __syncthreads();
    for (int k = tid; k < all[0]; k += kThreads) {
      const int b = last_le(s_a, p.B, k);
      const int row0 = s_cu[b], n = s_cu[b + 1] - row0;
      const int pages_b = pages_of(min(s_cached[b] + n, room)), ns = s_a[b + 1] - s_a[b];
      const int step = share(pages_b, ns), i = k - s_a[b], page0 = i * step;
      int4* dst = (int4*)(plan + p.shorts + (long)PI_INTS * (s_b[b] + i));
      dst[0] = make_int4(b, row0, n, s_cached[b]);
      dst[1] = make_int4(page0, min(page0 + step, pages_b), ns, 0);
    }
    return;
  }

  // workgroup 1: the tiles
  int first[1] = {0}, tiles[1];
  {
    unsigned long long keys = 0;  // over all tiles
    int most = 0;
    for (int b = b0; b < b1; ++b) {
      const int c = s_cached[b], n = new_of(b);
      if (n * p.G > kShortRows) {
        const long nt = (n + p.tile_tok - 1) / p.tile_tok;
        first[0] += (int)nt;
        keys += nt * c + p.tile_tok * (nt * (nt - 1) / 2) + n;
        most = max(most, min(c + n, room));
      }
    }
    if (keys) {
      atomicAdd(&s_sum, keys);
      atomicMax(&s_most, most);
    }
  }
  s_class[tid] = 0;
  block_scan(first, tiles, s_wave);  // its barriers complete the sums, too
  for (int b = b0; b < b1; ++b) {
    s_a[b] = first[0];
    if (new_of(b) * p.G > kShortRows) first[0] += (new_of(b) + p.tile_tok - 1) / p.tile_tok;
  }
  __syncthreads();
  // keys that an item has at least
  long chunk = ((long)s_sum * p.Hkv + kTileTarget - 1) / kTileTarget;
  chunk = (long)tiles[0] * p.Hkv < kTileFew ? max(chunk, (long)kTileMinKeys) : 1L << 40;

  // Those with the most keys first, over all sequences: the launch drains on short ones (447 against 462 us for
  // seven prompts of 1 to 1500 tokens in sequence order).  A counting sort by 256 classes of keys; within a class the
  // order is the atomics', on which no result depends.
  struct Tile {
    int b, tok, count, pos, pages, step, ns, cls;  // step: pages per item
  };
  auto tile = [&](int k) __attribute__((always_inline)) {
    Tile x;
    x.b = last_le(s_a, p.B, k);
    const int row0 = s_cu[x.b], n = s_cu[x.b + 1] - row0, i = k - s_a[x.b];
    x.tok = row0 + i * p.tile_tok;
    x.count = min(p.tile_tok, n - i * p.tile_tok);
    x.pos = s_cached[x.b] + i * p.tile_tok;
    const int keys = min(x.pos + x.count, room);
    x.pages = pages_of(keys);
    const int ns = max(1, (int)(keys / chunk));
    x.step = (x.pages + kTilePages * ns - 1) / (kTilePages * ns) * kTilePages;
    x.ns = (x.pages + x.step - 1) / x.step;
    x.cls = kClasses - 1 - (int)((long)keys * kClasses / (s_most + 1));
    return x;
  };
  for (int k = tid; k < tiles[0]; k += kThreads) {
    const Tile x = tile(k);
    atomicAdd(&s_class[x.cls], x.ns);
  }
  __syncthreads();
  int items[1] = {s_class[tid]}, all_items[1];
  block_scan(items, all_items, s_wave);
  s_class[tid] = items[0];
  __syncthreads();
  for (int k = tid; k < tiles[0]; k += kThreads) {
    const Tile x = tile(k);
    const int item = atomicAdd(&s_class[x.cls], x.ns);
    if (x.ns > 1) *(int4*)(plan + p.tile_merges + 4L * atomicAdd(&s_merged, 1)) = make_int4(x.ns, item, x.tok, x.count);
    for (int s = 0; s < x.ns; ++s) {
      int4* dst = (int4*)(plan + p.tiles + (long)PI_INTS * (item + s));
      dst[0] = make_int4(x.b, x.tok, x.count, x.pos);
      dst[1] = make_int4(s * x.step, min((s + 1) * x.step, x.pages), x.ns, 0);
    }
  }
  __syncthreads();
  if (tid == 0) {
    plan[PH_TILES] = all_items[0];
    plan[PH_TILE_MERGES] = s_merged;
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
  const int blocks = (a.p.T + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(2 + (blocks < 1 ? 1 : blocks)), dim3(kThreads), 0, (hipStream_t)stream, a);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
