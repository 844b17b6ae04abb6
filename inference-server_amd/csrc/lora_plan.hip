// moe_mi355x_lora_plan: a step's rows sorted by their adapter, stably, and cut into tiles (lora.h), on the GPU from
// the adapters' numbers alone.
//
// A counting sort in one launch.  Each workgroup places 1024 rows; where they go it works out by itself, from
// counts over all rows (by sequence, where the numbers are the sequences').  Within a wave the rows of one adapter find each
// other by the bits of its number (9 ballots), so that the order does not depend on atomics.  Steps of some thousand rows are
// bound by latency: 4.2 us in a graph for 64 rows of 100 adapters, 4.4 for 9044 rows of 12 sequences, of which a launch
// is 1.7; the rest are four phases between barriers.
// By row every workgroup reads all T numbers, 1024 a turn, so its time goes with T: 1024 rows 4.5 us, 2048 5.6, 4096 7.3, 8192
// 10.6, 16384 17, 65536 57, 262144 216 (with 4 adapters or 100, shuffled or sorted).  By sequence it does not: 262144 rows
// of 64 sequences 5.4 us, of 4096 7.8, and 13.1 where all 4096 add to the count of one adapter.
#include "lora.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / MOE_WAVE;
constexpr int kBins = kLoraMaxAdapters + 1;  // the last one used: rows without an adapter
constexpr int kPerLane = (kBins + MOE_WAVE - 1) / MOE_WAVE;

struct LoraPlanArgs {
  const int32_t *ids, *cu;  // ids [seqs] with cu [seqs + 1], else [T]
  int seqs;
  int32_t* plan;
  LoraLayout p;
};

// The lanes whose bin is this one's, among those with `live`.
__device__ __forceinline__ uint64_t same_bin(int bin, bool live) {
  uint64_t same = __ballot(live);
#pragma unroll
  for (int bit = 0; bit < 9; ++bit) {
    const bool one = (bin >> bit) & 1;
    const uint64_t with = __ballot(one);
    same &= one ? with : ~with;
  }
  return same;
}

__global__ __launch_bounds__(kThreads) void lora_plan_kernel(LoraPlanArgs a) {
  __shared__ int s_cu[kLoraMaxSeqs + 1];
  __shared__ int s_total[kBins], s_before[kBins];  // rows of each adapter: all, and those in front of this workgroup's
  __shared__ int s_wave[kWaves][kBins];
  __shared__ int s_first[kBins + 1], s_tile[kBins + 1], s_pair[kBins + 1];
  const LoraLayout& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int T = p.T, L = p.L, bins = L + 1;
  const int row0 = blockIdx.x * kThreads, row = row0 + tid;
  auto bin_of = [&](int id) { return id >= 0 && id < L ? id : L; };

  for (int i = tid; i < bins; i += kThreads) s_total[i] = s_before[i] = 0;
  for (int i = tid; i < kWaves * kBins; i += kThreads) (&s_wave[0][0])[i] = 0;
  int bin = L;
  if (a.cu) {
    for (int i = tid; i <= a.seqs; i += kThreads) s_cu[i] = min(max(a.cu[i], 0), T);
    __syncthreads();
    for (int b = tid; b < a.seqs; b += kThreads) {
      const int lo = s_cu[b], n = s_cu[b + 1] - lo, front = min(s_cu[b + 1], row0) - lo;
      const int id = bin_of(a.ids[b]);
      if (n > 0) atomicAdd(&s_total[id], n);
      if (front > 0) atomicAdd(&s_before[id], front);
    }
    const int first = s_cu[0], end = s_cu[a.seqs];
    if (tid == 0) {  // in front of the first sequence and behind the last
      atomicAdd(&s_total[L], first + max(T - max(first, end), 0));
      atomicAdd(&s_before[L], min(row0, first) + max(row0 - max(first, end), 0));
    }
    if (row >= first && row < end) {
      int lo = 0, hi = a.seqs - 1;  // the first sequence that ends behind the row
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (s_cu[mid + 1] > row) hi = mid;
        else lo = mid + 1;
      }
      bin = bin_of(a.ids[lo]);
    }
  } else {
    __syncthreads();
    for (int i0 = 0; i0 < T; i0 += kThreads) {
      const int i = i0 + tid;
      const bool live = i < T;
      const int id = live ? bin_of(a.ids[i]) : L;
      if (i0 == row0) bin = id;
      const uint64_t same = same_bin(id, live);
      if (live && (same & lanemask_lt()) == 0) {
        atomicAdd(&s_total[id], __popcll(same));
        if (i0 < row0) atomicAdd(&s_before[id], __popcll(same));
      }
    }
  }
  const bool live = row < T;
  const uint64_t same = same_bin(bin, live);
  const int in_wave = __popcll(same & lanemask_lt());
  if (live && in_wave == 0) s_wave[wave][bin] = __popcll(same);
  __syncthreads();

  if (wave == 0) {  // where each adapter's rows and tiles begin
    int n[kPerLane], rows = 0, tiles = 0, pairs = 0;
    auto of = [&](int i, int height) { return lane * kPerLane + i < L ? (n[i] + height - 1) / height : 0; };
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int b = lane * kPerLane + i;
      n[i] = b < bins ? s_total[b] : 0;
      rows += n[i], tiles += of(i, kLoraRows), pairs += of(i, kLoraPair);
    }
    int rows_to = rows, tiles_to = tiles, pairs_to = pairs;
#pragma unroll
    for (int d = 1; d < MOE_WAVE; d *= 2) {
      const int r = __shfl_up(rows_to, d), s = __shfl_up(tiles_to, d), q = __shfl_up(pairs_to, d);
      if (lane >= d) rows_to += r, tiles_to += s, pairs_to += q;
    }
    rows_to -= rows, tiles_to -= tiles, pairs_to -= pairs;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int b = lane * kPerLane + i;
      if (b <= bins) s_first[b] = rows_to, s_tile[b] = tiles_to, s_pair[b] = pairs_to;
      rows_to += n[i], tiles_to += of(i, kLoraRows), pairs_to += of(i, kLoraPair);
    }
  }
  __syncthreads();
  if (live) {
    int at = s_before[bin] + in_wave;  // among its adapter's rows
#pragma unroll
    for (int w = 0; w < kWaves; ++w) at += w < wave ? s_wave[w][bin] : 0;
    const int to = s_first[bin] + at;
    if (to < T) a.plan[p.rows + to] = row;
    // the row that begins a tile writes its record
    auto record = [&](const int* from, int height, int room, long list) {
      const int tile = from[bin] + at / height;
      if (at % height == 0 && tile < room)
        *(int4*)(a.plan + list + 4L * tile) = make_int4(bin, to, min(s_total[bin] - at, height), 0);
    };
    if (bin < L) {
      record(s_tile, kLoraRows, p.N, p.tiles);
      if (p.M > 0) record(s_pair, kLoraPair, p.M, p.pairs);
    }
  }
  if (blockIdx.x == 0) {
    for (int i = tid; i <= bins; i += kThreads) a.plan[p.offsets + i] = s_first[i];
    if (tid == 0) a.plan[LH_TILES] = s_tile[L], a.plan[LH_PAIRS] = s_pair[L];
  }
}

}  // namespace

extern "C" size_t moe_mi355x_lora_plan_bytes(int T, int L, int32_t* offsets) {
  if (!lora_plan_ok(T, L)) return 0;
  const LoraLayout p = lora_layout(T, L);
  if (offsets) offsets[0] = (int32_t)p.offsets, offsets[1] = (int32_t)p.rows;
  return (size_t)p.ints * 4;
}

extern "C" int moe_mi355x_lora_plan(const int32_t* adapter_ids, const int32_t* cu_rows, int seqs, int T, int L,
                                    void* plan, size_t plan_bytes, void* stream) {
  MOE_RETURN_IF(!lora_plan_ok(T, L), MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(cu_rows && (seqs < 0 || seqs > kLoraMaxSeqs), MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(!adapter_ids && (cu_rows ? seqs : T) > 0, MOE_ERR_INVALID_ARG);
  LoraPlanArgs a{adapter_ids, cu_rows, seqs, (int32_t*)plan, lora_layout(T, L)};
  MOE_RETURN_IF(!plan || plan_bytes < (size_t)a.p.ints * 4, MOE_ERR_WORKSPACE);
  MOE_RETURN_IF(!moe_aligned16(plan), MOE_ERR_ALIGNMENT);
  hipLaunchKernelGGL(lora_plan_kernel, dim3(T > kThreads ? (T + kThreads - 1) / kThreads : 1), dim3(kThreads), 0,
                     (hipStream_t)stream, a);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
