// What the adapters of a step's rows add to a shared projection: for row t with adapter l, column n in part p of the
// projection (q, k and v are parts of one), r < rank_l,
//   u[t, p, r] = scale_l sum_k x[t, k] A_l[p R + r, k]          y[t, n] = bf16( y[t, n] + sum_r u[t, p, r] B_l[n, r] )
// with fp32 sums and one rounding, of y.  Bound by bytes: x, y and the adapters in use once each.  Consecutive lanes read
// consecutive bytes everywhere, MFMA operands go through LDS, and no branch lies around a load, for the compiler waits
// where it joins.  (4642 rows beside q/k/v, 2048 to 5120, ranks up to 64: 49 us with operands straight from memory, a lane a
// row; 45 through LDS; 39 without the branches, 33.5 now: 117 MB at 3.5 TB/s, u's launch 12 us and the columns' 20.8.)
//
// Two forms over the plan's tiles (rows of one adapter, lora.h):
//   few rows (tiles of 2): one launch, a workgroup per (tile, run of columns), which forms the u of its part by
//     itself; dot products over the lanes, no MFMA;
//   many (tiles of 64): u of every (tile, part, share of K) to the workspace in fp32, then the columns, both on MFMAs.
//     For the second product u is split in two bf16 values, u = hi + lo to 2^-17 of it.
#include "lora.h"

namespace {

constexpr int kGroup = 16;     // ranks of an MFMA operand
constexpr int kMaxRank = 128;
constexpr int kMaxParts = 4;

struct LoraArgs {
  uint16_t* y;        // [T][N], rows y_stride values apart
  const uint16_t* x;  // [T][K], rows x_stride values apart
  long y_stride, x_stride;
  const uint16_t *a, *b;  // [L][P R][K], [L][N][R]
  const int32_t* ranks;   // [L]
  const float* scales;    // [L]
  const int32_t* plan;
  float* u;               // before the scale; [shares][T][P][R], rows in the plan's order
  LoraLayout p;
  int K, R, N, parts, shares, chunk, runs;  // chunk: columns of a workgroup, in one part; runs: of them in all parts
  int col[kMaxParts + 1];             // where the parts begin
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}
__device__ __forceinline__ float lo_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The first `live` of 8 values: ranks that the adapter has
__device__ __forceinline__ uint4 mask8(uint4 v, int live) {
  auto keep = [&](uint32_t w, int i) __attribute__((always_inline)) {
    return live >= i + 2 ? w : live == i + 1 ? w & 0xffffu : 0u;
  };
  return make_uint4(keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6));
}

// A workgroup's tile.  What the plan says is kept within the step and the pool, whatever it holds (behind its last tile,
// anything), so that the rows and the adapter can be asked for before it is known whether there is work: `n` > 0.
struct Tile {
  int l, first, n, rank;  // adapter, first entry of the sorted rows, rows, rank

  // tile `tile` of the plan's list of kRows ones
  template <int kRows>
  __device__ __forceinline__ static Tile of(const LoraArgs& a, int tile) {
    constexpr bool pair = kRows == kLoraPair;
    const int room = pair ? a.p.M : a.p.N;
    const int4 e = *(const int4*)(a.plan + (pair ? a.p.pairs : a.p.tiles) + 4L * min(tile, room - 1));
    const int tiles = min(a.plan[pair ? LH_PAIRS : LH_TILES], room);
    Tile t;
    t.l = min(max(__builtin_amdgcn_readfirstlane(e.x), 0), a.p.L - 1);
    t.first = min(max(__builtin_amdgcn_readfirstlane(e.y), 0), a.p.T - 1);
    t.rank = min(a.ranks[t.l], a.R);
    const int rows = min(min(__builtin_amdgcn_readfirstlane(e.z), kRows), a.p.T - t.first);
    t.n = tile < tiles && t.rank > 0 ? rows : 0;
    t.last = max(rows, 1) - 1;
    return t;
  }
  __device__ __forceinline__ int row(const LoraArgs& a, int i) const {  // of entry first + i, or of the last one
    return min(max(a.plan[a.p.rows + first + min(i, last)], 0), a.p.T - 1);
  }
  __device__ __forceinline__ bool narrow() const { return last < 16; }

 private:
  int last;
};

// Workgroups that follow each other go to different XCDs (8): those of one tile, which share its rows of x and its
// adapter, are 8 apart, so that they find them in one L2.
__device__ __forceinline__ int tile_of(int per_tile) { return blockIdx.x / 8 / per_tile * 8 + blockIdx.x % 8; }
__device__ __forceinline__ int turn_of(int per_tile) { return blockIdx.x / 8 % per_tile; }
unsigned lora_grid(int tiles, int per_tile) { return (unsigned)((tiles + 7) / 8 * 8 * per_tile); }

// The part and the columns of run `run` (every part has its own runs)
__device__ __forceinline__ void run_of(const LoraArgs& a, int run, int* part, int* c0, int* c1) {
  int p = 0, c = run * a.chunk;
  for (;;) {
    const int n = a.col[p + 1] - a.col[p], runs = (n + a.chunk - 1) / a.chunk * a.chunk;
    if (c < runs) break;
    c -= runs;
    ++p;
  }
  *part = p;
  *c0 = c + a.col[p];
  *c1 = min(*c0 + a.chunk, a.col[p + 1]);
}

// fn of the number of 16-rank groups that `rank` takes, 1, 2, 4 or 8 (RG at most), as a constant
template <int RG, typename F>
__device__ __forceinline__ void by_groups(int rank, F fn) {
  if (RG == 1 || rank <= 16) return fn(std::integral_constant<int, 1>());
  if constexpr (RG >= 2)
    if (RG == 2 || rank <= 32) return fn(std::integral_constant<int, 2>());
  if constexpr (RG >= 4)
    if (RG == 4 || rank <= 64) return fn(std::integral_constant<int, 4>());
  if constexpr (RG >= 8) return fn(std::integral_constant<int, 8>());
}

// ---------------------------------------------------------------------------
// few rows.  u: a wave takes every eighth rank, its lanes 8 values of a row each; the sums over the lanes go to LDS.
// Columns: kLanes lanes have 8 ranks of a column each, a wave 64 columns at a time; over kLanes turns lane i
// ends with the sum of column i.  Bound by latency and, at ranks of 64, by the rate at which a CU takes A in (about 50 bytes a
// clock): 4.1 us for one row of rank 16, 4096 to 2048; 13.4 for 128 rows of 100 adapters, 4096 to 9216, 45 MB at 3.3 TB/s.
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;
constexpr int kFewRows = kLoraPair;

__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, a), __builtin_bit_cast(v2bf, b), c, false);
}
__device__ __forceinline__ float dot8(v4i a, v4i b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = dot2((uint32_t)a[i], (uint32_t)b[i], c);
  return c;
}

// Sum over kLanes adjacent lanes
template <int CTRL>
__device__ __forceinline__ float dpp_add(float s) {
  return s + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(s), CTRL, 0xf, 0xf, false));
}
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float s) {
  s = dpp_add<0xb1>(s);                              // of a pair
  if constexpr (kLanes >= 4) s = dpp_add<0x4e>(s);   // of 4: the other pair
  if constexpr (kLanes >= 8) s = dpp_add<0x141>(s);  // of 8, mirrored
  if constexpr (kLanes >= 16) s = dpp_add<0x140>(s);  // of 16, mirrored
  return s;
}

// 64 columns' operands: lane's 8 ranks of kLanes columns, and its own column of each row
template <int NR, int kLanes>
struct FewColumns {
  v4i b[kLanes];
  uint16_t y[NR];

  __device__ __forceinline__ void load(const LoraArgs& a, const Tile& t, const int (&row)[NR], int c, int end, int lane) {
    const int sub = lane % kLanes, group = lane / kLanes * kLanes;
    const uint16_t* src = a.b + (long)t.l * a.N * a.R + (8 * sub < t.rank ? 8 * sub : 0);
#pragma unroll
    for (int i = 0; i < kLanes; ++i) b[i] = *(const v4i*)(src + (long)min(c + group + i, end - 1) * a.R);
#pragma unroll
    for (int r = 0; r < NR; ++r) y[r] = a.y[row[r] * a.y_stride + min(c + lane, end - 1)];
  }
  // mask: of the lane's 8 ranks those that the adapter has
  __device__ __forceinline__ void add(const LoraArgs& a, const Tile& t, const int (&row)[NR], int c, int end, int lane, uint4 mask,
                                      const float (&u)[NR][8]) {
    const int sub = lane % kLanes;
    float sum[NR];
#pragma unroll
    for (int i = 0; i < kLanes; ++i) {
      const uint32_t w[4] = {(uint32_t)b[i][0] & mask.x, (uint32_t)b[i][1] & mask.y, (uint32_t)b[i][2] & mask.z,
                             (uint32_t)b[i][3] & mask.w};
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(hi_of(w[e]), u[r][2 * e + 1], fmaf(lo_of(w[e]), u[r][2 * e], s));
        s = lanes_sum<kLanes>(s);
        sum[r] = i == 0 || sub == i ? s : sum[r];
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r)
      if (r < t.n && c + lane < end) a.y[row[r] * a.y_stride + c + lane] = f32_to_bf16(bf16_to_f32(y[r]) + sum[r]);
  }
};

// kLanes: of a column; 8 kLanes ranks at most, kLanes of them a wave's
template <int NR, int kLanes>
__device__ __forceinline__ void few_rows(const LoraArgs& a, const Tile& t, const int (&rows)[kFewRows], int part, int c0, int c1,
                                         int lane, int wave, float (&s_u)[kFewRows][8 * kLanes]) {
  int row[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) row[r] = rows[r];
  const float scale = a.scales[t.l];
  // a wave's columns side by side; the first 64 on their way before u
  const int per = (c1 - c0 + 64 * kFewWaves - 1) / (64 * kFewWaves) * 64, end = min(c0 + (wave + 1) * per, c1);
  int c = c0 + wave * per;
  constexpr bool kEarly = NR * kLanes <= 16;  // where there are registers for them
  FewColumns<NR, kLanes> now;
  if (kEarly && c < end) now.load(a, t, row, c, end, lane);

  float acc[kLanes][NR];
#pragma unroll
  for (int i = 0; i < kLanes; ++i)
#pragma unroll
    for (int r = 0; r < NR; ++r) acc[i][r] = 0.f;
  // kTogether ranks by kBlock times 512 values are in flight together.  (Four ranks, or twice the values, take registers that
  // another workgroup of the CU misses: 24 rows of up to 64 ranks beside q/k/v 11.0 us with two, 11.3 with four.)
  constexpr int kTogether = 2, kBlock = 4;
  const uint16_t* ap = a.a + ((long)t.l * a.parts + part) * a.R * a.K;
  // No branch around a load: the compiler waits where it joins.  Behind K (`whole` is false) both operands are zeros.
  auto block = [&](int k0, auto whole) __attribute__((always_inline)) {
    auto load = [&](const uint16_t* row, int j) __attribute__((always_inline)) {
      const int k = k0 + 512 * j + 8 * lane;
      if (whole) return *(const v4i*)(row + k);
      const v4i v = *(const v4i*)(row + min(k, a.K - 8));
      const int keep = k < a.K ? -1 : 0;
      return (v4i){v[0] & keep, v[1] & keep, v[2] & keep, v[3] & keep};
    };
    v4i xv[kBlock][NR];
#pragma unroll
    for (int j = 0; j < kBlock; ++j)
#pragma unroll
      for (int r = 0; r < NR; ++r) xv[j][r] = load(a.x + row[r] * a.x_stride, j);
#pragma unroll
    for (int i0 = 0; i0 < kLanes; i0 += kTogether) {
      if (wave + kFewWaves * i0 < t.rank) {
        v4i av[kTogether][kBlock];
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
#pragma unroll
          for (int j = 0; j < kBlock; ++j) av[i][j] = load(ap + (long)min(wave + kFewWaves * (i0 + i), t.rank - 1) * a.K, j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
#pragma unroll
          for (int j = 0; j < kBlock; ++j)
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[i0 + i][r] = dot8(av[i][j], xv[j][r], acc[i0 + i][r]);
      }
    }
  };
  int k0 = 0;
  for (; k0 + 512 * kBlock <= a.K; k0 += 512 * kBlock) block(k0, std::true_type());
  if (k0 < a.K) block(k0, std::false_type());
#pragma unroll
  for (int i = 0; i < kLanes; ++i) {
    const int rank = wave + kFewWaves * i;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float s = rank < t.rank ? wave_sum_uniform(acc[i][r]) * scale : 0.f;
      if (lane == 0) s_u[r][rank] = s;
    }
  }
  __syncthreads();
  float u[NR][8];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const v4f lo = *(const v4f*)&s_u[r][8 * (lane % kLanes)], hi = *(const v4f*)&s_u[r][8 * (lane % kLanes) + 4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[r][e] = lo[e], u[r][4 + e] = hi[e];
  }
  const uint4 mask = mask8(make_uint4(~0u, ~0u, ~0u, ~0u), t.rank - 8 * (lane % kLanes));
  for (; c < end; c += 64) {
    if constexpr (kEarly) {
      FewColumns<NR, kLanes> next;
      if (c + 64 < end) next.load(a, t, row, c + 64, end, lane);
      __builtin_amdgcn_sched_barrier(0);
      now.add(a, t, row, c, end, lane, mask, u);
      now = next;
    } else {
      now.load(a, t, row, c, end, lane);
      now.add(a, t, row, c, end, lane, mask, u);
    }
  }
}

template <int kLanes>
__global__ __launch_bounds__(kFewThreads) void lora_few_kernel(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) float s_u[kFewRows][8 * kLanes];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile t = Tile::of<kLoraPair>(a, tile_of(a.runs));
  int row[kFewRows];
#pragma unroll
  for (int r = 0; r < kFewRows; ++r) row[r] = __builtin_amdgcn_readfirstlane(t.row(a, r));
  int part, c0, c1;
  run_of(a, turn_of(a.runs), &part, &c0, &c1);
  if (t.n <= 0) return;
  if (t.n == 1)
    few_rows<1, kLanes>(a, t, row, part, c0, c1, lane, wave, s_u);
  else
    few_rows<kFewRows, kLanes>(a, t, row, part, c0, c1, lane, wave, s_u);
}

// ---------------------------------------------------------------------------
// many rows: u.  64 rows by up to 64 ranks, 128 k at a time through LDS, of which each of the 4 waves multiplies 32; the
// next 3 times 128 are on their way meanwhile.  In LDS a row has 16 pieces of 8 values, piece c at c ^ (row % 16), so that
// the 16 rows of an operand lie in different banks.  (4078 rows of K 8192, rank 32: 20 us, of which 10.5 stream x at 6.3 TB/s;
// the launch, the plan's tile, its rows and then their first values, in turn, are most of the rest.)
// ---------------------------------------------------------------------------
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRowsM = kLoraRows, kMT = kRowsM / 16;
constexpr int kSlice = 128;
constexpr int kRanksM = 64;  // of a workgroup

template <int NG>
struct ShrinkLds {
  union {
    struct {
      v4i a[16 * NG][16], x[kRowsM][16];
    } slice[2];
    v4f part[kWaves][kMT][NG][64];
  };
};

template <int MT, int NG, int RG>
__device__ __forceinline__ void shrink(const LoraArgs& a, const Tile& t, const uint16_t* const (&xr)[kMT], int part, int rank0,
                                       int s0, int s1, int share, int lane, int wave, ShrinkLds<RG>& lds) {
  const int lr = lane & 15, lg = lane >> 4;
  const int q = threadIdx.x >> 4, piece = threadIdx.x & 15, to = piece ^ (q & 15);  // rows q + 16 i of both
  const uint16_t* ar[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) ar[i] = a.a + (((long)t.l * a.parts + part) * a.R + min(rank0 + q + 16 * i, t.rank - 1)) * a.K;
  struct Slice {
    v4i a[NG], x[MT];
  } r0, r1, r2, r3;
  // No branch around a load: the compiler waits where it joins.  Rows and ranks that there are not repeat the last one, and
  // are not stored; k behind K repeat the last 8, and are not multiplied.
  auto load = [&](int s, Slice& into) __attribute__((always_inline)) {
    const int k = min(kSlice * min(s, s1 - 1) + 8 * piece, a.K - 8);
#pragma unroll
    for (int i = 0; i < MT; ++i) into.x[i] = *(const v4i*)(xr[i] + k);
#pragma unroll
    for (int i = 0; i < NG; ++i) into.a[i] = *(const v4i*)(ar[i] + k);
  };
  auto store = [&](int buf, const Slice& from) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NG; ++i) lds.slice[buf].a[q + 16 * i][to] = from.a[i];
#pragma unroll
    for (int i = 0; i < MT; ++i) lds.slice[buf].x[q + 16 * i][to] = from.x[i];
  };
  v4f u[MT][NG];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int g = 0; g < NG; ++g) u[m][g] = (v4f){0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int buf) __attribute__((always_inline)) {
    const int at = (4 * wave + lg) ^ lr;
    v8bf xf[MT], af[NG];
#pragma unroll
    for (int m = 0; m < MT; ++m) xf[m] = __builtin_bit_cast(v8bf, lds.slice[buf].x[16 * m + lr][at]);
#pragma unroll
    for (int g = 0; g < NG; ++g) af[g] = __builtin_bit_cast(v8bf, lds.slice[buf].a[16 * g + lr][at]);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g < NG; ++g) u[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[g], xf[m], u[m][g], 0, 0, 0);
  };
  // slice s + 4 is loaded while slice s is multiplied, and goes to LDS during slice s + 3
  auto turn = [&](int s, int buf, Slice& mine, Slice& after) __attribute__((always_inline)) {
    if (s + 4 < s1) load(s + 4, mine);  // these registers went to LDS in the last turn
    __builtin_amdgcn_sched_barrier(0);
    if (kSlice * s + 32 * wave < a.K) multiply(buf);
    if (s + 1 < s1) store(buf ^ 1, after);  // last read a slice ago, before the last barrier
    __syncthreads();
  };
  load(s0, r0);
  load(s0 + 1, r1);
  load(s0 + 2, r2);
  load(s0 + 3, r3);
  store(0, r0);
  __syncthreads();
  for (int s = s0; s < s1; s += 4) {
    turn(s, 0, r0, r1);
    if (s + 1 >= s1) break;
    turn(s + 1, 1, r1, r2);
    if (s + 2 >= s1) break;
    turn(s + 2, 0, r2, r3);
    if (s + 3 >= s1) break;
    turn(s + 3, 1, r3, r0);
  }
  // lane l has ranks 4 (l / 16) + i of row l % 16 of each: joined over the waves
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int g = 0; g < NG; ++g) lds.part[wave][m][g][lane] = u[m][g];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * NG * 64; i += kThreads) {
    const int m = i / (64 * NG), g = i / 64 % NG, row = 16 * m + i % 16, rank = rank0 + kGroup * g + 4 * (i % 64 / 16);
    v4f sum = lds.part[0][m][g][i % 64];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += lds.part[w][m][g][i % 64];
    if (row < t.n && rank < a.R) *(v4f*)(a.u + (((long)share * a.p.T + t.first + row) * a.parts + part) * a.R + rank) = sum;
  }
}

template <int RG>
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) ShrinkLds<RG> lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = a.parts * a.shares * ((a.R + kRanksM - 1) / kRanksM), at = turn_of(blocks);
  const Tile t = Tile::of<kLoraRows>(a, tile_of(blocks));
  const uint16_t* xr[kMT];
#pragma unroll
  for (int i = 0; i < kMT; ++i) xr[i] = a.x + t.row(a, threadIdx.x / 16 + 16 * i) * a.x_stride;
  if (t.n <= 0) return;
  const int part = at % a.parts, share = at / a.parts % a.shares, rank0 = at / a.parts / a.shares * kRanksM;
  if (rank0 >= t.rank) return;
  const int slices = (a.K + kSlice - 1) / kSlice, per = (slices + a.shares - 1) / a.shares;
  const int s0 = min(share * per, slices), s1 = min(s0 + per, slices);
  by_groups<RG>(t.rank - rank0, [&](auto groups) __attribute__((always_inline)) {
    constexpr int NG = decltype(groups)::value;
    if (t.narrow())
      shrink<1, NG, RG>(a, t, xr, part, rank0, s0, s1, share, lane, wave, lds);
    else
      shrink<kMT, NG, RG>(a, t, xr, part, rank0, s0, s1, share, lane, wave, lds);
  });
}

// ---------------------------------------------------------------------------
// many rows: columns.  A wave has 16 of the 64 rows, all of them 128 columns of B at a time, through LDS.  Lane l has 8
// columns in a row, from 8 (l % 16), of rows 4 (l / 16) + i: column 8 (l % 16) + j is column l % 16 of product j,
// and B's columns lie in LDS in that order.  (4642 rows, 2048 to 5120, ranks up to 64: 20.8 us, y read and written at 4.6 TB/s.)
// ---------------------------------------------------------------------------
constexpr int kPiece = 128;

// 8 values of B, infinite ones as zeros
__device__ __forceinline__ v8bf finite8(v8bf b) {
  const v4i w = __builtin_bit_cast(v4i, b);
  v4i keep;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    keep[i] = ((w[i] & 0x7fff) == 0x7f80 ? 0 : w[i] & 0xffff) | ((w[i] & 0x7fff0000) == 0x7f800000 ? 0 : w[i] & (int)0xffff0000);
  return __builtin_bit_cast(v8bf, keep);
}

// 4 ranks' u as they enter the product.  A finite one past bf16's largest value is that and a rest, not an infinity.
__device__ __forceinline__ void split_u(v4f s, float scale, int live, uint2* hi, uint2* lo) {
  constexpr float kMost = 0x1.fep127f;
  float v[4], rest[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float u = e < live ? s[e] * scale : 0.f;
    const bool finite = fabsf(u) < INFINITY;
    v[e] = finite ? __builtin_amdgcn_fmed3f(round_bf16(u), -kMost, kMost) : u;
    rest[e] = finite ? u - v[e] : 0.f;  // not inf - inf
  }
  *hi = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  *lo = make_uint2(pack2(rest[0], rest[1]), pack2(rest[2], rest[3]));
}

template <int NG>
struct ExpandLds {
  static constexpr int kRow = 32 * NG + 16;  // bytes of a column, 16 of them so that 8 columns' banks differ
  uint16_t u[kRowsM][2][16 * NG + 8];        // hi, lo
  uint8_t b[kPiece * kRow];
};

template <int J, int NG>
__device__ __forceinline__ void expand(const LoraArgs& a, const Tile& t, uint16_t* const (&yr)[4], int part, int c0, int c1,
                                       int lane, int wave, ExpandLds<NG>& lds) {
  constexpr int kRow = ExpandLds<NG>::kRow, kRows = J == 8 ? kRowsM : 16;
  constexpr int kY = J / 2;  // 32-bit words of a row's columns
  const int lr = lane & 15, lg = lane >> 4;
  const int row0 = J == 8 ? 16 * wave : 0, tile0 = J == 8 ? 0 : J * wave, mine = J * lr + 16 * tile0;  // of the piece
  const float scale = a.scales[t.l];
  const uint16_t* bl = a.b + (long)t.l * a.N * a.R;
  // No branch around a load: columns behind the run repeat its last ones, and are not stored
  typedef uint32_t Words __attribute__((ext_vector_type(kY)));
  v4i bv[NG];
  Words yv[4];
  auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) yv[i] = *(const Words*)(yr[i] + min(c + mine, c1 - J));
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int at = threadIdx.x + kThreads * i, n = at / (2 * NG), r = at % (2 * NG) * 8;
      bv[i] = *(const v4i*)(bl + (long)min(c + n, c1 - 1) * a.R + (r < t.rank ? r : 0));
    }
  };
  auto store_b = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int at = threadIdx.x + kThreads * i, n = at / (2 * NG), r = at % (2 * NG) * 8;
      const uint4 v = mask8(__builtin_bit_cast(uint4, bv[i]), t.rank - r);
      *(uint4*)(lds.b + ((n / (16 * J) * J + n % J) * 16 + n % (16 * J) / J) * kRow + 2 * r) = v;
    }
  };
  load(c0);
  // u: the shares' sums, some shares of all this thread's values in flight together
  constexpr int kMine = (kRows * NG * 4 + kThreads - 1) / kThreads, kShares = kMine >= 8 ? 1 : kMine >= 4 ? 2 : 4;
  v4f su[kMine];
  const float* src[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = threadIdx.x + kThreads * i, r0 = 4 * (at % (NG * 4));
    src[i] = a.u + (((long)t.first + min(at / (NG * 4), t.n - 1)) * a.parts + part) * a.R + (r0 < t.rank ? r0 : 0);
    su[i] = (v4f){0.f, 0.f, 0.f, 0.f};
  }
  const long share = (long)a.p.T * a.parts * a.R;
  for (int z = 0; z < a.shares; z += kShares) {
    v4f v[kShares][kMine];
#pragma unroll
    for (int e = 0; e < kShares; ++e)
#pragma unroll
      for (int i = 0; i < kMine; ++i) v[e][i] = *(const v4f*)(src[i] + min(z + e, a.shares - 1) * share);
#pragma unroll
    for (int e = 0; e < kShares; ++e)
#pragma unroll
      for (int i = 0; i < kMine; ++i) su[i] += z + e < a.shares ? v[e][i] : (v4f){0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int at = threadIdx.x + kThreads * i, row = at / (NG * 4), r0 = 4 * (at % (NG * 4));
    if (row < kRows) split_u(su[i], scale, t.rank - r0, (uint2*)&lds.u[row][0][r0], (uint2*)&lds.u[row][1][r0]);
  }
  store_b();
  __syncthreads();
  // 16 ranks: hi and lo fill the 32 of one MFMA, against B twice; more: 32 ranks of hi, then of lo
  constexpr int kSteps = NG == 1 ? 1 : NG / 2;
  v8bf uv[kSteps][2];
#pragma unroll
  for (int g = 0; g < kSteps; ++g)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      uv[g][h] = NG == 1 ? *(const v8bf*)&lds.u[row0 + lr][lg >> 1][8 * (lg & 1)] : *(const v8bf*)&lds.u[row0 + lr][h][32 * g + 8 * lg];
  v4f acc[J];
  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j][i] = j % 2 ? hi_of(yv[i][j / 2]) : lo_of(yv[i][j / 2]);
  };
  auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int g = 0; g < kSteps; ++g) {
        const v8bf b = *(const v8bf*)(lds.b + (16 * (tile0 + j) + lr) * kRow + (NG == 1 ? 16 * (lg & 1) : 64 * g + 16 * lg));
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(uv[g][0], b, acc[j], 0, 0, 0);
        if (NG > 1) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(uv[g][1], b, acc[j], 0, 0, 0);
      }
  };
  auto store_y = [&](int c, auto check) __attribute__((always_inline)) {
    Words out[4];
    float odd = 0.f;  // NaN where something is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < kY; ++w) {
        out[i][w] = pack2(acc[2 * w][i], acc[2 * w + 1][i]);
        if (check) odd = dot2(out[i][w], 0, odd);
      }
    if (check && __any(odd != 0.f)) return false;
    if (c + mine < c1)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row0 + 4 * lg + i < t.n) *(Words*)(yr[i] + c + mine) = out[i];
    return true;
  };
  // The last piece apart, so that no branch lies around a load, and y's stores behind B's: a wait for a load waits for
  // every store in front of it.
  uint32_t left = 0;  // pieces that were not stored
  int c = c0;
  for (; c + kPiece < c1; c += kPiece) {
    begin();
    load(c + kPiece);
    __builtin_amdgcn_sched_barrier(0);
    multiply();
    __syncthreads();  // B's columns are read
    store_b();
    left |= store_y(c, std::true_type()) ? 0u : 1u << (c - c0) / kPiece;
    __syncthreads();
  }
  begin();
  multiply();
  left |= store_y(c, std::true_type()) ? 0u : 1u << (c - c0) / kPiece;
  // An infinite value of B makes NaN of lo's zeros, and of a lo of the other sign than hi.  Pieces with something that is not
  // finite once more, hi with B and lo with what is finite of it, from memory: each wave for itself.
  while (__builtin_expect(left != 0, 0)) {
    c = c0 + kPiece * __builtin_ctz(left);
    left &= left - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) yv[i] = *(const Words*)(yr[i] + min(c + mine, c1 - J));
    begin();
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int g = 0; g < kSteps; ++g) {
        const int r = NG == 1 ? 8 * (lg & 1) : 32 * g + 8 * lg;
        const uint4 w = mask8(*(const uint4*)(bl + (long)min(c + mine + j, c1 - 1) * a.R + (r < t.rank ? r : 0)), t.rank - r);
        const v8bf b = __builtin_bit_cast(v8bf, w), rest = finite8(b);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(uv[g][0], NG == 1 && lg >= 2 ? rest : b, acc[j], 0, 0, 0);
        if (NG > 1) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(uv[g][1], rest, acc[j], 0, 0, 0);
      }
    store_y(c, std::false_type());
  }
}

template <int RG>
__global__ __launch_bounds__(kThreads, RG <= 4 ? 4 : 2) void lora_expand_kernel(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[sizeof(ExpandLds<RG>)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Tile t = Tile::of<kLoraRows>(a, tile_of(a.runs));
  uint16_t* yr[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) yr[i] = a.y + t.row(a, (t.narrow() ? 0 : 16 * wave) + 4 * (lane >> 4) + i) * a.y_stride;
  int part, c0, c1;
  run_of(a, turn_of(a.runs), &part, &c0, &c1);
  if (t.n <= 0) return;
  by_groups<RG>(t.rank, [&](auto groups) __attribute__((always_inline)) {
    constexpr int NG = decltype(groups)::value;
    if (t.narrow())
      expand<2, NG>(a, t, yr, part, c0, c1, lane, wave, *(ExpandLds<NG>*)lds);
    else
      expand<8, NG>(a, t, yr, part, c0, c1, lane, wave, *(ExpandLds<NG>*)lds);
  });
}

bool lora_ok(int T, int L, int K, int R, int parts) {
  return lora_plan_ok(T, L) && K > 0 && K % 32 == 0 && K <= (1 << 24) && R > 0 && R % kGroup == 0 && R <= kMaxRank && parts >= 1 &&
         parts <= kMaxParts;
}

// How a call is cut up.
// Few rows: every run of columns of each pair of rows reads the part's A for itself, which one CU takes 1.2 us for 64 KB
// to do, so this pays where rank times K is small, and for the fewer rows the larger it is.  By the pool's rank: what its
// adapters' are is known on the GPU alone.  (us in a graph, few / many rows' form, "rows/adapters", as many rows for each adapter, of the
// pool's rank.  2048 to q/k/v 5120, rank 16: 1/1 3.8 / 5.6, 32/32 5.5 / 9.1, 128/64 8.5 / 11.9, 256/64 12.0 / 12.2; rank 32: 1/1
// 4.4 / 6.4, 64/64 11.8 / 15.7, 128/64 12.3 / 15.9, 192/64 17.6 / 16.0; rank 64: 1/1 7.1 / 7.8, 8/8 8.0 / 8.4, 32/32 13.8 / 13.9, 48/48
// 15.3 / 18.5, 64/64 22.5 / 22.5, 192/64 30.8 / 23.5; rank 128: 1/1 11.5 / 10.0, 16/16 14.5 / 16.2, 32/32 30.2 / 25.5.  4096 to 9216,
// rank 16: 128/64 13.1 / 17.6, 192/64 20.5 / 18.0.  4096 to 2048, rank 64: 1/1 7.8 / 6.9, 32/32 11.1 / 11.5, 64/64 12.7 / 15.1,
// 256/64 24.4 / 15.6.  8192 to 4096, rank 16: 32/32 7.2 / 10.0, 64/64 10.6 / 12.9, 192/64 15.3 / 13.3.)
// The rule sees neither the runs of columns nor how many rows share an adapter, and in between it gives up some us: it takes the
// form of many rows for 48/48 of rank 64 and 16/16 of rank 128 beside q/k/v, and for 48/48 to 64/64 of the last two projections.
constexpr long kFewAdapter = 1 << 17, kFewRead = 160L << 32;
// Runs of 512 columns at least, 64 for each wave, and more where that makes more workgroups than this: each forms u again.
// (128 rows of 100 adapters, 4096 to q/k/v 9216, for 512, 1024, 2048 and 4096 workgroups, which are runs of 4096 to 512 columns: 16.8,
// 13.4, 15.4 and 19.3 us.)
constexpr int kFewGroups = 1024;
// Many rows: at least two workgroups a CU, by shares of K and by shorter runs of columns.
constexpr int kManyGroups = 512, kShareK = 512, kManyRun = 512;
static_assert(kManyRun / kPiece <= 32, "a bit for each piece of a run");
static_assert(kManyRun / kPiece <= 32);  // bits of `left`

struct LoraForm {
  bool few;
  int tiles, shares, chunk;
};
LoraForm lora_form(const LoraLayout& p, int K, int R, int parts, int N) {
  const long part = (long)R * K;
  LoraForm f{p.M > 0 && part <= kFewAdapter && p.T * part * part <= kFewRead, p.N, 1, kManyRun};
  if (f.few) {
    f.tiles = p.M;
    for (f.chunk = 512; f.chunk < 4096 && (long)f.tiles * N / f.chunk > kFewGroups;) f.chunk *= 2;
  } else {
    while (f.shares < 8 && f.tiles * parts * f.shares < kManyGroups && K / (2 * f.shares) >= kShareK) f.shares *= 2;
    while (f.chunk > kPiece && (long)f.tiles * N / f.chunk < kManyGroups) f.chunk /= 2;
  }
  return f;
}

// Whether rows of y and of x share no value: they lie in different ranges, or side by side in rows of one length.  (What a
// workgroup adds to y is not ordered against what another reads of x.)
bool rows_disjoint(const uint16_t* y, long y_stride, long N, const uint16_t* x, long x_stride, long K, long T) {
  if (x + (T - 1) * x_stride + K <= y || y + (T - 1) * y_stride + N <= x) return true;
  if (y_stride != x_stride || T == 1) return false;
  const long at = ((x - y) % y_stride + y_stride) % y_stride;
  return at >= N && at + K <= y_stride;
}

size_t lora_ws(const LoraLayout& p, const LoraForm& f, int R, int parts) {
  return f.few ? 0 : moe_align_up((size_t)f.shares * p.T * parts * R * sizeof(float), 256);
}

template <int RG>
void launch(const LoraArgs& g, const LoraForm& f, hipStream_t s) {
  const dim3 columns(lora_grid(f.tiles, g.runs));
  if (f.few) {
    hipLaunchKernelGGL((lora_few_kernel<2 * RG>), columns, dim3(kFewThreads), 0, s, g);
    return;
  }
  const dim3 first(lora_grid(f.tiles, g.parts * g.shares * ((g.R + kRanksM - 1) / kRanksM)));
  hipLaunchKernelGGL((lora_shrink_kernel<(RG < 4 ? RG : 4)>), first, dim3(kThreads), 0, s, g);
  hipLaunchKernelGGL((lora_expand_kernel<RG>), columns, dim3(kThreads), 0, s, g);
}

}  // namespace

extern "C" size_t moe_mi355x_lora_add_workspace_bytes(int T, int L, int K, int R, int parts, const int* columns) {
  if (!lora_ok(T, L, K, R, parts) || !columns) return 0;
  long n = 0;
  for (int p = 0; p < parts; ++p) n += columns[p];
  if (n <= 0 || n > (1 << 24)) return 0;
  const LoraLayout p = lora_layout(T, L);
  return lora_ws(p, lora_form(p, K, R, parts, (int)n), R, parts);
}

extern "C" int moe_mi355x_lora_add(void* y, long long y_stride, const void* x, long long x_stride, const void* a,
                                   const void* b, const int32_t* ranks, const float* scales, const void* plan, int T,
                                   int L, int K, int R, int parts, const int* columns, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  MOE_RETURN_IF(!lora_ok(T, L, K, R, parts) || !columns, MOE_ERR_INVALID_ARG);
  LoraArgs g{};
  long n = 0;
  for (int p = 0; p < parts; ++p) {
    MOE_RETURN_IF(columns[p] <= 0 || columns[p] % 32, MOE_ERR_INVALID_ARG);
    n += columns[p];
    MOE_RETURN_IF(n > (1 << 24), MOE_ERR_INVALID_ARG);
    g.col[p + 1] = (int)n;
  }
  if (T == 0) return MOE_OK;
  MOE_RETURN_IF(!y || !x || !a || !b || !ranks || !scales || !plan, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(y_stride < n || x_stride < K, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(y_stride % 8 || x_stride % 8 || !moe_aligned16(y) || !moe_aligned16(x) || !moe_aligned16(a) ||
                    !moe_aligned16(b) || !moe_aligned16(plan),
                MOE_ERR_ALIGNMENT);
  g.p = lora_layout(T, L);
  const LoraForm f = lora_form(g.p, K, R, parts, (int)n);
  const size_t need = lora_ws(g.p, f, R, parts);
  MOE_RETURN_IF(need > 0 && (!workspace || workspace_bytes < need), MOE_ERR_WORKSPACE);
  MOE_RETURN_IF(need > 0 && !moe_aligned16(workspace), MOE_ERR_ALIGNMENT);
  MOE_RETURN_IF(!rows_disjoint((const uint16_t*)y, y_stride, n, (const uint16_t*)x, x_stride, K, T), MOE_ERR_INVALID_ARG);
  g.y = (uint16_t*)y, g.x = (const uint16_t*)x, g.y_stride = y_stride, g.x_stride = x_stride;
  g.a = (const uint16_t*)a, g.b = (const uint16_t*)b, g.ranks = ranks, g.scales = scales;
  g.plan = (const int32_t*)plan, g.u = (float*)workspace;
  g.K = K, g.R = R, g.N = (int)n, g.parts = parts, g.shares = f.shares, g.chunk = f.chunk;
  for (int p = 0; p < parts; ++p) g.runs += (columns[p] + f.chunk - 1) / f.chunk;
  MOE_RETURN_IF(!moe_grid_fits((long)(f.tiles + 7) * g.runs), MOE_ERR_INVALID_ARG);
  hipStream_t s = (hipStream_t)stream;
  if (R <= 16)
    launch<1>(g, f, s);
  else if (R <= 32)
    launch<2>(g, f, s);
  else if (R <= 64)
    launch<4>(g, f, s);
  else
    launch<8>(g, f, s);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
