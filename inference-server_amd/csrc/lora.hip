// What the adapters of a step's rows add to a shared projection: for row t with adapter l, column n in part p of the
// projection (q, k and v are parts of one), r < rank_l,
//   u[t, p, r] = sum_k x[t, k] A_l[p R + r, k]          y[t, n] = bf16( y[t, n] + scale_l sum_r u[t, p, r] B_l[n, r] )
// Both products on the bf16 MFMAs with fp32 sums.  u is split in two bf16 values for the second, u = hi + lo to 2^-17 of
// it: the 16 ranks of a group times {hi, lo} fill the 32 of an MFMA, so this costs B's operand read twice and no MFMA
// more than a group of 16 ranks takes anyway.  y enters as the accumulator and is rounded once.
//
// Two forms over the plan's tiles (up to tile_rows rows of one adapter):
//   one launch: a workgroup per (tile, run of columns) forms the u of its part by itself;
//   two: u of every (tile, part, share of K) to the workspace, in fp32, then the columns.
#include "lora.h"

namespace {

constexpr int kGroup = 16;     // ranks of an MFMA operand
constexpr int kMaxRank = 128;
constexpr int kMaxParts = 4;
constexpr int kCols = 32;      // columns that a wave takes at once

struct LoraArgs {
  uint16_t* y;        // [T][N], rows y_stride values apart
  const uint16_t* x;  // [T][K], rows x_stride values apart
  long y_stride, x_stride;
  const uint16_t *a, *b;  // [L][P R][K], [L][N][R]
  const int32_t* ranks;   // [L]
  const float* scales;    // [L]
  const int32_t* plan;
  float* u;               // [shares][T][P][R], rows in the plan's order
  LoraLayout p;
  int K, R, N, parts, shares, chunk;  // chunk: columns of a workgroup, in one part
  int col[kMaxParts + 1];             // where the parts begin
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}
__device__ __forceinline__ float lo_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The first `live` of a lane's 8 values: ranks that the adapter has
__device__ __forceinline__ uint4 mask8(uint4 v, int live) {
  auto keep = [&](uint32_t w, int i) __attribute__((always_inline)) {
    return live >= i + 2 ? w : live == i + 1 ? w & 0xffffu : 0u;
  };
  return make_uint4(keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6));
}

// A workgroup's rows: up to 16 MT of a tile
template <int MT>
struct Rows {
  int l, first, n, rank;  // adapter, first entry of the sorted rows, rows (0: nothing to do), rank
  int row[MT];            // this lane's, of each 16: l & 15

  __device__ __forceinline__ Rows(const LoraArgs& a, int block, int lane) {
    const int sub = a.p.tile_rows / (16 * MT), tile = block / sub, at = block % sub * 16 * MT;
    const int4 t = *(const int4*)(a.plan + a.p.tiles + 4L * tile);
    const bool live = tile < a.plan[LH_TILES];
    l = min(max(__builtin_amdgcn_readfirstlane(t.x), 0), a.p.L - 1);
    first = min(max(__builtin_amdgcn_readfirstlane(t.y) + at, 0), a.p.T - 1);
    n = live ? min(__builtin_amdgcn_readfirstlane(t.z) - at, 16 * MT) : 0;
    if (n <= 0) return;
    rank = min(a.ranks[l], a.R);
    if (rank <= 0) n = 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int i = min(first + min(16 * m + (lane & 15), max(n, 1) - 1), a.p.T - 1);
      row[m] = min(max(a.plan[a.p.rows + i], 0), a.p.T - 1);
    }
  }
};

// u of 16 MT rows and 16 NG ranks of a part, over the k steps (of 32) k0 .. k1: lane l holds ranks 16 g + 4 (l / 16) + i
// of row 16 m + l % 16.  kAhead steps' loads are in flight together.
template <int MT, int NG, int kAhead>
__device__ __forceinline__ void shrink(const LoraArgs& a, const Rows<MT>& r, int part, int k0, int k1, int lane, v4f (&u)[MT][NG]) {
  const int lr = lane & 15, lg = lane >> 4;
  const uint16_t *xr[MT], *ar[NG];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = a.x + r.row[m] * a.x_stride + 8 * lg;
#pragma unroll
  for (int g = 0; g < NG; ++g) ar[g] = a.a + (((long)r.l * a.parts + part) * a.R + min(kGroup * g + lr, a.R - 1)) * a.K + 8 * lg;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int g = 0; g < NG; ++g) u[m][g] = (v4f){0.f, 0.f, 0.f, 0.f};
  auto steps = [&](int k, auto count) __attribute__((always_inline)) {
    constexpr int n = decltype(count)::value;
    uint4 xv[n][MT], av[n][NG];
#pragma unroll
    for (int i = 0; i < n; ++i) {
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[i][m] = *(const uint4*)(xr[m] + 32 * (k + i));
#pragma unroll
      for (int g = 0; g < NG; ++g) av[i][g] = *(const uint4*)(ar[g] + 32 * (k + i));
    }
#pragma unroll
    for (int i = 0; i < n; ++i)
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          u[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, av[i][g]), __builtin_bit_cast(v8bf, xv[i][m]),
                                                            u[m][g], 0, 0, 0);
  };
  int k = k0;
  for (; k + kAhead <= k1; k += kAhead) steps(k, std::integral_constant<int, kAhead>());
  for (; k < k1; ++k) steps(k, std::integral_constant<int, 1>());
}

// 4 ranks' u as they enter the second product
__device__ __forceinline__ void split_u(v4f s, float scale, int live, uint2* hi, uint2* lo) {
  float v[4], rest[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = e < live ? s[e] * scale : 0.f;
    const float top = round_bf16(v[e]);
    rest[e] = fabsf(top) < INFINITY ? v[e] - top : 0.f;  // not inf - inf
  }
  *hi = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  *lo = make_uint2(pack2(rest[0], rest[1]), pack2(rest[2], rest[3]));
}

template <int MT, int RG>
struct ULds {
  uint16_t u[16 * MT][RG][2][kGroup];  // hi, lo
};

// The columns c0 .. c1 (in one part), 32 at a time for each of kWaves waves
template <int MT, int NG, int RG, int kWaves>
__device__ __forceinline__ void expand(const LoraArgs& a, const Rows<MT>& r, const ULds<MT, RG>& lds, int c0, int c1, int lane,
                                       int wave) {
  const int lr = lane & 15, lg = lane >> 4;
  v8bf uv[MT][NG];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int g = 0; g < NG; ++g) uv[m][g] = *(const v8bf*)&lds.u[16 * m + lr][g][lg >> 1][8 * (lg & 1)];
  // lane l holds columns 4 (l / 16) + i of row l % 16 of each product: two with their columns in turns of 4 make 8
  // in a row
  const uint16_t* bl = a.b + ((long)r.l * a.N + 8 * (lr >> 2) + (lr & 3)) * a.R + 8 * (lg & 1);
  for (int c = c0 + kCols * wave; c < c1; c += kCols * kWaves) {
    uint4 yv[MT], bv[2][NG];
#pragma unroll
    for (int m = 0; m < MT; ++m) yv[m] = *(const uint4*)(a.y + r.row[m] * a.y_stride + c + 8 * lg);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < NG; ++g) bv[j][g] = *(const uint4*)(bl + (long)(c + 4 * j) * a.R + min(kGroup * g, a.R - kGroup));
    v4f acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      acc[m][0] = (v4f){lo_of(yv[m].x), hi_of(yv[m].x), lo_of(yv[m].y), hi_of(yv[m].y)};
      acc[m][1] = (v4f){lo_of(yv[m].z), hi_of(yv[m].z), lo_of(yv[m].w), hi_of(yv[m].w)};
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint4 v = bv[j][g];
        if (kGroup * (g + 1) > r.rank) v = mask8(v, r.rank - kGroup * g - 8 * (lg & 1));
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, v), uv[m][g], acc[m][j], 0, 0, 0);
      }
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (16 * m + lr < r.n)
        *(uint4*)(a.y + r.row[m] * a.y_stride + c + 8 * lg) =
            make_uint4(pack2(acc[m][0][0], acc[m][0][1]), pack2(acc[m][0][2], acc[m][0][3]),
                       pack2(acc[m][1][0], acc[m][1][1]), pack2(acc[m][1][2], acc[m][1][3]));
  }
}

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

// fn of the number of 16-rank groups that the adapter has: 1, 2, 4 or 8 as a constant
template <int RG, typename F>
__device__ __forceinline__ void by_groups(int rank, F fn) {
  if (RG == 1 || rank <= 16) return fn(std::integral_constant<int, 1>());
  if constexpr (RG >= 2)
    if (RG == 2 || rank <= 32) return fn(std::integral_constant<int, 2>());
  if constexpr (RG >= 4)
    if (RG == 4 || rank <= 64) return fn(std::integral_constant<int, 4>());
  if constexpr (RG >= 8) return fn(std::integral_constant<int, 8>());
}

template <int RG>
__global__ __launch_bounds__(512) void lora_one_kernel(LoraArgs a) {
  constexpr int kWaves = 8, kThreads = 64 * kWaves;
  __shared__ __attribute__((aligned(16))) struct {
    v4f part[kWaves][RG][64];
    ULds<1, RG> u;
  } lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<1> r(a, blockIdx.y, lane);
  if (r.n <= 0) return;
  int part, c0, c1;
  run_of(a, blockIdx.x, &part, &c0, &c1);
  const float scale = a.scales[r.l];
  by_groups<RG>(r.rank, [&](auto groups) __attribute__((always_inline)) {
    constexpr int NG = decltype(groups)::value;
    v4f u[1][NG];
    const int steps = a.K / 32, per = (steps + kWaves - 1) / kWaves;
    shrink<1, NG, (NG <= 2 ? 8 : NG <= 4 ? 4 : 2)>(a, r, part, min(wave * per, steps), min((wave + 1) * per, steps), lane, u);
#pragma unroll
    for (int g = 0; g < NG; ++g) lds.part[wave][g][lane] = u[0][g];
    __syncthreads();
    for (int i = threadIdx.x; i < NG * 64; i += kThreads) {
      const int g = i / 64, r0 = 4 * (i % 64 / 16);
      v4f s = lds.part[0][g][i % 64];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s += lds.part[w][g][i % 64];
      split_u(s, scale, r.rank - kGroup * g - r0, (uint2*)&lds.u.u[i % 16][g][0][r0], (uint2*)&lds.u.u[i % 16][g][1][r0]);
    }
    __syncthreads();
    expand<1, NG, RG, kWaves>(a, r, lds.u, c0, c1, lane, wave);
  });
}

template <int MT, int RG>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a) {
  constexpr int kWaves = 4, kThreads = 64 * kWaves;
  __shared__ __attribute__((aligned(16))) v4f lds[kWaves][MT][RG][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<MT> r(a, blockIdx.y, lane);
  if (r.n <= 0) return;
  const int part = blockIdx.x % a.parts, share = blockIdx.x / a.parts;
  by_groups<RG>(r.rank, [&](auto groups) __attribute__((always_inline)) {
    constexpr int NG = decltype(groups)::value;
    v4f u[MT][NG];
    const int steps = a.K / 32, per = (steps + a.shares * kWaves - 1) / (a.shares * kWaves), at = (share * kWaves + wave) * per;
    shrink<MT, NG, (MT + NG <= 3 ? 8 : MT + NG <= 6 ? 4 : 2)>(a, r, part, min(at, steps), min(at + per, steps), lane, u);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g < NG; ++g) lds[wave][m][g][lane] = u[m][g];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * NG * 64; i += kThreads) {
      const int m = i / (64 * NG), g = i / 64 % NG, row = 16 * m + i % 16;
      v4f s = lds[0][m][g][i % 64];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) s += lds[w][m][g][i % 64];
      const int rank0 = kGroup * g + 4 * (i % 64 / 16);
      if (row < r.n && rank0 < a.R)
        *(v4f*)(a.u + (((long)share * a.p.T + r.first + row) * a.parts + part) * a.R + rank0) = s;
    }
  });
}

template <int MT, int RG>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  constexpr int kWaves = 4, kThreads = 64 * kWaves;
  __shared__ __attribute__((aligned(16))) ULds<MT, RG> lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<MT> r(a, blockIdx.y, lane);
  if (r.n <= 0) return;
  int part, c0, c1;
  run_of(a, blockIdx.x, &part, &c0, &c1);
  const float scale = a.scales[r.l];
  by_groups<RG>(r.rank, [&](auto groups) __attribute__((always_inline)) {
    constexpr int NG = decltype(groups)::value;
    for (int i = threadIdx.x; i < 16 * MT * NG * 4; i += kThreads) {
      const int row = i / (NG * 4), r0 = 4 * (i % (NG * 4)), from = min(row, r.n - 1);
      v4f s = {0.f, 0.f, 0.f, 0.f};
      const float* src = a.u + (((long)r.first + from) * a.parts + part) * a.R + min(r0, a.R - 4);
      for (int z = 0; z < a.shares; ++z) s += *(const v4f*)(src + (long)z * a.p.T * a.parts * a.R);
      uint16_t* dst = &lds.u[row][r0 / kGroup][0][r0 % kGroup];
      split_u(s, scale, r.rank - r0, (uint2*)dst, (uint2*)(dst + kGroup));
    }
    __syncthreads();
    expand<MT, NG, RG, kWaves>(a, r, lds, c0, c1, lane, wave);
  });
}

bool lora_ok(int T, int L, int K, int R, int parts) {
  return lora_plan_ok(T, L) && K > 0 && K % 32 == 0 && K <= (1 << 24) && R > 0 && R % kGroup == 0 && R <= kMaxRank && parts >= 1 &&
         parts <= kMaxParts;
}

// Which form a call takes, and its shape
struct LoraForm {
  bool one;
  int shares, mt, chunk;
};
#ifndef LORA_ONE
#define LORA_ONE 0
#endif
#ifndef LORA_CHUNK
#define LORA_CHUNK 512
#endif
#ifndef LORA_MT
#define LORA_MT 4
#endif
#ifndef LORA_WGS
#define LORA_WGS 256
#endif
LoraForm lora_form(const LoraLayout& p, int K, int R, int parts, int N) {
  LoraForm f{};
  f.one = p.tile_rows == 16 && LORA_ONE;
  f.mt = p.tile_rows == 16 ? 1 : R > 64 ? 2 : LORA_MT;
  f.shares = 1;
  if (!f.one)
    while (f.shares < 8 && p.N * parts * f.shares < LORA_WGS && K / (2 * f.shares) >= 512) f.shares *= 2;
  f.chunk = LORA_CHUNK;
  if (f.mt == 1) f.chunk = p.N * N / 256 > 1024 ? 512 : 256;
  if (f.mt == 1 && !f.one) f.chunk /= 2;
  return f;
}

size_t lora_ws(const LoraLayout& p, const LoraForm& f, int R, int parts) {
  return f.one ? 0 : moe_align_up((size_t)f.shares * p.T * parts * R * sizeof(float), 256);
}

template <int RG>
void launch(const LoraArgs& g, const LoraForm& f, int runs, hipStream_t s) {
  if (f.one) {
    hipLaunchKernelGGL((lora_one_kernel<RG>), dim3(runs, g.p.N), dim3(512), 0, s, g);
    return;
  }
  const int blocks = g.p.N * (g.p.tile_rows / (16 * f.mt));
  const dim3 first(g.parts * g.shares, blocks), second(runs, blocks);
#define LORA_LAUNCH(MT)                                                                       \
  do {                                                                                        \
    hipLaunchKernelGGL((lora_shrink_kernel<MT, RG>), first, dim3(256), 0, s, g);              \
    hipLaunchKernelGGL((lora_expand_kernel<MT, RG>), second, dim3(256), 0, s, g);             \
  } while (0)
  if (f.mt == 1) LORA_LAUNCH(1);
  else if (f.mt == 2) LORA_LAUNCH(2);
  else if constexpr (RG <= 4) LORA_LAUNCH(4);
#undef LORA_LAUNCH
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
    MOE_RETURN_IF(columns[p] <= 0 || columns[p] % kCols, MOE_ERR_INVALID_ARG);
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
  g.y = (uint16_t*)y, g.x = (const uint16_t*)x, g.y_stride = y_stride, g.x_stride = x_stride;
  g.a = (const uint16_t*)a, g.b = (const uint16_t*)b, g.ranks = ranks, g.scales = scales;
  g.plan = (const int32_t*)plan, g.u = (float*)workspace;
  g.K = K, g.R = R, g.N = (int)n, g.parts = parts, g.shares = f.shares, g.chunk = f.chunk;
  int runs = 0;
  for (int p = 0; p < parts; ++p) runs += (columns[p] + f.chunk - 1) / f.chunk;
  hipStream_t s = (hipStream_t)stream;
  if (R <= 16)
    launch<1>(g, f, runs, s);
  else if (R <= 32)
    launch<2>(g, f, runs, s);
  else if (R <= 64)
    launch<4>(g, f, runs, s);
  else
    launch<8>(g, f, runs, s);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
