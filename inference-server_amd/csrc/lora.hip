// What the adapters of a step's rows add to a shared projection: for row t with adapter l, column n in part p of the
// projection (q, k and v are parts of one), r < rank_l,
//   u[t, p, r] = sum_k x[t, k] A_l[p R + r, k]          y[t, n] = bf16( y[t, n] + scale_l sum_r u[t, p, r] B_l[n, r] )
// Both products on the bf16 MFMAs with fp32 sums.  u is split in two bf16 values for the second, u = hi + lo to 2^-17 of
// it: the 16 ranks of a group times {hi, lo} fill the 32 of an MFMA, so this costs B's operand read twice and no MFMA
// more than a group of 16 ranks takes anyway.  y enters as the accumulator and is rounded once.
//
// One workgroup per (tile of up to 16 MT rows of one adapter, run of columns): u by all waves, each with a share of K,
// joined in LDS; then each wave takes 32 columns at a time.
#include "lora.h"

namespace {

constexpr int kGroup = 16;     // ranks of an MFMA operand
constexpr int kMaxRank = 128;
constexpr int kMaxParts = 4;
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kCols = 32;      // columns that a wave takes at once

struct LoraArgs {
  uint16_t* y;        // [T][N], rows y_stride values apart
  const uint16_t* x;  // [T][K], rows x_stride values apart
  long y_stride, x_stride;
  const uint16_t *a, *b;  // [L][P R][K], [L][N][R]
  const int32_t* ranks;   // [L]
  const float* scales;    // [L]
  const int32_t* plan;
  LoraLayout p;
  int K, R, N, parts, chunk;  // chunk: columns of a workgroup, in one part
  int col[kMaxParts + 1];     // where the parts begin
};

template <int MT, int RG>
struct LoraLds {
  v4f part[kWaves][MT][RG][64];
  uint16_t u[16 * MT][RG][2][kGroup];  // hi, lo
};

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}
__device__ __forceinline__ float lo_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The first 8 * (lg & 1) + i < live of a lane's 8 values: ranks that the adapter has
__device__ __forceinline__ uint4 mask8(uint4 v, int live) {
  auto keep = [&](uint32_t w, int i) __attribute__((always_inline)) {
    return live >= i + 2 ? w : live == i + 1 ? w & 0xffffu : 0u;
  };
  return make_uint4(keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6));
}

template <int MT, int RG>
__global__ __launch_bounds__(kThreads) void lora_add_kernel(LoraArgs a) {
  __shared__ __attribute__((aligned(16))) LoraLds<MT, RG> lds;
  const int tile = blockIdx.y;
  if (tile >= a.plan[LH_TILES]) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int4 t = *(const int4*)(a.plan + a.p.tiles + 4L * tile);
  const int l = min(max(__builtin_amdgcn_readfirstlane(t.x), 0), a.p.L - 1), first = __builtin_amdgcn_readfirstlane(t.y);
  const int rows = __builtin_amdgcn_readfirstlane(t.z);
  const int rank = min(a.ranks[l], a.R);
  if (rank <= 0) return;
  int part = 0, c0 = blockIdx.x * a.chunk;  // every part has its own runs of columns
  for (;;) {
    const int n = a.col[part + 1] - a.col[part], runs = (n + a.chunk - 1) / a.chunk * a.chunk;
    if (c0 < runs) break;
    c0 -= runs;
    ++part;
  }
  c0 += a.col[part];
  const int c1 = min(c0 + a.chunk, a.col[part + 1]);

  int row[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int at = min(max(first + min(16 * m + lr, rows - 1), 0), a.p.T - 1);
    row[m] = min(max(a.plan[a.p.rows + at], 0), a.p.T - 1);
  }
  {
    v4f u[MT][RG];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g < RG; ++g) u[m][g] = (v4f){0.f, 0.f, 0.f, 0.f};
    const uint16_t* arow = a.a + ((long)l * a.parts + part) * a.R * a.K + (long)lr * a.K + 8 * lg;
    const int steps = a.K / 32, per = (steps + kWaves - 1) / kWaves;
    const int k0 = wave * per, k1 = min(k0 + per, steps);
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
      v8bf xv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m] = __builtin_bit_cast(v8bf, *(const uint4*)(a.x + row[m] * a.x_stride + 32 * k + 8 * lg));
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        if (g * kGroup >= rank) break;
        const v8bf av = __builtin_bit_cast(v8bf, *(const uint4*)(arow + (long)g * kGroup * a.K + 32 * k));
#pragma unroll
        for (int m = 0; m < MT; ++m) u[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, xv[m], u[m][g], 0, 0, 0);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g < RG; ++g) lds.part[wave][m][g][lane] = u[m][g];
  }
  __syncthreads();
  const float scale = a.scales[l];
  for (int i = threadIdx.x; i < MT * RG * 64; i += kThreads) {
    v4f s = (&lds.part[0][0][0][0])[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) s += (&lds.part[w][0][0][0])[i];
    const int g = i / 64 % RG, r0 = 4 * (i % 64 / 16);
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[2], rest[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[e] = g * kGroup + r0 + 2 * h + e < rank ? s[2 * h + e] * scale : 0.f;
        const float top = round_bf16(v[e]);
        rest[e] = fabsf(top) < INFINITY ? v[e] - top : 0.f;  // not inf - inf
      }
      hi[h] = pack2(v[0], v[1]);
      lo[h] = pack2(rest[0], rest[1]);
    }
    uint16_t* dst = &lds.u[i / 64 / RG * 16 + i % 16][g][0][r0];
    *(uint2*)dst = make_uint2(hi[0], hi[1]);
    *(uint2*)(dst + kGroup) = make_uint2(lo[0], lo[1]);
  }
  __syncthreads();

  v8bf uv[MT][RG];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int g = 0; g < RG; ++g) uv[m][g] = *(const v8bf*)&lds.u[16 * m + lr][g][lg >> 1][8 * (lg & 1)];
  // lane l holds columns 4 (l / 16) + i of row l % 16 of each product: two with their columns in turns of 4 make 8
  // in a row
  const uint16_t* bl = a.b + (long)l * a.N * a.R + 8 * (lg & 1);
  for (int c = c0 + kCols * wave; c < c1; c += kCols * kWaves) {
    v4f acc[MT][2];
    uint16_t* dst[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      dst[m] = a.y + row[m] * a.y_stride + c + 8 * lg;
      const uint4 v = *(const uint4*)dst[m];
      acc[m][0] = (v4f){lo_of(v.x), hi_of(v.x), lo_of(v.y), hi_of(v.y)};
      acc[m][1] = (v4f){lo_of(v.z), hi_of(v.z), lo_of(v.w), hi_of(v.w)};
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint16_t* bn = bl + (long)(c + 8 * (lr >> 2) + 4 * j + (lr & 3)) * a.R;
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        if (g * kGroup >= rank) break;
        const uint4 v = mask8(*(const uint4*)(bn + kGroup * g), rank - g * kGroup - 8 * (lg & 1));
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, v), uv[m][g], acc[m][j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (16 * m + lr < rows)
        *(uint4*)dst[m] = make_uint4(pack2(acc[m][0][0], acc[m][0][1]), pack2(acc[m][0][2], acc[m][0][3]),
                                     pack2(acc[m][1][0], acc[m][1][1]), pack2(acc[m][1][2], acc[m][1][3]));
  }
}

template <int MT>
void launch(const LoraArgs& a, dim3 grid, hipStream_t s) {
  const int groups = (a.R + kGroup - 1) / kGroup;
  if (groups == 1)
    hipLaunchKernelGGL((lora_add_kernel<MT, 1>), grid, dim3(kThreads), 0, s, a);
  else if (groups == 2)
    hipLaunchKernelGGL((lora_add_kernel<MT, 2>), grid, dim3(kThreads), 0, s, a);
  else if (groups <= 4)
    hipLaunchKernelGGL((lora_add_kernel<MT, 4>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((lora_add_kernel<MT, 8>), grid, dim3(kThreads), 0, s, a);
}

}  // namespace

extern "C" int moe_mi355x_lora_add(void* y, long long y_stride, const void* x, long long x_stride, const void* a,
                                   const void* b, const int32_t* ranks, const float* scales, const void* plan, int T,
                                   int L, int K, int R, int parts, const int* columns, void* stream) {
  MOE_RETURN_IF(!lora_plan_ok(T, L) || K <= 0 || K % 32 || R <= 0 || R % kGroup || R > kMaxRank, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(parts < 1 || parts > kMaxParts || !columns, MOE_ERR_INVALID_ARG);
  LoraArgs g{};
  long n = 0;
  for (int p = 0; p < parts; ++p) {
    MOE_RETURN_IF(columns[p] <= 0 || columns[p] % kCols, MOE_ERR_INVALID_ARG);
    n += columns[p];
    MOE_RETURN_IF(n > (1 << 24), MOE_ERR_INVALID_ARG);
    g.col[p + 1] = (int)n;
  }
  MOE_RETURN_IF(K > (1 << 24), MOE_ERR_INVALID_ARG);
  if (T == 0) return MOE_OK;
  MOE_RETURN_IF(!y || !x || !a || !b || !ranks || !scales || !plan, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(y_stride < n || x_stride < K, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(y_stride % 8 || x_stride % 8 || !moe_aligned16(y) || !moe_aligned16(x) || !moe_aligned16(a) ||
                    !moe_aligned16(b) || !moe_aligned16(plan),
                MOE_ERR_ALIGNMENT);
  g.y = (uint16_t*)y, g.x = (const uint16_t*)x, g.y_stride = y_stride, g.x_stride = x_stride;
  g.a = (const uint16_t*)a, g.b = (const uint16_t*)b, g.ranks = ranks, g.scales = scales;
  g.plan = (const int32_t*)plan, g.p = lora_layout(T, L);
  g.K = K, g.R = R, g.N = (int)n, g.parts = parts;
  g.chunk = g.p.N >= 64 ? 1024 : 256;
  int runs = 0;
  for (int p = 0; p < parts; ++p) runs += (columns[p] + g.chunk - 1) / g.chunk;
  const dim3 grid(runs, g.p.N);
  if (g.p.tile_rows == 16)
    launch<1>(g, grid, (hipStream_t)stream);
  else
    launch<2>(g, grid, (hipStream_t)stream);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
