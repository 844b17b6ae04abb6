// Writers of the 8-bit KV pages (kv_fp8.h): this step's keys and values, prompts' and single tokens' alike,
// quantised with one scale per (page, kv head).  moe_mi355x_kv_append_fp8 takes k and v as they are,
// moe_mi355x_qk_norm_rope_append_fp8 the fused q/k/v projections: it also does q_norm / k_norm, the rotary embedding
// and q's output (Qwen3MoeAttention.forward, TF/models/qwen3_moe/modeling_qwen3_moe.py:162-171).
//
// For a page that gets tokens, with a = the largest finite |x| among them,
//   s_need = the smallest power of two with a / s <= 448
//   s      = s_need where the page begins with these tokens, max(s_old, s_need) otherwise
//   code   = e4m3(clamp(x / s, -448, 448)),   old codes: e4m3(code * s_old / s)
// A page that begins is written whole (zeros behind its tokens), so nothing stale is ever read from it.
//
// One wave per (page that gets tokens, kv head, K or V), from the plan's list: it alone writes the block, so
// there are no atomics and no second pass, and the maximum is a wave's.  norm and rotary of q stay in fp32 from the bf16
// projection to the one rounding to bf16.  Its angle is position * inv_freq in 64 bits, reduced to a turn before
// it is rounded to 32: at position 10^5 a 32-bit product is off by up to 0.004.  Those of k, of which there are few
// rows, are in 64 bits throughout: in 32, two to eight codes of 4 million fell on the other side of a tie, each 2^-4 of
// its value away (8178 tokens, 64 / 4 heads: 54.4 -> 56.1 us; 16 tokens alike, 4.6).
// HBM bound for long prompts with q (512 B read and 256 B written per token and kv head, 512 B per token and q head:
// 5.2 TB/s for 8178 tokens, 64 / 4 heads).  K and V alone are too few bytes for that: 4499 tokens, 4 kv heads, take
// 5.8 us at 2.4 TB/s, for a wave's one chain of record, rows, maximum and stores.
#include "kv_fp8.h"
#include "paged_plan.h"

namespace {

constexpr int kHD = kKvHead;
constexpr int kPage = kPlanPage;

struct KvArgs {
  const uint16_t *k, *v;  // rows of Hkv * 128 values, k_stride and v_stride values apart
  long k_stride, v_stride;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;  // [num_pages][Hkv]
  const int32_t* plan;
  const int4* writes;
  int Hkv, num_pages, max_writes;
  // fused form
  const uint16_t *q, *qw, *kw;  // q rows, q_stride values apart
  long q_stride;
  const float* inv_freq;
  const int32_t* pos;
  uint16_t* q_out;  // [T][Hq][128]
  int T, Hq, write_blocks;
  float eps;
};

// 8 values that are read once: past the caches (3% at 8178 tokens and 64 / 4 heads)
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u4*)p));
}

__device__ __forceinline__ void unpack8(uint4 r, float* x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// |x| for the page's scale: infinities and NaN do not count
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// Norm and rotary of one head's row held by 8 adjacent lanes: lane j has dims 8 j .. +8 (x[0..8)) and
// 64 + 8 j .. +8 (x[8..16)), the pairs that the rotation mixes; w: the norm weight's same dims.
__device__ __forceinline__ void norm_rope(float* x, const float* w, const float* c, const float* s, float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
  ss += __shfl_xor(ss, 1);
  ss += __shfl_xor(ss, 2);
  ss += __shfl_xor(ss, 4);
  const float r = 1.0f / sqrtf(ss * (1.0f / kHD) + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i] * r * w[i], b = x[8 + i] * r * w[8 + i];
    x[i] = a * c[i] - b * s[i];
    x[8 + i] = b * c[i] + a * s[i];
  }
}

// cos and sin of pos * inv_freq.  What is left of the angle behind whole quarter turns is at most 1 / 8 turn, so
// its rounding to 32 bits moves it by 2^-28 turns (2.3e-8 rad), below fp32's step for cos and sin.
__device__ __forceinline__ void rope_angle(int pos, float inv_freq, float* c, float* s) {
  const double quarters = (double)pos * (double)inv_freq * 0.63661977236758134308;  // 2 / pi
  const double whole = rint(quarters);
  float cr, sr;
  sincospif(0.5f * (float)(quarters - whole), &sr, &cr);
  const int q = (int)(long long)whole & 3;
  const float a = q & 1 ? sr : cr, b = q & 1 ? cr : sr;
  *c = q == 1 || q == 2 ? -a : a;
  *s = q >= 2 ? -b : b;
}

// x in 32 bits, an inexact one with its last bit set: rounding that to e4m3 is rounding x to e4m3.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = (float)x;
  uint32_t b = __float_as_uint(f);
  if (fabs((double)f) > fabs(x)) b -= 1;
  if ((double)f < x || (double)f > x) b |= 1;
  return __uint_as_float(b);
}

// The same for a k row, angles included, in 64 bits.  Four pairs at a time are enough to fill the lanes' pipeline; all
// eight take registers that other waves miss (56.9 us against 56.1).
__device__ __forceinline__ void norm_rope_k(float* x, const float* w, const float* inv_freq, int pos, float eps) {
  double ss = 0.;
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = fma((double)x[i], (double)x[i], ss);
  ss += __shfl_xor(ss, 1);
  ss += __shfl_xor(ss, 2);
  ss += __shfl_xor(ss, 4);
  const double r = 1.0 / sqrt(ss * (1.0 / kHD) + (double)eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double quarters = (double)pos * (double)inv_freq[i] * 0.63661977236758134308;  // 2 / pi
    const double whole = rint(quarters);
    // Taylor's series on |angle| <= pi / 4, off by 4e-13 at most
    const double t = (quarters - whole) * 1.57079632679489661923, z = t * t;
    const double sr = t * fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, 1. / 6227020800., -1. / 39916800.), 1. / 362880.), -1. / 5040.),
                                            1. / 120.), -1. / 6.), 1.);
    const double cr = fma(z, fma(z, fma(z, fma(z, fma(z, fma(z, 1. / 479001600., -1. / 3628800.), 1. / 40320.), -1. / 720.), 1. / 24.),
                                 -.5), 1.);
    const int q = (int)(long long)whole & 3;
    const double u = q & 1 ? sr : cr, v = q & 1 ? cr : sr;
    const double c = q == 1 || q == 2 ? -u : u, s = q >= 2 ? -v : v;
    const double a = x[i] * r * w[i], b = x[8 + i] * r * w[8 + i];
    x[i] = round_to_odd(a * c - b * s);
    x[8 + i] = round_to_odd(b * c + a * s);
    if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
  }
}

template <bool FUSED>
__device__ __forceinline__ void write_k(const KvArgs& a, int4 w, int g, int lane) {
  const int tl = lane >> 3, j = lane & 7;  // rounds r = 0, 1: token tl + 8 r
  const bool fresh = w.z == 0;
  const long blk = (long)w.x * a.Hkv + g;
  uint8_t* dst = a.k_cache + blk * kKvBlock + (j >> 1) * 256 + (j & 1) * 8;  // + 16 token, + 1024 for the upper dims
  float x[2][16];
  uint2 old[2][2];
  float old_scale = 0.f;
  float wt[16];
  if constexpr (FUSED) {
    unpack8(*(const uint4*)(a.kw + 8 * j), wt);
    unpack8(*(const uint4*)(a.kw + 64 + 8 * j), wt + 8);
  }
  if (!fresh) {  // wave-uniform
    old_scale = a.k_scale[blk];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      old[r][0] = *(const uint2*)(dst + (tl + 8 * r) * 16);
      old[r][1] = *(const uint2*)(dst + (tl + 8 * r) * 16 + 1024);
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = tl + 8 * r;
    const bool live = t >= w.z && t < w.z + w.w;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[r][i] = 0.f;
    if (live) {
      const int row = w.y + t - w.z;
      const uint16_t* src = a.k + row * a.k_stride + (long)g * kHD + 8 * j;
      unpack8(load_once(src), x[r]);
      unpack8(load_once(src + 64), x[r] + 8);
    }
    if constexpr (FUSED) {
      if (8 * r < w.z + w.w && 8 * r + 8 > w.z) {  // wave-uniform: a round with tokens
        const int pos = a.pos[w.y - w.z + (live ? t : w.z)];
        norm_rope_k(x[r], wt, a.inv_freq + 8 * j, pos, a.eps);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (FUSED && !live) x[r][i] = 0.f;  // with eps 0 the norm of no token is NaN
      amax = fmaxf(amax, finite_abs(x[r][i]));
    }
  }
  const float need = kv_scale(wave_max_uniform(amax));
  const float scale = fresh ? need : fmaxf(old_scale, need);
  const float inv = 1.0f / scale, ratio = old_scale * inv;
  const bool recode = !fresh && scale != old_scale;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = tl + 8 * r;
    const bool live = t >= w.z && t < w.z + w.w;
    uint2 lo, hi;
    lo.x = kv_pack4(x[r][0], x[r][1], x[r][2], x[r][3], inv);
    lo.y = kv_pack4(x[r][4], x[r][5], x[r][6], x[r][7], inv);
    hi.x = kv_pack4(x[r][8], x[r][9], x[r][10], x[r][11], inv);
    hi.y = kv_pack4(x[r][12], x[r][13], x[r][14], x[r][15], inv);
    if (recode && !live) {
      lo = make_uint2(kv_recode4(old[r][0].x, ratio), kv_recode4(old[r][0].y, ratio));
      hi = make_uint2(kv_recode4(old[r][1].x, ratio), kv_recode4(old[r][1].y, ratio));
    }
    if (live || fresh || recode) {
      *(uint2*)(dst + t * 16) = lo;
      *(uint2*)(dst + t * 16 + 1024) = hi;
    }
  }
  if (lane == 0) a.k_scale[blk] = scale;
}

__device__ __forceinline__ void write_v(const KvArgs& a, int4 w, int g, int lane) {
  const int quad = lane >> 4, j = lane & 15;  // tokens 4 quad .. +4, dims 8 j .. +8
  const bool fresh = w.z == 0;
  const long blk = (long)w.x * a.Hkv + g;
  uint8_t* dst = a.v_cache + blk * kKvBlock + (j >> 3) * 1024 + quad * 256 + (j & 7) * 32;
  uint32_t old[8];
  float old_scale = 0.f;
  if (!fresh) {  // wave-uniform
    old_scale = a.v_scale[blk];
    const uint4 lo = *(const uint4*)dst, hi = *(const uint4*)(dst + 16);
    const uint32_t o[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) old[i] = o[i];
  }
  float x[4][8];
  uint32_t mask = 0;  // the new tokens' bytes
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * quad + i;
#pragma unroll
    for (int d = 0; d < 8; ++d) x[i][d] = 0.f;
    if (t >= w.z && t < w.z + w.w) {
      mask |= 0xffu << (8 * i);
      const int row = w.y + t - w.z;
      unpack8(load_once(a.v + row * a.v_stride + (long)g * kHD + 8 * j), x[i]);
#pragma unroll
      for (int d = 0; d < 8; ++d) amax = fmaxf(amax, finite_abs(x[i][d]));
    }
  }
  const float need = kv_scale(wave_max_uniform(amax));
  const float scale = fresh ? need : fmaxf(old_scale, need);
  const float inv = 1.0f / scale, ratio = old_scale * inv;
  const bool recode = !fresh && scale != old_scale;
  uint32_t y[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) y[d] = kv_pack4(x[0][d], x[1][d], x[2][d], x[3][d], inv);
  if (!fresh) {
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint32_t keep = recode ? kv_recode4(old[d], ratio) : old[d];
      y[d] = (y[d] & mask) | (keep & ~mask);
    }
  }
  if (fresh || recode || mask) {
    *(uint4*)dst = make_uint4(y[0], y[1], y[2], y[3]);
    *(uint4*)(dst + 16) = make_uint4(y[4], y[5], y[6], y[7]);
  }
  if (lane == 0) a.v_scale[blk] = scale;
}

// One token's q heads: norm, rotary, bf16.  8 heads at a time, 8 lanes each; the 64 angles once.
__device__ __forceinline__ void write_q(const KvArgs& a, int t, int lane) {
  const int hl = lane >> 3, j = lane & 7;
  const int pos = a.pos[t];
  uint16_t* out = a.q_out + (long)t * a.Hq * kHD;
  float ca, sa, c[8], s[8], wt[16];
  rope_angle(pos, a.inv_freq[lane], &ca, &sa);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = __shfl(ca, 8 * j + i);
    s[i] = __shfl(sa, 8 * j + i);
  }
  unpack8(*(const uint4*)(a.qw + 8 * j), wt);
  unpack8(*(const uint4*)(a.qw + 64 + 8 * j), wt + 8);
  for (int h0 = 0; h0 < a.Hq; h0 += 8) {  // wave-uniform
    const int h = min(h0 + hl, a.Hq - 1);
    const uint16_t* src = a.q + t * a.q_stride + (long)h * kHD + 8 * j;
    float x[16];
    unpack8(load_once(src), x);
    unpack8(load_once(src + 64), x + 8);
    norm_rope(x, wt, c, s, a.eps);
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)  // a row behind the last sequence: zeros
      o[i] = pos < 0 ? 0u : (uint32_t)f32_to_bf16(x[2 * i]) | ((uint32_t)f32_to_bf16(x[2 * i + 1]) << 16);
    if (h0 + hl < a.Hq) {
      uint16_t* dst = out + (long)h * kHD + 8 * j;
      *(uint4*)dst = make_uint4(o[0], o[1], o[2], o[3]);
      *(uint4*)(dst + 64) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

template <bool FUSED>
__global__ __launch_bounds__(256) void kv_append_fp8_kernel(KvArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (FUSED && (int)blockIdx.x >= a.write_blocks) {
    const int t = ((int)blockIdx.x - a.write_blocks) * 4 + wave;
    if (t < a.T) write_q(a, t, lane);
    return;
  }
  const int item = (int)blockIdx.x * 4 + wave;
  const int part = item % (2 * a.Hkv), i = item / (2 * a.Hkv);
  const int count = a.plan[PH_WRITES];
  int4 w = a.writes[min(i, a.max_writes - 1)];
  asm volatile("" : "+v"(w.x));  // one round trip: the record, in the list or behind its end, with the count
  if (i >= count) return;
  w = make_int4(__builtin_amdgcn_readfirstlane(w.x), __builtin_amdgcn_readfirstlane(w.y), __builtin_amdgcn_readfirstlane(w.z),
                __builtin_amdgcn_readfirstlane(w.w));
  if (w.x < 0 || w.x >= a.num_pages) return;  // no page: the tokens are not kept
  if (part < a.Hkv)
    write_k<FUSED>(a, w, part, lane);
  else
    write_v(a, w, part - a.Hkv, lane);
}

bool kv_args_ok(const moe_mi355x_plan_shape* shape, int head_dim, int page_size, int num_pages) {
  return plan_shape_ok(shape) && head_dim == kHD && page_size == kPage && num_pages >= 0;
}

// The cache and the plan as the kernels take them.
KvArgs kv_args(void* k_cache, void* v_cache, float* k_scale, float* v_scale, int num_pages, const PlanLayout& p,
               const void* plan) {
  KvArgs a{};
  a.k_cache = (uint8_t*)k_cache, a.v_cache = (uint8_t*)v_cache;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.plan = (const int32_t*)plan;
  a.writes = (const int4*)(a.plan + p.writes);
  a.pos = a.plan + p.pos;
  a.Hkv = p.Hkv, a.num_pages = num_pages, a.max_writes = p.W, a.T = p.T, a.Hq = p.Hq;
  return a;
}

long write_blocks(const PlanLayout& p) { return ((long)p.W * 2 * p.Hkv + 3) / 4; }

}  // namespace

extern "C" int moe_mi355x_kv_append_fp8(const void* k, const void* v, long long k_stride, long long v_stride,
                                        void* k_cache, void* v_cache, float* k_scale, float* v_scale, int head_dim,
                                        int page_size, int num_pages, const moe_mi355x_plan_shape* shape,
                                        const void* plan, void* stream) {
  MOE_RETURN_IF(!kv_args_ok(shape, head_dim, page_size, num_pages), MOE_ERR_INVALID_ARG);
  if (shape->tokens == 0) return MOE_OK;
  MOE_RETURN_IF(!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !plan, MOE_ERR_INVALID_ARG);
  const PlanLayout p = plan_layout(shape);
  MOE_RETURN_IF(k_stride < (long)p.Hkv * kHD || v_stride < (long)p.Hkv * kHD, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(k_stride % 8 || v_stride % 8 || !moe_aligned16(k) || !moe_aligned16(v) || !moe_aligned16(k_cache) ||
                    !moe_aligned16(v_cache) || !moe_aligned16(plan),
                MOE_ERR_ALIGNMENT);
  MOE_RETURN_IF(!moe_grid_fits(write_blocks(p)), MOE_ERR_INVALID_ARG);
  if (p.W == 0) return MOE_OK;
  KvArgs a = kv_args(k_cache, v_cache, k_scale, v_scale, num_pages, p, plan);
  a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.k_stride = k_stride, a.v_stride = v_stride;
  hipLaunchKernelGGL(kv_append_fp8_kernel<false>, dim3((unsigned)write_blocks(p)), dim3(256), 0, (hipStream_t)stream, a);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

extern "C" int moe_mi355x_qk_norm_rope_append_fp8(const void* qkv, const void* q_norm_w, const void* k_norm_w,
                                                  const float* inv_freq, float eps, void* q_out, void* k_cache,
                                                  void* v_cache, float* k_scale, float* v_scale, int head_dim,
                                                  int page_size, int num_pages, const moe_mi355x_plan_shape* shape,
                                                  const void* plan, void* stream) {
  MOE_RETURN_IF(!kv_args_ok(shape, head_dim, page_size, num_pages), MOE_ERR_INVALID_ARG);
  if (shape->tokens == 0) return MOE_OK;
  MOE_RETURN_IF(!qkv || !q_norm_w || !k_norm_w || !inv_freq || !q_out || !k_cache || !v_cache || !k_scale ||
                    !v_scale || !plan,
                MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(!moe_aligned16(qkv) || !moe_aligned16(q_norm_w) || !moe_aligned16(k_norm_w) || !moe_aligned16(q_out) ||
                    !moe_aligned16(k_cache) || !moe_aligned16(v_cache) || !moe_aligned16(plan),
                MOE_ERR_ALIGNMENT);
  const PlanLayout p = plan_layout(shape);
  const long blocks = write_blocks(p) + (p.T + 3) / 4;
  MOE_RETURN_IF(!moe_grid_fits(blocks), MOE_ERR_INVALID_ARG);
  KvArgs a = kv_args(k_cache, v_cache, k_scale, v_scale, num_pages, p, plan);
  const uint16_t* x = (const uint16_t*)qkv;
  a.q = x, a.k = x + (long)p.Hq * kHD, a.v = a.k + (long)p.Hkv * kHD;
  a.q_stride = a.k_stride = a.v_stride = (long)(p.Hq + 2 * p.Hkv) * kHD;
  a.qw = (const uint16_t*)q_norm_w, a.kw = (const uint16_t*)k_norm_w, a.inv_freq = inv_freq, a.eps = eps;
  a.q_out = (uint16_t*)q_out;
  a.write_blocks = (int)write_blocks(p);
  hipLaunchKernelGGL(kv_append_fp8_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}
