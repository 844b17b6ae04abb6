// Causal GQA attention over the 8-bit paged KV cache (kv_fp8.h) for a step that mixes prompts, chunks of them and
// single tokens (paged_plan.h): for token t of a sequence at position p, query head h and kv head h / G,
//   o = sum_{j <= p} softmax_j(scale q . K_j) V_j
// with K and V the values that the codes stand for, everything in fp32 but for two operands: the bf16 q, and
// the probabilities, rounded to bf16 (by 2^-8 at most) for the second MFMA and summed as rounded, so that the value of
// a key that dominates its row comes out exact.  The codes become bf16 exactly (v_cvt_scalef32_pk_bf16_fp8 with the
// page's power-of-two scale), so both products run on the bf16 MFMAs without a further error.
//
// Two forms, by the rows (tokens x heads of the group) that a sequence has for one kv head:
//   short: up to 16 rows (a decoding sequence), bound by the cache's bytes.  One workgroup per (sequence, kv
//     head, run of pages); its 4 waves take pairs of pages round robin, straight from HBM to the MFMA.
//   tile: more rows (prompts), bound by the MFMA and the softmax.  One workgroup per (128 or 256 rows, kv
//     head); pages are widened to bf16 once per workgroup, in LDS.
// Rows whose keys are split over several workgroups leave fp32 partial results that the merge kernel joins in key
// order, so results do not depend on timing.
#include "kv_fp8.h"
#include "paged_plan.h"

namespace {

constexpr int kHD = kKvHead;
constexpr int kPage = kPlanPage;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCachePolicyNT = 2;  // the instruction's cache-policy field: nt (streaming)
constexpr int kPadBlocks = 8;      // workgroups that clear the rows behind the last sequence
constexpr int kMergeBlocks = 512;  // for each of 16 rows, where a step has tiles.  Mostly nothing is split then: 4.6 us
                                   // for the 8192 workgroups to find that
constexpr int kMergeFew = 8;       // items of a row that one group of the merge takes alone
constexpr int kFewItems = 256;     // one per CU
constexpr float kSlack = 8.f;      // log2 of what an unnormalised probability may reach

typedef float v16f __attribute__((ext_vector_type(16)));

struct AttnFp8Args {
  const uint16_t* q;  // [T][Hq][128], rows of a token q_stride values apart
  long q_stride;
  const uint8_t *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int32_t* tables;
  const int32_t* plan;
  uint16_t* out;         // [T][Hq][128]
  float *short_o, *short_ml, *tile_o, *tile_ml;  // partial results, by item
  int num_pages;
  float scale;  // times log2(e)
  PlanLayout p;
};

// A (page, kv head) block; no page: a size of 0, so its loads read zeros and touch no memory.  Word 3 is the
// 32-bit data format (untyped loads return zeros without one).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const uint8_t* cache, int page, int Hkv, int g) {
  const long blk = page < 0 ? 0 : (long)page * Hkv + g;
  return __builtin_amdgcn_make_buffer_rsrc((void*)(cache + blk * kKvBlock), (short)0, page < 0 ? 0 : kKvBlock, 0x00020000);
}
template <int POLICY>
__device__ __forceinline__ uint4 block_load(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, POLICY));
}

// 8 codes -> 8 bf16 values times the power of two `scale`, exactly
__device__ __forceinline__ v8bf widen8(uint32_t lo, uint32_t hi, float scale) {
  const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return (v8bf){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Reductions over lanes l, l ^ 16, l ^ 32, l ^ 48, resp. l, l ^ 32 (gfx950's row and half swaps)
__device__ __forceinline__ float half_max(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float rows_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
}
__device__ __forceinline__ float rows_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// The bytes of a quad of tokens (4 codes of one dim) of which the first `live` count
__device__ __forceinline__ uint32_t quad_mask(int live) {
  return live >= 4 ? 0xffffffffu : live <= 0 ? 0u : (1u << (8 * live)) - 1u;
}

// 0xff in the bytes of 4 codes that are no finite value under the scale: NaN, and 2^128 or more.  With e the scale's
// exponent a code of exponent field f is below 2^(f - 6 + e), so the latter are those with f >= 135 - e.
__device__ __forceinline__ uint32_t not_finite4(uint32_t codes, float scale) {
  const int least = min(127, 8 * (262 - (int)((__float_as_uint(scale) >> 23) & 255)));
  const uint32_t high = ((codes & 0x7f7f7f7fu) + 0x01010101u * (uint32_t)(128 - least)) & 0x80808080u;
  return high | (high - (high >> 7));
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}

// ---------------------------------------------------------------------------
// short: S^T [16 keys x 16 rows] = K [16 x 128] Q^T (4 MFMAs 16x16x32 a page), then
// O^T [128 x 16 rows] += V^T [128 x 32 keys] P^T (8 MFMAs for two pages).  Lane l has row l & 15 throughout, and
// of its scores keys 4 (l >> 4) + i of each page, which are the 8 keys that the second MFMA wants from it.
// ---------------------------------------------------------------------------
template <int kWaves>
struct ShortLds {  // for joining the waves
  float m[kWaves][kShortRows], l[kWaves][kShortRows], o[kWaves][kShortRows][kHD + 4];
  int late[kWaves];
};

template <int kWaves>
__device__ __forceinline__ void short_item(const AttnFp8Args& a, int item, int g, ShortLds<kWaves>& lds) {
  constexpr int kThreads = 64 * kWaves;
  const PlanLayout& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int Hkv = p.Hkv, G = p.G;
  const int4* it = (const int4*)(a.plan + p.shorts + (long)PI_INTS * item);
  const int4 i0 = it[0], i1 = it[1];
  const int seq = __builtin_amdgcn_readfirstlane(i0.x), tok = __builtin_amdgcn_readfirstlane(i0.y);
  const int ntok = __builtin_amdgcn_readfirstlane(i0.z), pos = __builtin_amdgcn_readfirstlane(i0.w);
  const int page0 = __builtin_amdgcn_readfirstlane(i1.x), page1 = __builtin_amdgcn_readfirstlane(i1.y);
  const int parts = __builtin_amdgcn_readfirstlane(i1.z);
  const int rows = ntok * G;

  // Q^T operand: row lr, dims in the order in which the K block's loads bring them
  const int row_tok = lr / G, row_head = lr % G;
  v8bf qop[4];
  {
    const bool live = lr < rows;
    const uint16_t* src = a.q + (tok + (live ? row_tok : 0)) * a.q_stride + (long)(g * G + (live ? row_head : 0)) * kHD;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const uint4 v = *(const uint4*)(src + 64 * (kk >> 1) + 16 * lg + 8 * (kk & 1));
      qop[kk] = __builtin_bit_cast(v8bf, live ? v : make_uint4(0, 0, 0, 0));
    }
  }
  const int key_end = pos + row_tok + 1;  // of this lane's row

  float m_run = -INFINITY, l_run = 0.f;
  v4f o[8];  // o[4 j + d][i]: dim 64 j + 16 lg + 4 i + d of row lr
#pragma unroll
  for (int n = 0; n < 8; ++n) o[n] = (v4f){0.f, 0.f, 0.f, 0.f};

  bool late = false;  // this wave has met values that are not finite and that not every row sees
  const int32_t* table = a.tables + (long)seq * p.max_pages;
  // 32 pairs of pages at a time: lane l holds the id and the scales of page l & 1 of this wave's pair l >> 1, so
  // that a page's loads wait for no other
  for (int first = page0; first < page1; first += 64 * kWaves) {
    const int mine = first + 2 * (wave + kWaves * (lane >> 1)) + (lane & 1);
    int my_page = mine < page1 ? table[mine] : -1;
    if (my_page >= a.num_pages || my_page < 0) my_page = -1;  // a pad or a stale id: an empty page
    const long my_blk = my_page < 0 ? 0 : (long)my_page * Hkv + g;
    float my_ks = a.num_pages > 0 ? a.k_scale[my_blk] : 1.f, my_vs = a.num_pages > 0 ? a.v_scale[my_blk] : 1.f;
    if (my_page < 0) my_ks = my_vs = 1.f;  // zeros under page 0's scale, which may never have been written, could be NaN
    const int pairs = (min(page1 - first, 64 * kWaves) + 1) / 2;  // of all waves
    const int n = pairs > wave ? (pairs - wave + kWaves - 1) / kWaves : 0;

    uint4 kr[2][2], vr[2][2];
    auto page_at = [&](int i, int h) __attribute__((always_inline)) {
      return i < 32 ? __builtin_amdgcn_readlane(my_page, 2 * i + h) : -1;
    };
    auto scale_at = [&](float s, int i, int h) __attribute__((always_inline)) {
      return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s), 2 * i + h));
    };
    // issued unconditionally (a branch around loads makes the compiler wait where it joins)
    auto load = [&](uint4 (&r)[2][2], const uint8_t* cache, int i) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const __amdgpu_buffer_rsrc_t rs = block_rsrc(cache, page_at(i, h), Hkv, g);
#pragma unroll
        for (int j = 0; j < 2; ++j) r[h][j] = block_load<kCachePolicyNT>(rs, lane * 16 + j * 1024);
      }
    };
    load(kr, a.k_cache, 0);
    load(vr, a.v_cache, 0);
    for (int i = 0; i < n; ++i) {
      v4f s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float ks = scale_at(my_ks, i, h);
        s[h] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(kr[h][j].x, kr[h][j].y, ks), qop[2 * j], s[h], 0, 0, 0);
          s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(kr[h][j].z, kr[h][j].w, ks), qop[2 * j + 1], s[h], 0, 0, 0);
        }
      }
      load(kr, a.k_cache, i + 1);
      const int key0 = (first + 2 * (wave + kWaves * i)) * kPage;
      const bool all = page_at(i, 0) >= 0 && page_at(i, 1) >= 0 && key0 + 2 * kPage <= pos + 1;  // uniform
      float sv[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[h][e] = s[h][e] * a.scale;
      if (!all) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int end = page_at(i, h) < 0 ? 0 : key_end;
#pragma unroll
          for (int e = 0; e < 4; ++e) sv[h][e] = key0 + kPage * h + 4 * lg + e < end ? sv[h][e] : -INFINITY;
          // Codes behind the last key may be anything, a NaN too: zero them rather than multiply them by zero.
          const int key = key0 + kPage * h + 4 * lg;
          const uint32_t mask = quad_mask(pos + ntok - key);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            vr[h][j].x &= mask;
            vr[h][j].y &= mask;
            vr[h][j].z &= mask;
            vr[h][j].w &= mask;
          }
          // So with what is not finite among the keys that not every row sees: the rows that do get it at the end.  (A
          // single token has no such keys; one sequence of 1000 tokens, looked over like the others: 7.9 us for 7.4.)
          if (ntok > 1) {
            const uint32_t some = ~quad_mask(pos + 1 - key);
            const float vs = scale_at(my_vs, i, h);
            uint32_t drop = 0;
            auto finite = [&](uint32_t v) __attribute__((always_inline)) {
              const uint32_t x = not_finite4(v, vs) & some;
              drop |= x;
              return v & ~x;
            };
#pragma unroll
            for (int j = 0; j < 2; ++j)
              vr[h][j] = make_uint4(finite(vr[h][j].x), finite(vr[h][j].y), finite(vr[h][j].z), finite(vr[h][j].w));
            late |= __any(drop != 0);
          }
        }
      }
      float pm = fmaxf(fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[0][2], sv[0][3])),
                       fmaxf(fmaxf(sv[1][0], sv[1][1]), fmaxf(sv[1][2], sv[1][3])));
      pm = rows_max(pm);
      if (__any(pm > m_run + kSlack)) {  // as in the tile kernel
        const float m_new = fmaxf(m_run, pm);
        const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= corr;
#pragma unroll
        for (int d = 0; d < 8; ++d) o[d] *= corr;
      }
      const float m_ref = m_run == -INFINITY ? 0.f : m_run;
      v8bf pb;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const v2bf x = {(__bf16)__builtin_amdgcn_exp2f(sv[h][e] - m_ref), (__bf16)__builtin_amdgcn_exp2f(sv[h][e + 1] - m_ref)};
          pb[4 * h + e] = x[0];
          pb[4 * h + e + 1] = x[1];
          // this lane's keys, as the second product sees them; the row's lanes are summed at the end
          l_run = __builtin_amdgcn_fdot2_f32_bf16(x, (v2bf){(__bf16)1.f, (__bf16)1.f}, l_run, false);
        }
      const float vs0 = scale_at(my_vs, i, 0), vs1 = scale_at(my_vs, i, 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t v0[4] = {vr[0][j].x, vr[0][j].y, vr[0][j].z, vr[0][j].w};
        const uint32_t v1[4] = {vr[1][j].x, vr[1][j].y, vr[1][j].z, vr[1][j].w};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const v2bf w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v0[d], vs0, false);
          const v2bf w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v0[d], vs0, true);
          const v2bf w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v1[d], vs1, false);
          const v2bf w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v1[d], vs1, true);
          const v8bf va = {w0[0], w0[1], w1[0], w1[1], w2[0], w2[1], w3[0], w3[1]};
          o[4 * j + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, o[4 * j + d], 0, 0, 0);
        }
      }
      load(vr, a.v_cache, i + 1);
    }
  }
  l_run = rows_sum(l_run);

  // join the waves
  if (lg == 0) {
    lds.m[wave][lr] = m_run;
    lds.l[wave][lr] = l_run;
  }
  if (lane == 0) lds.late[wave] = late;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(v4f*)&lds.o[wave][lr][64 * j + 16 * lg + 4 * i] = (v4f){o[4 * j][i], o[4 * j + 1][i], o[4 * j + 2][i], o[4 * j + 3][i]};
  __syncthreads();
  constexpr int kDims = kShortRows * kHD / kThreads;  // of a row, a thread's
  const int r = threadIdx.x / (kHD / kDims), d0 = threadIdx.x % (kHD / kDims) * kDims;
  if (r >= rows) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, lds.m[w][r]);
  float acc[kDims], L = 0.f;
#pragma unroll
  for (int d = 0; d < kDims; ++d) acc[d] = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float wgt = lds.m[w][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lds.m[w][r] - M);
    L += lds.l[w][r] * wgt;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] += lds.o[w][r][d0 + d] * wgt;
  }
  int any_late = 0;
  if (ntok > 1)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) any_late |= lds.late[w];
  if (any_late)
    for (int key = max(pos + 1, page0 * kPage); key < min(pos + r / G + 1, page1 * kPage); ++key) {
      const int page = table[key / kPage];
      if (page < 0 || page >= a.num_pages) continue;
      const long blk = (long)page * Hkv + g;
      const float vs = a.v_scale[blk];
      const uint8_t* src = a.v_cache + blk * kKvBlock + (d0 >> 6) * 1024 + key % kPage / 4 * 256 + key % 4;
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        const uint32_t c = src[(d0 % 64 + d) * 4];
        if (not_finite4(c, vs) & 1) acc[d] += __builtin_amdgcn_cvt_f32_fp8(c, 0) * vs;
      }
    }
  if (parts == 1) {
    const float inv = M == -INFINITY ? 0.f : 1.0f / L;  // no key at all: zeros
    uint16_t* dst = a.out + ((long)(tok + r / G) * p.Hq + g * G + r % G) * kHD + d0;
#pragma unroll
    for (int d = 0; d < kDims; d += 2) *(uint32_t*)(dst + d) = pack_bf16(acc[d] * inv, acc[d + 1] * inv);
    return;
  }
  const long base = ((long)item * Hkv + g) * kShortRows + r;
  float* dst = a.short_o + base * kHD + d0;
#pragma unroll
  for (int d = 0; d < kDims; d += 2) *(float2*)(dst + d) = make_float2(acc[d], acc[d + 1]);
  if (d0 == 0) *(float2*)(a.short_ml + 2 * base) = make_float2(M, L);
}

// ---------------------------------------------------------------------------
// tile: 32 rows a wave, 4 or 8 waves, 64 keys (4 pages) a step.  S^T [32 keys x 32 rows] = K Q^T (8 MFMAs 32x32x16
// per 32 keys), O^T [128 x 32 rows] += V^T [128 x 16 keys] P^T (4 MFMAs a page).  Lane l has row l & 31 and,
// of a page's keys, 4 (l >> 5) + {0..3, 8..11}: again the 8 that the second MFMA wants from it.
// In LDS, bf16: K [dim / 8][key 64][8 dims] and V [page][quad & 1][dim slot][8 keys], quads q and q + 2 together;
// the slot 64 j + 16 d + x of dim 64 j + 4 x + d makes the writes contiguous.  Every read and write of 16
// bytes is contiguous over the lanes that the LDS serves together.
// ---------------------------------------------------------------------------

// Schedules a step's half so far as 16 MFMAs with four vector instructions behind each, the LDS reads two MFMAs
// ahead of their use.  (8192 tokens, 64 / 4 heads: the compiler's own order 1120 us, one read ahead 1100, two 1067,
// four 1070, eight 1082; three to seven vector instructions within 1%.)
#define MIX_MFMAS()                                                            \
  do {                                                                         \
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                         \
    _Pragma("unroll") for (int _i = 0; _i < 16; ++_i) {                        \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                       \
      if (_i + 2 < 16) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      \
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);                       \
    }                                                                          \
  } while (0)

// Steps whose K and V are in LDS.  Two: a barrier after each step, and room for two workgroups in a CU.  Four, where
// the registers leave room for one only: a barrier after two steps.
constexpr int tile_ring(int waves) { return waves == 4 ? 2 : 4; }

template <int kWaves>
struct TileLds {
  struct {
    uint4 k[kHD / 8][kTileKeys], v[kTilePages][2][kHD];
  } step[tile_ring(kWaves)];
  int late[kWaves];
};

template <int kWaves>
__device__ __forceinline__ void tile_item(const AttnFp8Args& a, int item, int g, TileLds<kWaves>& lds) {
  constexpr int kTileRows = 32 * kWaves;
  constexpr int kRing = tile_ring(kWaves);
  constexpr int kAheadK = kRing == 4 ? 3 : 2, kAheadV = kAheadK - 1;  // steps from storing to use
  constexpr int kLoads = 8 / kWaves;  // 16-byte pieces of a step's K, and 8-byte ones of a quad of V, for each thread
  const PlanLayout& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, kg = lane >> 5;
  const int Hkv = p.Hkv, G = p.G;
  const int4* it = (const int4*)(a.plan + p.tiles + (long)PI_INTS * item);
  const int4 i0 = it[0], i1 = it[1];
  const int seq = __builtin_amdgcn_readfirstlane(i0.x), tok = __builtin_amdgcn_readfirstlane(i0.y);
  const int ntok = __builtin_amdgcn_readfirstlane(i0.z), pos = __builtin_amdgcn_readfirstlane(i0.w);
  const int page0 = __builtin_amdgcn_readfirstlane(i1.x), page1 = __builtin_amdgcn_readfirstlane(i1.y);
  const int parts = __builtin_amdgcn_readfirstlane(i1.z);

  const int r = 32 * wave + lr;
  const bool live = r < ntok * G;
  const int row_tok = min(r / G, ntok - 1);
  const long row = (long)(tok + row_tok);
  v8bf qop[8];
  {
    const uint16_t* src = a.q + row * a.q_stride + (long)(g * G + r % G) * kHD + 8 * kg;
#pragma unroll
    for (int s = 0; s < 8; ++s) qop[s] = __builtin_bit_cast(v8bf, *(const uint4*)(src + 16 * s));
  }
  const int key_end = pos + row_tok + 1;                       // of this lane's row
  const int all_end = pos + min(32 * wave / G, ntok - 1) + 1;  // keys that every row of the wave sees

  float m_ref = -INFINITY, l_run = 0.f;
  v16f o[4];  // o[db][i]: dim slot 32 db + 8 (i / 4) + 4 kg + i % 4 of row lr
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  // Page ids and scales, 64 pages (16 steps) at a time, one a lane; the next 64 are fetched two steps ahead.
  const int32_t* table = a.tables + (long)seq * p.max_pages;
  int my_page, next_page = -1;
  float my_ks, my_vs, next_ks = 1.f, next_vs = 1.f;
  auto fetch_ids = [&](int first) __attribute__((always_inline)) {
    const int mine = first + lane;
    next_page = mine < page1 ? table[mine] : -1;
  };
  auto fetch_scales = [&]() __attribute__((always_inline)) {
    if (next_page >= a.num_pages || next_page < 0) next_page = -1;  // a pad or a stale id: an empty page
    const long blk = next_page < 0 ? 0 : (long)next_page * Hkv + g;
    next_ks = a.num_pages > 0 ? a.k_scale[blk] : 1.f;
    next_vs = a.num_pages > 0 ? a.v_scale[blk] : 1.f;
    if (next_page < 0) next_ks = next_vs = 1.f;  // not page 0's, which may never have been written
  };
  auto lane_f = [&](float x, int l) __attribute__((always_inline)) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), l));
  };
  // This thread's codes of a step.  K: 16 bytes (16 dims of a token) of kLoads pages.  V: of one page the quads vq
  // and vq + 2 of 2 kLoads dims.  K runs a step ahead of V.
  uint4 kr[kLoads];
  uint32_t vr[2][2 * kLoads];
  float ks[kLoads], vs = 1.f, vs_next = 1.f;
  int v_page = -1;      // of the step that K was last loaded for
  uint32_t held = 0;    // which of that step's pages there are
  const int k_page = wave >> 1, k_part = wave & 1;  // the first of the K pages (2 apart), the half of a block
  const int v_at = wave * kTilePages / kWaves;      // the V page
  // four waves: a lane has dims 64 vj + 4 vx .. +4; eight: of those two, 2 vd .. +2
  const int vj = kWaves == 4 ? lane >> 5 : wave & 1, vd = kWaves == 4 ? 0 : lane >> 5, vq = (lane >> 4) & 1, vx = lane & 15;
  auto load_k = [&](int step) __attribute__((always_inline)) {
    const int l = (step & 15) * kTilePages;
    if (l == 0) {
      my_page = next_page;
      my_ks = next_ks;
      my_vs = next_vs;
    }
    if ((step & 15) == 13) fetch_ids(page0 + (step + 3) * kTilePages);
    if ((step & 15) == 14) fetch_scales();
    held = (uint32_t)(__ballot(my_page >= 0) >> l) & 15u;
    v_page = __builtin_amdgcn_readlane(my_page, l + v_at);
    vs_next = lane_f(my_vs, l + v_at);
#pragma unroll
    for (int h = 0; h < kLoads; ++h) {
      const int at = l + 2 * h + k_page;
      ks[h] = lane_f(my_ks, at);
      kr[h] = block_load<0>(block_rsrc(a.k_cache, __builtin_amdgcn_readlane(my_page, at), Hkv, g), k_part * 1024 + lane * 16);
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {  // of the step that K was last loaded for
    const __amdgpu_buffer_rsrc_t rv = block_rsrc(a.v_cache, v_page, Hkv, g);
    vs = vs_next;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = vj * 1024 + (vq + 2 * h) * 256 + vx * 16 + vd * 8;
      if constexpr (kWaves == 4) {
        const uint4 x = block_load<0>(rv, at);
        vr[h][0] = x.x, vr[h][1] = x.y, vr[h][2] = x.z, vr[h][3] = x.w;
      } else {
        const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rv, at, 0, 0));
        vr[h][0] = x.x, vr[h][1] = x.y;
      }
    }
  };
  auto store_k = [&](int buf) __attribute__((always_inline)) {
    const int c = 4 * k_part + (lane >> 4);  // dims 16 c .. +16 of token lane & 15
#pragma unroll
    for (int h = 0; h < kLoads; ++h) {
      const int key = (2 * h + k_page) * kPage + (lane & 15);
      lds.step[buf].k[2 * c][key] = __builtin_bit_cast(uint4, widen8(kr[h].x, kr[h].y, ks[h]));
      lds.step[buf].k[2 * c + 1][key] = __builtin_bit_cast(uint4, widen8(kr[h].z, kr[h].w, ks[h]));
    }
  };
  // Codes behind the last key may be anything, a NaN too: zeros.  So with what is not finite among the keys that not
  // every row sees, for a zero probability times it is no zero: the rows that do see it get it at the end.  A barrier
  // lies between a step's staging and its use, so also between this wave's note and the end.
  if (lane == 0) lds.late[wave] = 0;
  auto mask_v = [&](int page) __attribute__((always_inline)) {
    uint32_t drop = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = (page + v_at) * kPage + 4 * (vq + 2 * h);
      const uint32_t mask = quad_mask(pos + ntok - key), some = ~quad_mask(pos + 1 - key);
#pragma unroll
      for (int d = 0; d < 2 * kLoads; ++d) {
        vr[h][d] &= mask;
        const uint32_t x = not_finite4(vr[h][d], vs) & some;
        vr[h][d] &= ~x;
        drop |= x;
      }
    }
    if (__any(drop != 0) && lane == 0) lds.late[wave] = 1;
  };
  auto store_v = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < 2 * kLoads; ++d)
      lds.step[buf].v[v_at][vq][64 * vj + 16 * (2 * vd + d) + vx] = __builtin_bit_cast(uint4, widen8(vr[0][d], vr[1][d], vs));
  };
  auto scores = [&](v16f (&s)[2], int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, lds.step[buf].k[2 * k + kg][32 * b + lr]), qop[k], s[b],
                                                       0, 0, 0);
  };
  auto mask_scores = [&](v16f (&s)[2], int key0, uint32_t there) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 32 * b + 8 * (i >> 2) + 4 * kg + (i & 3);
        const bool ok = key < key_end && ((there >> (2 * b + (i >> 3))) & 1);
        s[b][i] = ok ? s[b][i] : -INFINITY;
      }
  };
  auto score_max = [&](const v16f (&s)[2]) __attribute__((always_inline)) {
    float x = s[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) x = fmaxf(x, s[0][i]);
#pragma unroll
    for (int i = 0; i < 16; ++i) x = fmaxf(x, s[1][i]);
    return x;
  };
  // 32 keys' probabilities, and their sum as the second product will see them
  auto probabilities = [&](const v16f& s, v8bf (&pb)[2], float m) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const v2bf x = {(__bf16)__builtin_amdgcn_exp2f(fmaf(s[i], a.scale, -m)),
                      (__bf16)__builtin_amdgcn_exp2f(fmaf(s[i + 1], a.scale, -m))};
      pb[i >> 3][i & 7] = x[0];
      pb[i >> 3][(i & 7) + 1] = x[1];
      l_run = __builtin_amdgcn_fdot2_f32_bf16(x, (v2bf){(__bf16)1.f, (__bf16)1.f}, l_run, false);
    }
  };
  auto output = [&](const v8bf (&pb)[2], int buf, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < 4; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, lds.step[buf].v[2 * half + h][kg][32 * d + lr]), pb[h],
                                                       o[d], 0, 0, 0);
  };

  // Step n's scores are formed in the course of step n - 1, beside its softmax, so that the wave has MFMAs and vector
  // work at the same time: K of step n + kAheadK and V of step n + kAheadV go into LDS during step n.
  const int steps = (page1 - page0 + kTilePages - 1) / kTilePages;
  v16f s0[2], s1[2];
  float pm;
  uint32_t queue = 0;  // the held pages of the steps from n + 1 to that which K was last loaded for, 4 bits each
  auto step = [&](v16f (&s)[2], v16f (&next)[2], int n, int buf) __attribute__((always_inline)) {
    const int next_key = (page0 + (n + 1) * kTilePages) * kPage;
    const uint32_t held_next = queue & 15;
    load_v();  // step n + kAheadV
    load_k(n + kAheadK);
    queue = (queue >> 4) | (held << (4 * (kAheadK - 2)));
    // A row's reference need not be its maximum: only where a score passes it by more than 2^kSlack are the sums
    // scaled down (exp stays below 2^kSlack, and bf16 and fp32 are as exact there as below 1)
    pm = half_max(pm) * a.scale;
    if (__any(pm > m_ref + kSlack)) {
      const float m_new = fmaxf(m_ref, pm);
      const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_new);
      m_ref = m_new;
      l_run *= corr;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= corr;
    }
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
    v8bf pa[2], pb[2];
    scores(next, (buf + 1) % kRing);
    probabilities(s[0], pa, m_use);
    MIX_MFMAS();
    asm volatile("" : "+v"(pa[0]), "+v"(pa[1]), "+v"(l_run));  // not to be put off past the branches
    if (next_key + kTileKeys > all_end || held_next != 15) mask_scores(next, next_key, held_next);
    const int v_page0 = page0 + (n + kAheadV) * kTilePages;
    if ((v_page0 + kTilePages) * kPage > pos + 1) mask_v(v_page0);
    output(pa, buf, 0);
    probabilities(s[1], pb, m_use);
    output(pb, buf, 1);
    pm = score_max(next);
    store_v((buf + kAheadV) % kRing);
    store_k((buf + kAheadK) % kRing);
    MIX_MFMAS();
    if (kRing == 2 || buf % 2 == 1) __syncthreads();
  };
  fetch_ids(page0);
  fetch_scales();
  uint32_t held0 = 0;
#pragma unroll
  for (int n = 0; n < kAheadK; ++n) {
    load_k(n);
    store_k(n);
    if (n == 0) held0 = held;
    if (n > 0) queue |= held << (4 * (n - 1));
    if (n < kAheadV) {
      load_v();
      const int v_page0 = page0 + n * kTilePages;
      if ((v_page0 + kTilePages) * kPage > pos + 1) mask_v(v_page0);
      store_v(n);
    }
  }
  __syncthreads();
  scores(s0, 0);
  if (page0 * kPage + kTileKeys > all_end || held0 != 15) mask_scores(s0, page0 * kPage, held0);
  pm = score_max(s0);
  __syncthreads();  // every wave has read the first step's K, whose place a later step's K takes before the next barrier
  for (int n = 0; n < steps; n += kRing) {
    step(s0, s1, n, 0);
    if (n + 1 >= steps) break;
    step(s1, s0, n + 1, 1);
    if constexpr (kRing == 4) {
      if (n + 2 >= steps) break;
      step(s0, s1, n + 2, 2);
      if (n + 3 >= steps) break;
      step(s1, s0, n + 3, 3);
    }
  }
  const float m_run = m_ref;
  l_run = half_sum(l_run);
  if (page1 * kPage > pos + 1) {  // some of the item's keys are not every row's
    int any_late = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) any_late |= lds.late[w];
    const int end = any_late ? min(key_end, page1 * kPage) : 0;
#pragma unroll 1
    for (int key = max(pos + 1, page0 * kPage); key < end; ++key) {
      const int page = table[key / kPage];
      if (page < 0 || page >= a.num_pages) continue;
      const long blk = (long)page * Hkv + g;
      const float scale = a.v_scale[blk];
      const uint8_t* src = a.v_cache + blk * kKvBlock + key % kPage / 4 * 256 + 16 * 4 * kg;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = 8 * (i >> 2) + (i & 3);  // dims 64 j + 4 (x + 4 kg) .. +4
          const uint4 c = *(const uint4*)(src + j * 1024 + 16 * x);
          const uint32_t code[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const uint32_t u = code[d] >> 8 * (key % 4);
            const float add = not_finite4(u, scale) & 1 ? __builtin_amdgcn_cvt_f32_fp8(u, 0) * scale : 0.f;
            o[2 * j + (d >> 1)][i + 8 * (d & 1)] += add;
          }
        }
    }
  }
  if (!live) return;
  if (parts == 1) {
    const float inv = m_run == -INFINITY ? 0.f : 1.0f / l_run;  // no key at all: zeros
    uint16_t* dst = a.out + (row * p.Hq + g * G + r % G) * kHD;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = 8 * (i >> 2) + 4 * kg + (i & 3);
        *(uint2*)(dst + 64 * j + 4 * x) = make_uint2(pack_bf16(o[2 * j][i] * inv, o[2 * j][i + 8] * inv),
                                                     pack_bf16(o[2 * j + 1][i] * inv, o[2 * j + 1][i + 8] * inv));
      }
    return;
  }
  const long base = ((long)item * Hkv + g) * kTileRows + r;
  float* dst = a.tile_o + base * kHD;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = 8 * (i >> 2) + 4 * kg + (i & 3);
      *(float4*)(dst + 64 * j + 4 * x) = make_float4(o[2 * j][i], o[2 * j][i + 8], o[2 * j + 1][i], o[2 * j + 1][i + 8]);
    }
  if (kg == 0) *(float2*)(a.tile_ml + 2 * base) = make_float2(m_run, l_run);
}

// ---------------------------------------------------------------------------
// The launches.  A step of short sequences alone is the short kernel's.  Any other is the step kernel's, which takes
// both kinds, the tiles first, so that its short items fill the CUs that the last tiles leave (2048 tokens of a prompt
// and 63 decoding sequences 172 -> 160 us, 64 and 64 84 -> 59, 100 tokens alone 13.6 -> 11.2 against two launches; both
// kinds side by side from the start: 170, 71 and 10.7).  Workgroups that follow each other go to different XCDs (8), so
// with 1, 2, 4 or 8 kv heads a tile's XCD sees few heads of the cache.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void clear_padding(const AttnFp8Args& a, int block) {  // rows behind the last sequence: zeros
  const long row = (long)a.p.Hq * kHD / 8;  // 16-byte pieces of a token
  const long end = a.p.T * row;
  for (long i = a.plan[PH_TOKENS] * row + (long)block * blockDim.x + threadIdx.x; i < end; i += (long)kPadBlocks * blockDim.x)
    ((uint4*)a.out)[i] = make_uint4(0, 0, 0, 0);
}

template <int kWaves>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(4))) void attn_fp8_short_kernel(AttnFp8Args a) {
  __shared__ __attribute__((aligned(16))) ShortLds<kWaves> lds;
  const int items = a.p.S * a.p.Hkv;
  if ((int)blockIdx.x >= items) return clear_padding(a, (int)blockIdx.x - items);
  const int item = blockIdx.x / a.p.Hkv;
  if (item < a.plan[PH_SHORTS]) short_item<kWaves>(a, item, blockIdx.x % a.p.Hkv, lds);
}

template <int kWaves>
__global__ __launch_bounds__(64 * kWaves, 2) void attn_fp8_step_kernel(AttnFp8Args a) {
  __shared__ __attribute__((aligned(16))) union {
    ShortLds<kWaves> s;
    TileLds<kWaves> t;
  } lds;
  const int Hkv = a.p.Hkv, items = (a.p.S + a.p.N) * Hkv, i = blockIdx.x;
  if (i >= items) return clear_padding(a, i - items);
  const int tiles = a.plan[PH_TILES] * Hkv, shorts = a.plan[PH_SHORTS] * Hkv;
  if (i < tiles)
    tile_item<kWaves>(a, i / Hkv, i % Hkv, lds.t);
  else if (i < tiles + shorts)
    short_item<kWaves>(a, (i - tiles) / Hkv, (i - tiles) % Hkv, lds.s);
}

// ---------------------------------------------------------------------------
// merge: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a row's items, in key order, a lane of 32 with 4 dims.
// Up to kMergeFew items: the 8 groups of 32 lanes take a row each.  More: they share a row's items.  Either way a
// group has four items' loads in flight.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void attn_fp8_merge_kernel(AttnFp8Args a) {
  const PlanLayout& p = a.p;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  __shared__ float s_m[8], s_l[8];
  __shared__ __attribute__((aligned(16))) v4f s_o[8][32];
  const int tile_chunks = p.tile_rows / kShortRows;  // of a tile's rows
  const int shorts = a.plan[PH_SHORT_MERGES], chunks = shorts + a.plan[PH_TILE_MERGES] * tile_chunks;
  for (int x = blockIdx.x; x < chunks * p.Hkv; x += gridDim.x) {  // workgroup-uniform
    const int chunk = x / p.Hkv, g = x % p.Hkv;
    const bool tile = chunk >= shorts;
    const int r0 = blockIdx.y + (tile ? (chunk - shorts) % tile_chunks * kShortRows : 0);
    const int4 e = *(const int4*)(a.plan + (tile ? p.tile_merges + 4L * ((chunk - shorts) / tile_chunks) : p.short_merges + 4L * chunk));
    const int ns = e.x;
    const bool few = ns <= kMergeFew;
    if (r0 >= e.w * p.G || (few && r0 % 8 != 0)) continue;
    const int r = few ? r0 + grp : r0;
    const bool live = r < e.w * p.G;
    const float* part = tile ? a.tile_o : a.short_o;
    const float* ml = tile ? a.tile_ml : a.short_ml;
    float M = -INFINITY, L = 0.f;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    const int by = few ? 1 : 8;
    for (int s0 = few ? 0 : grp; s0 < ns; s0 += 4 * by) {
      float2 x[4];
      v4f v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = min(s0 + by * u, ns - 1);
        const long base = ((long)(e.y + s) * p.Hkv + g) * (tile ? p.tile_rows : kShortRows) + (live ? r : r0);
        x[u] = *(const float2*)(ml + 2 * base);
        v[u] = *(const v4f*)(part + base * kHD + 4 * lane);
      }
      float m_new = M;
#pragma unroll
      for (int u = 0; u < 4; ++u) m_new = fmaxf(m_new, x[u].x);  // the last item again changes nothing
      // Without a maximum, an item has only empty pages and zeros, or only NaN: either is added with weight 0, which
      // leaves the one nothing and the other NaN.
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float old = __builtin_amdgcn_exp2f(M - m_use);
      M = m_new;
      L *= old;
      acc *= old;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = s0 + by * u < ns ? __builtin_amdgcn_exp2f(x[u].x - m_use) : 0.f;
        L += x[u].y * w;
        acc += v[u] * w;
      }
    }
    if (!few) {
      s_o[grp][lane] = acc;
      if (lane == 0) {
        s_m[grp] = M;
        s_l[grp] = L;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) M = fmaxf(M, s_m[k]);
      L = 0.f;
      acc = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = s_m[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[k] - M);
        L += s_l[k] * w;
        acc += s_o[k][lane] * w;
      }
      __syncthreads();  // the sums are read
    }
    if (few ? live : grp == 0) {
      const float inv = M == -INFINITY ? 0.f : 1.0f / L;
      uint16_t* dst = a.out + ((long)(e.z + r / p.G) * p.Hq + g * p.G + r % p.G) * kHD + 4 * lane;
      *(uint2*)dst = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
    }
  }
}

// Partial results: an item's rows and their (max, sum), for both kinds; none where no item is split.
struct Parts {
  long shorts, tiles;  // rows
};
Parts attn_parts(const PlanLayout& p) {
  return {p.short_whole ? 0 : (long)p.S * p.Hkv * kShortRows,
          (long)p.max_pages * kPage >= 2 * kTileMinKeys ? (long)p.split_tiles * p.Hkv * p.tile_rows : 0};
}

void attn_carve(WsCarver& c, const Parts& n, AttnFp8Args* a) {
  a->short_o = c.take<float>(n.shorts * kHD);
  a->short_ml = c.take<float>(n.shorts * 2);
  a->tile_o = c.take<float>(n.tiles * kHD);
  a->tile_ml = c.take<float>(n.tiles * 2);
}

bool attn_grid_ok(const PlanLayout& p) {
  return moe_grid_fits((long)(p.S + p.N) * p.Hkv + kPadBlocks) &&
         moe_grid_fits((long)(p.SM + p.TM) * p.Hkv);
}

}  // namespace

extern "C" size_t moe_mi355x_paged_attn_fp8_workspace_bytes(const moe_mi355x_plan_shape* shape) {
  if (!plan_shape_ok(shape)) return 0;
  const PlanLayout p = plan_layout(shape);
  if (!attn_grid_ok(p)) return 0;
  WsCarver c(nullptr);
  AttnFp8Args a{};
  attn_carve(c, attn_parts(p), &a);
  return moe_align_up(c.off, 256);
}

extern "C" int moe_mi355x_paged_attn_fp8(const void* q, long long q_stride, const void* k_cache, const void* v_cache,
                                         const float* k_scale, const float* v_scale, const int32_t* block_tables,
                                         int head_dim, int page_size, int num_pages, float scale,
                                         const moe_mi355x_plan_shape* shape, const void* plan, void* out,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  MOE_RETURN_IF(!plan_shape_ok(shape) || head_dim != kHD || page_size != kPage || num_pages < 0, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(!(scale > 0.f) || !(scale * kLog2e < INFINITY), MOE_ERR_INVALID_ARG);
  if (shape->tokens == 0) return MOE_OK;
  MOE_RETURN_IF(!q || !k_cache || !v_cache || !k_scale || !v_scale || !plan || !out, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(shape->seqs > 0 && !block_tables, MOE_ERR_INVALID_ARG);
  const PlanLayout p = plan_layout(shape);
  MOE_RETURN_IF(!attn_grid_ok(p) || q_stride < (long)p.Hq * kHD, MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF(q_stride % 8 || !moe_aligned16(q) || !moe_aligned16(k_cache) || !moe_aligned16(v_cache) ||
                    !moe_aligned16(plan) || !moe_aligned16(out),
                MOE_ERR_ALIGNMENT);
  const size_t need = moe_mi355x_paged_attn_fp8_workspace_bytes(shape);
  MOE_RETURN_IF(need > 0 && (!workspace || workspace_bytes < need), MOE_ERR_WORKSPACE);
  AttnFp8Args a{};
  a.q = (const uint16_t*)q, a.q_stride = q_stride;
  a.k_cache = (const uint8_t*)k_cache, a.v_cache = (const uint8_t*)v_cache, a.k_scale = k_scale, a.v_scale = v_scale;
  a.tables = block_tables, a.plan = (const int32_t*)plan, a.out = (uint16_t*)out;
  a.num_pages = num_pages, a.scale = scale * kLog2e, a.p = p;
  const Parts parts = attn_parts(p);
  WsCarver c(workspace);
  attn_carve(c, parts, &a);
  hipStream_t s = (hipStream_t)stream;
  if (p.N > 0) {
    const dim3 grid((unsigned)((p.N + p.S) * p.Hkv + kPadBlocks));
    if (p.tile_rows == kTileRowsMany)
      hipLaunchKernelGGL(attn_fp8_step_kernel<8>, grid, dim3(512), 0, s, a);
    else
      hipLaunchKernelGGL(attn_fp8_step_kernel<4>, grid, dim3(256), 0, s, a);
    MOE_CHECK_LAUNCH();
  } else {
    const dim3 grid((unsigned)(p.S * p.Hkv + kPadBlocks));
    // Whole sequences, and no more of them than CUs: 8 waves each, of up to eight pairs of pages.  (One sequence of 1000
    // tokens, in a graph: 4 waves 9.1 us, 8 waves 7.5, 16 waves 8.3; two to four pairs in flight per wave 7.9 to 8.6,
    // for the code that has to be fetched.)
    if (p.short_whole && p.S * p.Hkv <= kFewItems)
      hipLaunchKernelGGL(attn_fp8_short_kernel<8>, grid, dim3(512), 0, s, a);
    else
      hipLaunchKernelGGL(attn_fp8_short_kernel<4>, grid, dim3(256), 0, s, a);
    MOE_CHECK_LAUNCH();
  }
  if (parts.shorts + parts.tiles > 0 && p.SM > 0) {
    // with tiles among them mostly nothing is split: fewer workgroups, that come back for more
    const long x = (long)(p.SM + p.TM) * p.Hkv;
    hipLaunchKernelGGL(attn_fp8_merge_kernel, dim3(parts.tiles > 0 && x > kMergeBlocks ? kMergeBlocks : x, p.short_rows), dim3(256),
                       0, s, a);
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}
