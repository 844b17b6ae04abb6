// Log probabilities of given tokens, entropy and the most likely tokens of rows of logits (the softmax that ends a
// step, beside the router's in route.hip): for row x[0 .. V) and token g,
//   m = max x, Z = sum e^(x - m)      logprob = x[g] - m - ln Z      entropy = ln Z - (1 / Z) sum e^(x - m) (x - m)
// and the k largest by (value, lower index first) with their logprobs.
//
// One pass over the logits, bound by their bytes and, for bf16, nearly by the vector unit (an exponential takes four
// of the nine and a half issue slots that a value costs).  A wave keeps a reference near its maximum instead of the
// maximum: the sums are scaled only where a value passes it by 2^8, which after the first values happens rarely.
//
// The largest are found on the way.  The maxima of the 16-byte vectors are kept in LDS and looked through a batch of turns at a
// time, the last batch at the end.  The lanes' running maxima give a bound: where j of the lanes of each of c rows of 16 lanes have
// seen a value of at least b, with c j >= k, the k largest are all >= b.  Vectors that reach it are candidates; those that
// do so at the end are read again, and their values that reach it sorted by counting.  What only equals the bound (the value that
// a mask has left nearly everywhere, say) is taken up to the k-th in the order of the row; -inf not at all, for where fewer
// than k values are above it the first of the rest are at the row's start.
//
// Few rows are split over workgroups, whose sums and lists a second kernel joins.  Rows with NaN or +inf, whose maximum is
// of a size past 7 * 10^5 (the type's lowest everywhere, say) or with more candidates than there is room for (values that rise
// along the row) are gone over again by a plainer scan.
//
// (151936 bf16 values a row, in a graph: one row with 5 alternatives 8.4 us, 64 with 20 15.4; 6000 rows without 317, 5.75
// TB/s.  777 fp32 rows of 50257 with 8 36.3, 4.3 TB/s: all start and end together, with nothing to load at either end.  777
// bf16 rows with 5 alternatives: 59 us, 4.0 TB/s, and with all but 10 tokens masked by -inf 58.5, by -10^9 67; before equals and far
// parts were told apart, 289 and 282, on the same logits again and again.)
#include "common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / MOE_WAVE;
constexpr int kMaxTop = 64;
constexpr int kMaxV = 1 << 30;  // places in a row, and a little past it, are ints
constexpr int kPer = 2;        // vectors of a lane's turn (4: 777 fp32 rows level, one row with 5 alternatives 9.4 -> 10.0 us)
constexpr int kTurn = kPer * kThreads;
constexpr int kBatch = 16;     // vectors of a lane whose maxima are looked through together
constexpr int kBatchTurns = kBatch / kPer;
constexpr int kCand = 192;     // vectors that a wave keeps as candidates (128 or 256: 777 rows with 5 alternatives 1% more)
constexpr int kBuf = 512;      // values that it does in the plain scan
constexpr int kKeep = 128;     // ... after they are cut down, at most
// Candidates that are taken without a look for those that only equal the bound.  (16: 64 rows with 20 alternatives 15.7 -> 16.8 us,
// 256 rows 25.5 -> 27.6; 96: level, but 777 rows masked by -10^9 67 -> 161.)
constexpr int kFewCand = 48;
constexpr int kFewLanes = 12;  // lanes with values for the list that are (4 or 32: level, the masked rows 67 -> 68)
constexpr int kBoundRows = kThreads / 16;
constexpr int kList = kWaves * kKeep;  // ... and a workgroup at the end
constexpr int kMaxSplits = 64;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 5.5f;  // 8 ln 2: what a value may be above the reference
constexpr float kFar = 1 << 20;  // a reference up to here, times log2(e), is off by 2^-5 at most, which is undone exactly
constexpr float kFarSlack = 300.f;  // log2 of what weighs nothing next to a maximum within kFar of zero
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kNoTerm = -200.f;  // log2 of a term that is zero in fp32, in the place of -inf times zero

struct LpArgs {
  const void* x;  // [T][V], rows `stride` values apart
  long stride;
  const void* tokens;  // [T] or null
  int id_bytes;
  int T, V, k, splits;
  float *logprobs, *entropy;  // [T]
  int64_t* top_ids;           // [T][k]
  float* top_logprobs;        // [T][k]
  float4* sums;               // [T][splits] {m, s, t, -}
  uint64_t* keys;             // [T][splits][k]
};

// Values as whole numbers of the same order; -0 as 0, NaN above all.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = x != x ? 0x7fc00000u : __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o ^ ((uint32_t)((int)~o >> 31) | 0x80000000u));
}
// The larger the better: the value, then the lower index.  No key of a value is 0.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  return (uint64_t)ordered(x) << 32 | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ float value_of(uint64_t key) { return from_ordered((uint32_t)(key >> 32)); }

__device__ __forceinline__ void unpack(uint4 r, float (&v)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(uint4 r, float (&v)[4]) {
  v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ float value_at(const uint16_t* x, long i) { return bf16_to_f32(x[i]); }
__device__ __forceinline__ float value_at(const float* x, long i) { return x[i]; }

// s = sum 2^((x - m) log2 e), t = sum of each times its exponent, for one reference m
struct Sums {
  float m, s, t;
};
// b's sums added to a's, under the larger reference (-inf: no value yet)
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  auto under = [&](Sums v) {
    const float d = v.m == m ? 0.f : fmaxf((v.m - m) * kLog2e, kNoTerm);
    const float c = v.m == m ? 1.f : __builtin_amdgcn_exp2f((v.m - m) * kLog2e);
    return Sums{m, v.s * c, fmaf(v.s, d, v.t) * c};
  };
  const Sums x = under(a), y = under(b);
  return Sums{m, x.s + y.s, x.t + y.t};
}
// ... over a wave, as its first lane has it (lanes differ in which of two sums the compiler's fused product takes)
__device__ __forceinline__ Sums join_wave(Sums v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = join(v, Sums{__shfl_xor(v.m, d), __shfl_xor(v.s, d), __shfl_xor(v.t, d)});
  auto first = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };
  return Sums{first(v.m), first(v.s), first(v.t)};
}

// From a row's sums to its results
struct Row {
  double m, ln_z;
  float entropy;
};
__device__ __forceinline__ Row row_of(Sums v) {
  const float m = v.m == -INFINITY ? 0.f : v.m;
  const double ln_z = log((double)v.s), entropy = ln_z - 0.69314718055994530942 * ((double)v.t / (double)v.s);
  return Row{(double)m, ln_z, entropy < 0. ? 0.f : (float)entropy};
}
__device__ __forceinline__ float logprob(const Row& r, float x) { return (float)((double)x - r.m - r.ln_z); }

// A row's given token, asked for at a kernel's start: at its end the number and then the value would each be a wait for
// memory (64 rows with 20 alternatives 16.9 -> 16.5 us).
struct Given {
  int64_t token;
  float x;
};
template <typename E>
__device__ __forceinline__ Given given_of(const LpArgs& a, int row) {
  Given g{-1, 0.f};
  if (a.tokens) {
    g.token = a.id_bytes == 8 ? ((const int64_t*)a.tokens)[row] : ((const int32_t*)a.tokens)[row];
    g.x = value_at((const E*)a.x + row * a.stride, g.token < 0 || g.token >= a.V ? 0 : g.token);
  }
  return g;
}
// Entropy and the given token's logprob, by one thread
__device__ __forceinline__ void finish(const LpArgs& a, int row, const Row& r, const Given& g) {
  a.entropy[row] = r.entropy;
  if (a.tokens) a.logprobs[row] = g.token < 0 ? 0.f : g.token < a.V ? logprob(r, g.x) : NAN;
}

template <int D>
__device__ __forceinline__ float ror(float v) {
  return __uint_as_float(row_ror<D>(__float_as_uint(v)));
}
// of the D next lanes of the 16 those with more
template <int D>
__device__ __forceinline__ void count_more(float mine, int& more) {
  more += ror<D>(mine) > mine;
  if constexpr (D > 1) count_more<D - 1>(mine, more);
}

// A bound that at least n of the wave's 64 values reach, close to the n-th largest: down from the largest by growing steps,
// of 1/32 of a binade at first, then the last one in 16 parts.  Some thresholds at a time, for each is a wait of the scalar unit
// for the vector unit and back.
__device__ __forceinline__ uint32_t bound_of(uint32_t mine, int n) {
  const uint32_t most = wave_max_u32_uniform(mine);
  auto reached = [&](uint32_t b) __attribute__((always_inline)) { return __popcll(__ballot(mine >= b)) >= n; };
  auto below = [&](uint32_t by) __attribute__((always_inline)) { return most > by ? most - by : 0; };  // 0 is reached by all
  uint32_t lo = most, step = 1u << 18, from = 0, width = 0;
#pragma unroll 1
  while (!reached(lo)) {
    const uint32_t a = below(from + step), b = below(from + 3 * step), c = below(from + 7 * step), d = below(from + 15 * step);
    const bool ra = reached(a), rb = reached(b), rc = reached(c);
    lo = ra ? a : rb ? b : rc ? c : d;
    width = ra ? step : rb ? 2 * step : rc ? 4 * step : 8 * step;
    from += 15 * step;
    step *= 16;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    width /= 4;
    const uint32_t a = lo + width, b = a + width, c = b + width;
    const bool ra = reached(a), rb = reached(b), rc = reached(c);
    lo = rc ? c : rb ? b : ra ? a : lo;
  }
  return ~wave_max_u32_uniform(mine >= lo ? ~mine : 0);  // the least of them, so that what only equals it is known
}

struct TopLds {
  union {
    float most[kBatchTurns][kThreads][kPer];  // maxima of a batch's vectors
    uint64_t buf[kWaves][kBuf];
  };
  uint64_t cand[kWaves][kCand];
  uint64_t list[kList + 4];  // of all waves, at the end
  float bound[kBoundRows];  // of 16 lanes each
  int n_list;
};

// A wave's candidates in the plain scan
struct Top {
  uint64_t* buf;
  int count;       // wave-uniform
  uint64_t least;  // keys below are not among the k largest; wave-uniform
};

// There is room for 64 more.
__device__ __forceinline__ void offer(Top& t, float x, int index, bool valid) {
  const uint64_t key = key_of(x, index);
  const bool pass = valid && key >= t.least;
  const uint64_t mask = __ballot(pass);
  if (pass) t.buf[t.count + __popcll(mask & lanemask_lt())] = key;
  t.count += __popcll(mask);
}

// Cuts the candidates down to between k and kKeep (all k of those from `least` on where they are fewer).
__device__ __forceinline__ void cut(Top& t, int k, int lane) {
  constexpr int kPer = kBuf / MOE_WAVE;
  uint64_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = i * MOE_WAVE + lane;
    key[i] = at < t.count ? t.buf[at] : 0;
  }
  uint64_t lo = t.least, hi = ~0ull;  // fewer than k are > hi; at least k are >= lo, or lo is `least`
#pragma unroll 1
  while (lo < hi) {
    const uint64_t mid = lo + (hi - lo) / 2 + 1;
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) n += __popcll(__ballot(key[i] >= mid));
    if (n >= k) {
      lo = mid;
      if (n <= kKeep) break;
    } else {
      hi = mid - 1;
    }
  }
  t.least = lo;
  t.count = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool keep = key[i] >= lo && key[i] != 0;
    const uint64_t mask = __ballot(keep);
    if (keep) t.buf[t.count + __popcll(mask & lanemask_lt())] = key[i];
    t.count += __popcll(mask);
  }
}

// Writes the k largest of list[0 .. n), in order, as fn(place, key).  list has room to n + 3 and is 16-byte aligned.
template <typename F>
__device__ __forceinline__ void write_top(uint64_t* list, int n, int k, F fn) {
  if (threadIdx.x < 3) list[n + threadIdx.x] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const uint64_t mine = list[j];
    int rank = 0;
    for (int o = 0; o < n; o += 4) {
      const ulonglong2 a = *(const ulonglong2*)(list + o), b = *(const ulonglong2*)(list + o + 2);
      rank += (a.x > mine) + (a.y > mine) + (b.x > mine) + (b.y > mine);
    }
    if (rank < k) fn(rank, mine);
  }
}

template <typename E, bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LpArgs a) {
  constexpr int kVec = 16 / sizeof(E);
  __shared__ __attribute__((aligned(16))) TopLds lds;
  __shared__ Sums s_sums[kWaves];
  __shared__ float s_max[kWaves];
  __shared__ int s_odd[kWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const E* x = (const E*)a.x + row * a.stride;
  // values in front of the first 16-byte boundary, vectors, values behind the last
  const int head = min(a.V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(E));
  const int vecs = (a.V - head) / kVec;
  const int per = (vecs + a.splits - 1) / a.splits;
  const int v0 = min(split * per, vecs), v1 = min(v0 + per, vecs);
  const uint4* xv = (const uint4*)(x + head);
  // the first and the last workgroup of a row take its edges too, their first wave a lane each
  const int tail0 = head + vecs * kVec;
  const int n_head = split == 0 ? head : 0, n_edge = wave == 0 ? n_head + (split == a.splits - 1 ? a.V - tail0 : 0) : 0;
  const int edge = lane < n_head ? lane : tail0 + lane - n_head;
  // where `rows` of the workgroup's rows of 16 lanes have per_row values of at least b, there are k of them
  const int per_row = (a.k + kBoundRows - 1) / kBoundRows, rows = (a.k + max(per_row, 1) - 1) / max(per_row, 1);

  const int first = v0 + wave * MOE_WAVE;
  // candidates: vectors, as {bits of the maximum, index}
  uint64_t* cand = lds.cand[wave];
  int count = 0;
  bool full = false;   // more of them than there is room for
  bool stale = false;  // of which some the bound may have passed
  bool ordered = true;  // in the order of the row
  float lane_max = -INFINITY, least = -INFINITY;  // values below `least` are not among the k largest
  float m = -INFINITY, m2 = 0.f, limit = -INFINITY, s = 0.f, t = 0.f;
  auto reference = [&](float pm) __attribute__((always_inline)) {
    if (__any(pm > limit)) {
      const float old = m2;
      const bool first = m == -INFINITY;
      m = wave_max_uniform(fmaxf(m, pm));
      m2 = fmaxf(m * kLog2e, -kFar);  // values below leave nothing
      asm("" : "+v"(m2));  // rounded: as an operand of a fused difference it would not be what the terms were formed with
      limit = m + kSlack;
      if (!first) {  // before the first value that is not -inf the sums are 0, or NaN
        const float d = old - m2, c = __builtin_amdgcn_exp2f(d);
        t = fmaf(s, d, t) * c;
        s *= c;
      }
    }
  };
  auto add = [&](float v) __attribute__((always_inline)) {
    const float d = fmaf(v, kLog2e, -m2), e = __builtin_amdgcn_exp2f(d);
    s += e;
    t = fmaf(e, fmaxf(d, kNoTerm), t);
  };
  auto row_max = [&](float v) __attribute__((always_inline)) {
    v = fmaxf(v, ror<1>(v));
    v = fmaxf(v, ror<2>(v));
    v = fmaxf(v, ror<4>(v));
    return fmaxf(v, ror<8>(v));
  };
  auto renew = [&]() __attribute__((always_inline)) {
    float rest = lane_max, best = row_max(rest);
#pragma unroll 1
    for (int i = 1; i < per_row; ++i) {
      const uint32_t at = (uint32_t)(__ballot(rest == best) >> (lane & 48)) & 0xffffu;  // the row's lanes that have it
      rest = 1u << (lane & 15) == (at & -at) ? -INFINITY : rest;
      best = row_max(rest);
    }
    if (lane % 16 == 0) ((volatile float*)lds.bound)[wave * 4 + lane / 16] = best;
  };
  auto take_bound = [&]() __attribute__((always_inline)) {  // the rows' `rows`-th largest
    const float mine = ((volatile float*)lds.bound)[lane % 16];
    int more = 0;
    count_more<15>(mine, more);
    const float b = -row_max(more < rows ? -mine : -INFINITY);
    least = fmaxf(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(b))), kLowest);  // -inf: only where there is nothing else
    stale = true;
  };
  auto push = [&](float most, int index, bool pass) __attribute__((always_inline)) {
    const uint64_t mask = __ballot(pass);
    if (count > kCand - MOE_WAVE) full = true, count = 0;
    if (pass) cand[count + __popcll(mask & lanemask_lt())] = (uint64_t)__float_as_uint(most) << 32 | (uint32_t)index;
    count += __popcll(mask);
  };
  auto drop = [&]() __attribute__((always_inline)) {  // candidates that the bound has passed
    const int n = count;
    count = 0;
#pragma unroll 1
    for (int j = 0; j < n; j += MOE_WAVE) {
      const uint64_t e = cand[min(j + lane, n - 1)];
      const float most = __uint_as_float((uint32_t)(e >> 32));
      push(most, (int)(uint32_t)e, j + lane < n && !(most < least));
    }
    stale = false;
  };
  // A batch's vectors, of turns from `turn0` on.  Few are taken a lane's at a time, many in the order of the row: then behind k
  // candidates those that only equal the bound have none of the largest.
  auto offer_batch = [&](int turn0, int turns) __attribute__((always_inline)) {
    uint32_t mine = 0;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) mine |= lds.most[b / kPer][threadIdx.x][b % kPer] < least ? 0u : 1u << b;
    mine &= (2u << (kPer * turns - 1)) - 1;
    auto value = [&](int b) __attribute__((always_inline)) { return lds.most[b / kPer][threadIdx.x][b % kPer]; };
    auto place = [&](int b) __attribute__((always_inline)) { return first + lane + (kPer * turn0 + b) * kThreads; };
    if (count + __popcll(__ballot(mine != 0)) <= kFewCand) {
#pragma unroll 1
      while (__any(mine != 0)) {
        const int b = __builtin_ctz(mine | 1u << 31) % kBatch;
        push(value(b), place(b), mine != 0);
        mine &= mine - 1;
        ordered = false;
      }
      return;
    }
    if (stale) drop();
#pragma unroll 1
    for (int b = 0; b < kPer * turns; ++b) {
      const float most = value(b);
      const uint64_t mask = __ballot(!(most < least));
      push(most, place(b), !(most < least) && (most != least || count + __popcll(mask & lanemask_lt()) < a.k));
    }
  };
  // kPer vectors a turn, those of the next one on their way, and before them the edges.
  auto load = [&](int i) __attribute__((always_inline)) { return xv[min(i, max(v1, 1) - 1)]; };
  uint4 now[kPer], next[kPer];
  if (vecs > 0) {
#pragma unroll
    for (int h = 0; h < kPer; ++h) now[h] = load(first + h * kThreads + lane);
  }
  const float edge_value = lane < n_edge ? value_at(x, edge) : -INFINITY;
  Given given{};
  if (a.splits == 1) given = given_of<E>(a, row);
  if (wave == 0) {  // the other waves' is -inf
    if (TOP) lane_max = edge_value;
    reference(edge_value);
    add(edge_value);
  }
  const bool brief = v1 - v0 <= kTurn;  // all in the first turn's registers
  const int turns = max((v1 - v0 + kTurn - 1) / kTurn, 1);
  float v[kPer][kVec], pm[kPer];
#pragma unroll 1
  for (int turn = 0; turn < turns; ++turn) {
    const int i0 = first + turn * kTurn;
    const int i = i0 + lane;
    if (turn + 1 < turns) {
#pragma unroll
      for (int h = 0; h < kPer; ++h) next[h] = load(i + kTurn + h * kThreads);
    }
    float most = -INFINITY;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      unpack(now[h], v[h]);
      if (i0 + h * kThreads + MOE_WAVE > v1) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[h][e] = i + h * kThreads < v1 ? v[h][e] : -INFINITY;
      }
      pm[h] = v[h][0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) pm[h] = fmaxf(pm[h], v[h][e]);
      most = fmaxf(most, pm[h]);
    }
    reference(most);
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      if (i0 + h * kThreads >= v1) continue;  // nothing but -inf
#pragma unroll
      for (int e = 0; e < kVec; ++e) add(v[h][e]);
    }
    if (TOP) {
      lane_max = fmaxf(lane_max, most);
      if (!brief) {
#pragma unroll
        for (int h = 0; h < kPer; ++h) lds.most[turn % kBatchTurns][threadIdx.x][h] = pm[h];
      }
      if (turn % kBatchTurns == kBatchTurns - 1 && turn + 1 < turns) {
        renew();
        if (turn < kBatchTurns) __syncthreads();  // later the other waves' may be a batch old
        take_bound();
        offer_batch(turn + 1 - kBatchTurns, kBatchTurns);
      }
    }
#pragma unroll
    for (int h = 0; h < kPer; ++h) now[h] = next[h];
  }
  // from the reference as the sums used it, m log2(e) rounded, to m itself; all lanes' is the same
  const float off = m == -INFINITY ? 0.f : fmaf(m, kLog2e, -m2), undo = __builtin_amdgcn_exp2f(-off);
  s = wave_sum_uniform(s);
  t = wave_sum_uniform(t);
  Sums sum{m, s * undo, fmaf(-off, s, t) * undo};
  if (m * kLog2e < -kFar) sum.s = sum.t = 0.f;  // to another wave's maximum, or the row is gone over again

  if (lane == 0) s_max[wave] = m;
  if (TOP && threadIdx.x == 0) lds.n_list = 0;
  if (TOP) renew();
  uint64_t* list = lds.list;
  if (lane == 0) s_odd[wave] = !(fabsf(s) < INFINITY) || !(fabsf(t) < INFINITY);
  __syncthreads();
  bool again = false;
  m = s_max[0];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    again |= s_odd[w] != 0;
    m = fmaxf(m, s_max[w]);
  }
  bool redo = again;  // the largest too
  again |= m != -INFINITY && !(fabsf(m * kLog2e) < kFar - kFarSlack);
  if (TOP && !redo) {
    take_bound();
    // The values that reach the bound go to the list: value e is index + e, and `before` of them came earlier in the row; behind
    // k of them none that only equals the bound, which is looked at where there are many.
    auto keep = [&](const float* v, int n, int index, bool valid, int& before) __attribute__((always_inline)) {
      uint32_t reach = 0, over = 0;  // bit e: value e reaches the bound, passes it
#pragma unroll
      for (int e = 0; e < n; ++e) {
        reach |= v[e] < least ? 0u : 1u << e;
        over |= v[e] > least ? 1u << e : 0u;
      }
      reach = valid ? reach : 0u;
      const int lanes = __popcll(__ballot(reach != 0));
      if (lanes > kFewLanes && ordered) {
        int rank = before;
#pragma unroll 1
        for (int e = 0; e < n; ++e) rank += __popcll(__ballot(reach >> e & 1) & lanemask_lt());
        const uint32_t all = reach;
#pragma unroll 1
        for (int e = 0; e < n; ++e) {
          if (!(over >> e & 1) && rank >= a.k) reach &= ~(1u << e);
          rank += all >> e & 1;
        }
      }
      before += lanes;
#pragma unroll 1
      for (;;) {
        const uint64_t mask = __ballot(reach != 0);
        if (mask == 0) break;
        const int e = __builtin_ctz(reach | 1u << 31);
        float value = v[0];
#pragma unroll
        for (int o = 1; o < n; ++o) value = e == o ? v[o] : value;
        int to = 0;
        if (lane == 0) to = atomicAdd(&lds.n_list, __popcll(mask));
        to = __builtin_amdgcn_readfirstlane(to) + __popcll(mask & lanemask_lt());
        if (reach != 0 && to < kList) list[to] = key_of(value, index + e);
        reach &= reach - 1;
      }
    };
    int before = 0, edges = 0;
    if (brief) {
#pragma unroll
      for (int h = 0; h < kPer; ++h) {
        const int at = first + lane + h * kThreads;
        keep(v[h], kVec, head + at * kVec, at < v1, before);
      }
    } else {
      drop();
      offer_batch((turns - 1) / kBatchTurns * kBatchTurns, (turns - 1) % kBatchTurns + 1);
      if (full && lane == 0) atomicAdd(&lds.n_list, kList + 1);
#pragma unroll 1
      for (int j = 0; j < count; j += MOE_WAVE) {  // their other values are read again
        const int at = (int)(uint32_t)cand[min(j + lane, count - 1)];
        unpack(xv[at], v[0]);
        keep(v[0], kVec, head + at * kVec, j + lane < count, before);
      }
    }
    keep(&edge_value, 1, edge, lane < n_edge, edges);
    __syncthreads();
    const int found = lds.n_list;
    redo = found > kList;
    again |= redo;
    if (!redo && found < a.k) {  // all others are -inf: the first of them
      __syncthreads();
      if (wave == 0) {
        const int i = (split == 0 ? 0 : head + v0 * kVec) + lane, end = split == a.splits - 1 ? a.V : head + v1 * kVec;
        const bool more = lane < a.k && i < end && value_at(x, min(i, a.V - 1)) == -INFINITY;
        const uint64_t mask = __ballot(more);
        if (more) list[found + __popcll(mask & lanemask_lt())] = key_of(-INFINITY, i);
        if (lane == 0) lds.n_list = found + __popcll(mask);
      }
    }
  }

  // NaN, +inf, a maximum so far out that its product with log2(e) is rounded by much, more candidates than there is
  // room for (values that rise along the row): again, from the maximum and, for the largest, value by value.
  if (again) {
    __syncthreads();  // the counts are read
    s = t = 0.f;
    const float ref = m == -INFINITY ? 0.f : m;
    auto term = [&](float v) __attribute__((always_inline)) {
      const float d = (v - ref) * kLog2e, e = __builtin_amdgcn_exp2f(d);
      s += e;
      t = fmaf(e, fmaxf(d, kNoTerm), t);
    };
    term(edge_value);
    Top top{lds.buf[wave], 0, 0};
    if (TOP && redo) {
      if (threadIdx.x == 0) lds.n_list = 0;
      offer(top, edge_value, edge, lane < n_edge);
    }
    if (first < v1) now[0] = load(first + lane);
    for (int i0 = first; i0 < v1; i0 += kThreads) {
      const int j = i0 + lane, index = head + j * kVec;
      unpack(now[0], v[0]);
      now[0] = load(j + kThreads);
      // whether a value may be among the largest; later ones lose against equal earlier ones
      const float bound_value = value_of(top.least);
      bool maybe = top.least == 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        term(j < v1 ? v[0][e] : -INFINITY);
        maybe |= !(v[0][e] <= bound_value) || (v[0][e] == bound_value && index < index_of(top.least));
      }
      if (!TOP || !redo || !__any(maybe && j < v1)) continue;
#pragma unroll 1
      for (int e = 0; e < kVec; ++e) {
        offer(top, j < v1 ? value_at(x, index + e) : 0.f, index + e, j < v1);
        if (top.count > kBuf - MOE_WAVE) cut(top, a.k, lane);
      }
    }
    if (TOP && redo && top.count > kKeep) cut(top, a.k, lane);
    sum = Sums{m, wave_sum_uniform(s), wave_sum_uniform(t)};
    if (TOP && redo) {
      __syncthreads();  // the list is empty
      for (int j = lane; j < top.count; j += MOE_WAVE) list[atomicAdd(&lds.n_list, 1)] = top.buf[j];
    }
  }
  if (lane == 0) s_sums[wave] = sum;
  __syncthreads();
  sum = s_sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum = join(sum, s_sums[w]);
  Row r{};
  if (a.splits == 1) r = row_of(sum);
  if (TOP) {
    const int n = lds.n_list;
    uint64_t* out = a.splits > 1 ? a.keys + (long)blockIdx.x * a.k : nullptr;
    if (out)  // a short split has fewer
      for (int j = n + threadIdx.x; j < a.k; j += kThreads) out[j] = 0;
    write_top(list, n, a.k, [&](int place, uint64_t key) __attribute__((always_inline)) {
      if (out) {
        out[place] = key;
      } else {
        a.top_ids[(long)row * a.k + place] = index_of(key);
        a.top_logprobs[(long)row * a.k + place] = logprob(r, value_of(key));
      }
    });
  }
  if (threadIdx.x != 0) return;
  if (a.splits > 1) {
    a.sums[blockIdx.x] = make_float4(sum.m, sum.s, sum.t, 0.f);
    return;
  }
  finish(a, row, r, given);
}

// Joins a row's splits: their sums, and the k largest of their lists.  (3.6 us for one row's 38, 4.0 for 64 rows' 12.)
template <typename E>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LpArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t list[kMaxSplits * kMaxTop + 4];
  __shared__ int s_count;
  __shared__ uint32_t s_bound[kWaves];
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float4* parts = a.sums + (long)row * a.splits;
  const uint64_t* keys = a.keys + (long)row * a.splits * a.k;
  const int n = a.splits * a.k;
  // everything asked for at once
  const float4 v = lane < a.splits ? parts[lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  const int j = min(1 << wave, a.k), c = a.k > 0 ? (a.k + j - 1) / j : 0;
  const uint64_t mine = a.k > 0 && lane < a.splits ? keys[(long)lane * a.k + j - 1] : 0;
  const uint64_t first = (int)threadIdx.x < n ? keys[threadIdx.x] : 0;
  const Given given = given_of<E>(a, row);
  if (threadIdx.x == 0) s_count = 0;
  if (a.k > 0) {
    // Where c splits have j values of at least b each, with c j >= k, the k largest are all >= b: wave w looks at j = 1, 2, 4, 8.
    const uint32_t b = c <= a.splits ? bound_of((uint32_t)(mine >> 32), c) : 0;
    if (lane == 0) s_bound[wave] = b;
  }
  const Row r = row_of(join_wave(Sums{v.x, v.y, v.z}));
  if (a.k > 0) {
    __syncthreads();
    const uint32_t least = max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3]));
    int equal = 0;  // keys of the wave that only equal the bound: of those the first k, which the splits' order is
    for (int i0 = 0; i0 < n; i0 += kThreads) {
      const int i = i0 + (int)threadIdx.x;
      const uint64_t key = i0 == 0 ? first : i < n ? keys[i] : 0;
      const uint32_t value = (uint32_t)(key >> 32);
      const uint64_t mask = __ballot(key != 0 && value == least);
      if (key != 0 && (value > least || (value == least && equal + __popcll(mask & lanemask_lt()) < a.k)))
        list[atomicAdd(&s_count, 1)] = key;
      equal += __popcll(mask);
    }
    __syncthreads();
    write_top(list, s_count, a.k, [&](int place, uint64_t key) __attribute__((always_inline)) {
      a.top_ids[(long)row * a.k + place] = index_of(key);
      a.top_logprobs[(long)row * a.k + place] = logprob(r, value_of(key));
    });
  }
  if (threadIdx.x == 0) finish(a, row, r, given);
}

bool lp_ok(int T, int V, int k) { return T >= 0 && T < (1 << 24) && V >= 1 && V <= kMaxV && k >= 0 && k <= kMaxTop && k <= V; }

// Workgroups of a row: for three workgroups a CU in all, each with 4096 values at least.  (us in a graph, for 512 / 768 /
// 1024 / 1280 workgroups, 151936 bf16 values a row: 64 rows with 20 alternatives 15.0 / 15.7 / 16.6 / 16.5, 256 rows 27.7 /
// 25.5 / 26.1 / 25.5, 777 rows without alternatives 50 / 50 / 53 / 53, with 5 59 / 59 / 67 / 67; 777 fp32 rows of 50257 with 8 36.3 /
// 36.3 / 48 / 48.  Three sets of logits in turn, those of 256 rows and fewer partly from the cache behind L2.)
constexpr int kGroups = 768, kMinValues = 4096;
int lp_splits(int T, int V) {
  const int most = (V + kMinValues - 1) / kMinValues, want = (kGroups + T - 1) / (T > 0 ? T : 1);
  const int n = want < most ? want : most;
  return n < 1 ? 1 : n < kMaxSplits ? n : kMaxSplits;
}

size_t lp_carve(WsCarver& c, int T, int k, int splits, LpArgs* a) {
  if (splits > 1) {
    a->sums = c.take<float4>((size_t)T * splits);
    a->keys = c.take<uint64_t>((size_t)T * splits * k);
  }
  return moe_align_up(c.off, 256);
}

template <typename E>
int lp_launch(const LpArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((long)a.T * a.splits));
  if (a.k > 0)
    hipLaunchKernelGGL((logprobs_kernel<E, true>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((logprobs_kernel<E, false>), grid, dim3(kThreads), 0, s, a);
  MOE_CHECK_LAUNCH();
  if (a.splits > 1) {
    hipLaunchKernelGGL((logprobs_join_kernel<E>), dim3((unsigned)a.T), dim3(kThreads), 0, s, a);
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}

}  // namespace

extern "C" size_t moe_mi355x_token_logprobs_workspace_bytes(int T, int V, int k) {
  if (!lp_ok(T, V, k)) return 0;
  WsCarver c(nullptr);
  LpArgs a{};
  return lp_carve(c, T, k, lp_splits(T, V), &a);
}

extern "C" int moe_mi355x_token_logprobs(const void* logits, int dtype, long long stride, const void* tokens, int id_bytes,
                                         int T, int V, int k, float* logprobs, float* entropy, int64_t* top_ids,
                                         float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  MOE_RETURN_IF(!lp_ok(T, V, k) || (dtype != 0 && dtype != 1) || stride < V || (id_bytes != 4 && id_bytes != 8), MOE_ERR_INVALID_ARG);
  if (T == 0) return MOE_OK;
  MOE_RETURN_IF(!logits || !entropy || (tokens && !logprobs) || (k > 0 && (!top_ids || !top_logprobs)), MOE_ERR_INVALID_ARG);
  MOE_RETURN_IF((uintptr_t)logits % (dtype == 0 ? 2 : 4), MOE_ERR_ALIGNMENT);
  const size_t need = moe_mi355x_token_logprobs_workspace_bytes(T, V, k);
  MOE_RETURN_IF(need > 0 && (!workspace || workspace_bytes < need), MOE_ERR_WORKSPACE);
  MOE_RETURN_IF(need > 0 && !moe_aligned16(workspace), MOE_ERR_ALIGNMENT);
  LpArgs a{};
  a.x = logits, a.stride = stride, a.tokens = tokens, a.id_bytes = id_bytes, a.T = T, a.V = V, a.k = k, a.splits = lp_splits(T, V);
  a.logprobs = logprobs, a.entropy = entropy, a.top_ids = top_ids, a.top_logprobs = top_logprobs;
  WsCarver c(workspace);
  lp_carve(c, T, k, a.splits, &a);
  return dtype == 0 ? lp_launch<uint16_t>(a, (hipStream_t)stream) : lp_launch<float>(a, (hipStream_t)stream);
}
