// token_scores.cu -- what a row of logits says about a given token: its log
// probability, the log of the normaliser, the entropy and the best
// alternatives, from one read of the row.
//
// With m the row's maximum, d_j = x_j - m, s = sum e^{d_j}, u = sum e^{d_j} d_j:
//   log_sum = m + log s,  log_prob(t) = d_t - log s,  entropy = log s - u / s,
// and the K best (value, then lower index) with their d - log s.  The sums run
// in base 2: t_j = x_j L - b with L = log2(e) as rounded and b = m L rounded is
// one FMA, and exact up to its own rounding; b's rounding r = m L - b shifts
// every t alike and is taken out at the end.  r grows with m, so beyond 2^16
// (which no f16 reaches), where it is 2^-8, t_j = (x_j - m) L takes its place,
// with b = r = 0: a logit may be any finite number.  Parts of a row with bases b
// and b + g join as s 2^{-g}, (u - g s) 2^{-g}.  Statistics are f32 whatever the
// logits' type.  A masked (-inf) logit has t clamped, to where 2^t is zero, so
// that it adds 0 to u and not 0 * -inf; the clamp passes NaN on.  A row with a
// NaN or a +inf has no distribution: its numbers are NaN, its alternatives
// still rank (NaN as -inf).  A row of -inf alone scores -inf with entropy 0.
//
// Two routes.  HELD: the warps of a row hold it in registers, so the maximum
// is known before the first exponential; for few rows.  STREAM: many or long
// rows pass through once with a running (m, s, u) per thread.
//
// Alternatives cost nothing while the row is read: a lane knows its largest
// value, and the K-th largest of any maxima of parts of the row bounds the K-th
// best value from below.  Few values reach that bound (of 16 half warps, 11 for
// K = 8); they go to a pool in shared memory and each counts how many of the
// pool beat it: its rank.  A pool that
// overflows (a row of many equal values) is replaced by sorted lists, one per
// warp, into which candidates are inserted one at a time.  Where fewer than K
// columns are left by a mask, the lowest masked ids fill the places.
//
// Bound by reading the logits once where rows are long and many, and there by
// instructions on top: an element takes about ten (widen, compare, FMA, ex2, two
// sums).  4096x50257 f16 100 us, 4.1 TB/s or 63% of a copy's rate (80 us without
// alternatives: the warps of a row meet, read their candidates again and load
// nothing meanwhile); 16384x16384 f32 219 us, 4.9 TB/s.  Short calls are latency:
// 1x32000 f16 5.7 us, 1953x1025 f32 6.4 us; a row of 8 columns takes 3.1.
// A row belongs to one warp, to several
// warps of a CTA or to a cluster of CTAs (joined through distributed shared
// memory: no workspace, no atomics, so results do not depend on timing).
#include <algorithm>
#include <climits>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int TS_WARPS = 8;              // warps per CTA
constexpr int TS_THREADS = TS_WARPS * 32;
constexpr int TS_MAXK = 32;              // one alternative per lane
constexpr int TS_CLUSTER = 8;            // CTAs that share a row, at most
constexpr int TS_HELD = 10;              // 16-byte vectors per lane of a held row, at most
constexpr int TS_HELD_FEW = 4;           // and where there are few rows: more warps, shorter chains
constexpr int TS_AGAIN = 2;              // lanes whose vectors are read again at a time
constexpr int64_t TS_LIVE = 114000000;   // bytes of rows under way, at most: most of L2
constexpr int TS_UNR = 4;                // vectors per lane and tile of a streamed row
constexpr int TS_POOL = 128;             // candidates per warp of a row
constexpr uint32_t TS_MASKED = 0x007fffffu;  // ts_ordered(-inf)
constexpr float TS_LOG2E = 1.4426950408889634f;
constexpr float TS_LN2 = 0.6931471805599453f;
constexpr float TS_FAR = 65536.0f;  // beyond: t from x - m

struct TsParams {
  const void* logits;
  const uint32_t* targets;
  const uint32_t* row_count;
  const uint32_t* row_map;
  float* log_probs;
  float* log_sums;
  float* entropies;
  uint32_t* top_ids;
  float* top_log_probs;
  int64_t rows, stride, slots;
  int columns, k;
};

// A part of a row: its maximum, and the sums in base 2 relative to ts_base(m).
struct TsStat {
  float m, s, u;
};

struct TsSmem {
  alignas(16) unsigned char stage[TS_WARPS][TS_HELD * 16];  // one lane's values
  uint64_t pool[TS_WARPS * TS_POOL];     // candidates: TS_POOL places per warp of the row (or its sorted lists)
  uint64_t final[TS_WARPS][TS_MAXK];     // per row: the K best, in order
  uint64_t clist[TS_CLUSTER][TS_MAXK];   // the K best of the cluster's CTAs (rank 0 holds them all)
  TsStat stat[TS_WARPS];
  TsStat cstat[TS_CLUSTER];
  alignas(16) uint32_t lane_max[TS_WARPS][32];
  uint32_t bound[TS_WARPS];              // per warp
  uint32_t half_max[2 * TS_WARPS];
  int count[TS_WARPS];                   // per row: candidates
};

__device__ __forceinline__ float ts_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ts_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// Order-preserving bits of a float (its own zero: -0 counts as 0), and back.
__device__ __forceinline__ uint32_t ts_ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float ts_value(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
// A place in the order of alternatives: larger is better.  0 is an empty place.
__device__ __forceinline__ uint64_t ts_key(float v, uint32_t id) {
  return (uint64_t)ts_ordered(v != v ? -INFINITY : v) << 32 | (uint32_t)~id;
}

// Whether t is (x - m) L, the base of a maximum, and what its rounding leaves of
// m L.  A part whose maximum is -inf holds masked logits or NaN alone.
__device__ __forceinline__ bool ts_far(float m) { return fabsf(m) > TS_FAR && fabsf(m) < INFINITY; }
template <typename T>
__device__ __forceinline__ float ts_base(float m) {
  return m > -INFINITY && !(sizeof(T) == 4 && ts_far(m)) ? __fmul_rn(m, TS_LOG2E) : 0.0f;
}
template <typename T>
__device__ __forceinline__ float ts_rest(float m) {
  return sizeof(T) == 4 && ts_far(m) ? 0.0f : fmaf(m, TS_LOG2E, -ts_base<T>(m));
}
// The power of 2 that takes sums of maximum a (base ab) to maximum b (base bb).
template <typename T>
__device__ __forceinline__ float ts_gap(float a, float ab, float b, float bb) {
  if (sizeof(T) == 4 && (ts_far(a) || ts_far(b))) return fmaf(a - b, TS_LOG2E, ts_rest<T>(b) - ts_rest<T>(a));
  return ab - bb;
}

// (s, u) times 2^g, with t less by -g.
__device__ __forceinline__ void ts_shift(float g, float& s, float& u) {
  const float c = ts_ex2(g);
  u = c == 0.0f ? 0.0f : c * fmaf(g, s, u);  // once 2^g is 0 nothing is left
  s *= c;
}
// The same of a pair of sums.
__device__ __forceinline__ void ts_shift(float g, float2& s, float2& u) {
  const float c = ts_ex2(g);
  const float d = c == 0.0f ? 0.0f : g;
  const float2 c2 = make_float2(c, c), zero = make_float2(0.0f, 0.0f);
  u = ffma2(ffma2(s, make_float2(d, d), u), c2, zero);
  s = ffma2(s, c2, zero);
}

// The sums of the `n` (at most 8) parts of a row, in their order.
template <typename T>
__device__ __forceinline__ TsStat ts_join(const TsStat* part, int n) {
  TsStat r = part[0];
#pragma unroll
  for (int i = 1; i < 8; ++i)
    if (i < n) r.m = fmaxf(r.m, part[i].m);
  const float base = ts_base<T>(r.m);
  r.s = r.u = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= n) continue;
    TsStat p = part[i];
    if (p.s == 0.0f) continue;  // nothing but masked logits
    ts_shift(p.m == r.m ? 0.0f : ts_gap<T>(p.m, ts_base<T>(p.m), r.m, base), p.s, p.u);
    r.s += p.s;
    r.u += p.u;
  }
  return r;
}

// N 16-byte vectors of a row per lane.
template <typename T, int N>
struct TsTile {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr uint32_t NEG = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u;  // -inf
  uint4 raw[N];

  // Vector v of a row that starts `skew` elements into its first 16 bytes; what
  // is not of the row reads as -inf, and is not read.
  static __device__ __forceinline__ uint4 vector(const T* base, int skew, int columns, int v, int vectors) {
    const int c0 = v * VEC - skew;
    uint4 r = make_uint4(NEG, NEG, NEG, NEG);
    if (v < vectors) {
      if (c0 >= 0 && c0 + VEC <= columns) {
        r = __ldcs(reinterpret_cast<const uint4*>(base + c0));
      } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (c0 + j >= 0 && c0 + j < columns) e[j] = base[c0 + j];
      }
    }
    return r;
  }
  // Vectors v0 + lane + step q; `v0` is the warp's.
  __device__ __forceinline__ void load(const T* base, int skew, int columns, int v0, int lane, int step, int vectors) {
    if (v0 * VEC >= skew && (v0 + step * (N - 1) + 32) * VEC - skew <= columns) {  // all of them whole
      const uint4* src = reinterpret_cast<const uint4*>(base + (v0 + lane) * VEC - skew);
#pragma unroll
      for (int q = 0; q < N; ++q) raw[q] = __ldcs(src + step * q);
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) raw[q] = vector(base, skew, columns, v0 + lane + step * q, vectors);
    }
  }
  static __device__ __forceinline__ float largest(const uint4* raw, int n) {
    if constexpr (sizeof(T) == 2) {
      __half2 mx = *reinterpret_cast<const __half2*>(&raw[0].x);
#pragma unroll
      for (int q = 0; q < n; ++q) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[q]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = __hmax2(mx, h[j]);
      }
      const float2 f = __half22float2(mx);
      return fmaxf(fmaxf(f.x, f.y), -INFINITY);  // NaN counts as -inf
    } else {
      float mx = -INFINITY;
#pragma unroll
      for (int q = 0; q < n; ++q) {
        const float* f = reinterpret_cast<const float*>(&raw[q]);
        mx = fmaxf(mx, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
      }
      return mx;
    }
  }
  __device__ __forceinline__ float maximum() const { return largest(raw, N); }
  // s += sum 2^t, u += sum 2^t t, relative to the maximum m of that base (FAR: of any size).
  template <bool FAR = sizeof(T) == 4>
  __device__ __forceinline__ void sums(float m, float base, float2& s, float2& u) const {
    const float b = -base;
    const float2 a2 = make_float2(TS_LOG2E, TS_LOG2E), b2 = make_float2(b, b), one = make_float2(1.0f, 1.0f);
    auto add = [&](float2 t) {
      const float2 e = make_float2(ts_ex2(t.x), ts_ex2(t.y));
      s = ffma2(e, one, s);
      u = ffma2(e, t, u);
    };
    if constexpr (sizeof(T) == 2) {
      // -inf becomes the lowest f16 before the conversion, two at a time: for
      // any m above it by 300 or more that is a 2^t of 0.
      if (m > -60000.0f) {
        const __half2 low = __float2half2_rn(-65504.0f);
#pragma unroll
        for (int q = 0; q < N; ++q) {
          const __half2* h = reinterpret_cast<const __half2*>(&raw[q]);
#pragma unroll
          for (int j = 0; j < 4; ++j) add(ffma2(__half22float2(__hmax2_nan(h[j], low)), a2, b2));
        }
        return;
      }
    }
    auto clamp = [&](float2 t) {
      t.x = ts_max_nan(t.x, -300.0f);
      t.y = ts_max_nan(t.y, -300.0f);
      add(t);
    };
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[q]);
#pragma unroll
        for (int j = 0; j < 4; ++j) clamp(ffma2(__half22float2(h[j]), a2, b2));
      }
    } else if (!FAR || !ts_far(m)) {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const float2* h = reinterpret_cast<const float2*>(&raw[q]);
        clamp(ffma2(h[0], a2, b2));
        clamp(ffma2(h[1], a2, b2));
      }
    } else {
      const float2 m2 = make_float2(-m, -m), zero = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const float2* h = reinterpret_cast<const float2*>(&raw[q]);
        clamp(ffma2(ffma2(h[0], one, m2), a2, zero));
        clamp(ffma2(ffma2(h[1], one, m2), a2, zero));
      }
    }
  }
};

// Inserts `key`, the same in all lanes, into the list (lane i holds the i-th).
__device__ __forceinline__ void ts_insert(uint64_t& list, uint64_t key, int lane) {
  const int pos = __popc(__ballot_sync(0xffffffffu, list > key));
  const uint64_t prev = __shfl_up_sync(0xffffffffu, list, 1);
  if (lane == pos) list = key;
  else if (lane > pos) list = prev;
}

// Inserts those of the lanes' keys that beat the list's K-th (each lane offers
// one; 0 offers nothing).
__device__ __forceinline__ void ts_offer(uint64_t& list, uint64_t key, int k, int lane) {
  uint64_t last = __shfl_sync(0xffffffffu, list, k - 1);
  uint32_t lanes = __ballot_sync(0xffffffffu, key > last);
  while (lanes) {
    const int src = __ffs(lanes) - 1;
    const uint64_t c = __shfl_sync(0xffffffffu, key, src);
    ts_insert(list, c, lane);
    last = __shfl_sync(0xffffffffu, list, k - 1);
    if (lane == src) key = 0;
    lanes = __ballot_sync(0xffffffffu, key > last);
  }
}

// How many entries of the `lists` sorted lists (k entries each, `pitch` apart)
// come before entry `pos` of list `own`; equal entries in order of their lists.
template <typename U>
__device__ __forceinline__ int ts_rank(const U* list, int pitch, int lists, int k, int own, int pos) {
  const U key = list[own * pitch + pos];
  int rank = pos;
#pragma unroll
  for (int l = 0; l < 8; ++l) {
    if (l >= lists || l == own) continue;
    const U* other = list + l * pitch;
    int n = 0;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) {
      const int i = n + step;
      if (i <= k && (other[i - 1] > key || (other[i - 1] == key && l < own))) n = i;
    }
    rank += n;
  }
  return rank;
}

// Barrier of the `wpr` warps of a row (barrier 0 is the CTA's).
__device__ __forceinline__ void ts_row_sync(int group, int wpr) {
  if (wpr == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(wpr * 32) : "memory");
}

// A value (ordered bits) that at least k of the row's columns in this CTA
// reach, where k are unmasked.  While the row has k half warps, the k-th largest
// of their maxima; else the least of the warps' j-th largest lane maxima,
// j = ceil(k / wpr).  More than -inf: no masked value is a candidate.
__device__ __forceinline__ uint32_t ts_bound(TsSmem& sm, uint32_t mine, int group, int wpr, int k) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t bound;
  if (wpr > 1 && k <= 2 * wpr) {
    uint32_t top = mine;  // of the half warp
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((lane & 15) == 0) sm.half_max[2 * warp + (lane >> 4)] = top;
    ts_row_sync(group, wpr);
    const uint32_t* of = sm.half_max + 2 * group * wpr;
    const uint32_t v = lane < 2 * wpr ? of[lane] : 0;
    int above = 0;
#pragma unroll
    for (int i = 0; i < 2 * TS_WARPS; ++i)
      if (i < 2 * wpr) above += of[i] > v;
    bound = __reduce_min_sync(0xffffffffu, lane < 2 * wpr && above < k ? v : 0xffffffffu);
    return max(bound, TS_MASKED + 1);
  }
  const int j = (k + wpr - 1) / wpr;
  if (j == 1) {
    bound = __reduce_max_sync(0xffffffffu, mine);
  } else {
    sm.lane_max[warp][lane] = mine;
    __syncwarp();
    int above = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 o = reinterpret_cast<const uint4*>(sm.lane_max[warp])[i];
      above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
    }
    bound = __reduce_min_sync(0xffffffffu, above < j ? mine : 0xffffffffu);
  }
  if (wpr > 1) {
    if (lane == 0) sm.bound[warp] = bound;
    ts_row_sync(group, wpr);
    bound = sm.bound[group * wpr];
#pragma unroll
    for (int w = 1; w < 8; ++w)
      if (w < wpr) bound = min(bound, sm.bound[group * wpr + w]);
  }
  return max(bound, TS_MASKED + 1);
}

// Whether the row's candidates did not fit the pool.
__device__ __forceinline__ bool ts_overflow(TsSmem& sm, int group, int wpr) {
  ts_row_sync(group, wpr);
  return sm.count[group] > wpr * TS_POOL;
}

// `wpr` warps of the CTA read one row (8 / wpr rows per CTA); with CLUSTER the
// CTAs of a cluster share one row.  NV: vectors per lane of a held row, 0: the
// row is streamed.
template <typename T, int NV, bool CLUSTER>
__global__ void __launch_bounds__(TS_THREADS, sizeof(T) == 2 && NV > 0 ? (NV == TS_HELD ? 2 : 3) : NV == TS_HELD ? 3 : 4) token_scores_kernel(const TsParams p, int wpr) {
  pdl_entry();
  // Distributed shared memory is written only after this barrier's wait: by
  // then every CTA of the cluster runs.
  if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  __shared__ TsSmem sm;
  constexpr int VEC = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = warp / wpr, wig = warp % wpr;  // row of the CTA, warp of the row
  const int ranks = CLUSTER ? (int)gridDim.x : 1;  // the grid is (cluster, rows) then
  const int rank = CLUSTER ? (int)blockIdx.x : 0;
  const int64_t row = CLUSTER ? (int64_t)blockIdx.y : (int64_t)blockIdx.x * (TS_WARPS / wpr) + group;
  const int64_t rows = p.row_count ? min(p.rows, (int64_t)*p.row_count) : p.rows;
  int64_t slot = row;
  bool live = row < rows;
  if (live && p.row_map) {
    slot = p.row_map[row];
    live = slot < p.slots;
  }
  const int k = p.k;
  const T* base = static_cast<const T*>(p.logits) + (live ? row : 0) * p.stride;
  float given = -INFINITY;
  if (live && p.targets && wig == 0 && lane == 0 && rank == 0) {
    const uint32_t target = p.targets[slot];
    given = target < (uint32_t)p.columns ? (float)base[target] : NAN;  // an id outside the row has no probability
  }
  const int skew = (int)((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  const int vectors = live ? (int)(((int64_t)skew + p.columns + VEC - 1) / VEC) : 0;
  const int columns = p.columns;
  const int warps = wpr * ranks, gw = rank * wpr + wig;  // warps of the row, this one
  unsigned char* stage = sm.stage[warp];
  uint64_t list = 0;
  bool overflow = false;
  TsStat st;
  if (tid < TS_WARPS) sm.count[tid] = 0;
  __syncthreads();
  auto offer = [&](float v, int id) {
    const int at = atomicAdd(&sm.count[group], 1);
    if (at < wpr * TS_POOL) sm.pool[group * wpr * TS_POOL + at] = ts_key(v, (uint32_t)id);
  };

  if constexpr (NV > 0) {
    // Vector q of a lane: (q * warps + gw) * 32 + lane.
    const int step = warps * 32, v0 = gw * 32 + lane;
    TsTile<T, NV> tile;
    tile.load(base, skew, columns, gw * 32, lane, step, vectors);
    const float mine = tile.maximum();
    st.m = ts_value(__reduce_max_sync(0xffffffffu, ts_ordered(mine)));
    float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
    tile.sums(st.m, ts_base<T>(st.m), s2, u2);
    st.s = s2.x + s2.y;
    st.u = u2.x + u2.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
      st.u += __shfl_xor_sync(0xffffffffu, st.u, o);
    }
    if (k > 0) {
      const float bound = ts_value(ts_bound(sm, ts_ordered(mine), group, wpr, k));
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        if (TsTile<T, 1>::largest(&tile.raw[q], 1) >= bound) {
          const T* e = reinterpret_cast<const T*>(&tile.raw[q]);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if ((float)e[j] >= bound) offer((float)e[j], (v0 + step * q) * VEC - skew + j);
        }
      }
      if (ts_overflow(sm, group, wpr)) {
        uint32_t lanes = __ballot_sync(0xffffffffu, mine >= bound);
        while (lanes) {
          const int src = __ffs(lanes) - 1;
          lanes &= lanes - 1;
          __syncwarp();
          if (lane == src) {
#pragma unroll
            for (int q = 0; q < NV; ++q) reinterpret_cast<uint4*>(stage)[q] = tile.raw[q];
          }
          __syncwarp();
#pragma unroll
          for (int i0 = 0; i0 < NV * VEC; i0 += 32) {
            const int i = i0 + lane;
            uint64_t c = 0;
            if (i < NV * VEC) {
              const float v = (float)reinterpret_cast<const T*>(stage)[i];
              const int id = (v0 - lane + src + step * (i / VEC)) * VEC - skew + i % VEC;
              if (v >= bound) c = ts_key(v, (uint32_t)id);
            }
            ts_offer(list, c, k, lane);
          }
        }
        overflow = true;
      }
    }
  } else {
    const int step = warps * 32 * TS_UNR, first = gw * 32 * TS_UNR;
    float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
    float m = -INFINITY, mb = 0.0f;  // the maximum and its base
    auto take = [&](const TsTile<T, TS_UNR>& tile) {
      const float tm = tile.maximum();
      if (tm > m) {
        const float to = ts_base<__half>(tm);
        if (m > -INFINITY) ts_shift(mb - to, s2, u2);
        m = tm;
        mb = to;
      }
      tile.template sums<false>(m, mb, s2, u2);
    };
    // The warps of four CTAs an SM cover each other's loads (a second tile in
    // registers, loaded ahead, was 7% slower: fewer warps, more moves).
    TsTile<T, TS_UNR> tile;
    for (int v = first; v < vectors; v += step) {
      tile.load(base, skew, columns, v, lane, 32, vectors);
      take(tile);
    }
    // Every maximum was taken to be within 2^16: others leave sums that are not
    // finite or are multiplied by zero, unless the last is one of them.  Such rows
    // are read again with the maxima known (to ask before each tile took 3%).
    if constexpr (sizeof(T) == 4) {
      if (__any_sync(0xffffffffu, ts_far(m) || !(fabsf(s2.x + s2.y + u2.x + u2.y) < INFINITY))) {
        mb = ts_base<T>(m);
        s2 = u2 = make_float2(0.0f, 0.0f);
        for (int v = first; v < vectors; v += step) {
          tile.load(base, skew, columns, v, lane, 32, vectors);
          tile.sums(m, mb, s2, u2);
        }
      }
    }
    // The lanes' sums, brought to the warp's maximum.
    st = TsStat{ts_value(__reduce_max_sync(0xffffffffu, ts_ordered(m))), s2.x + s2.y, u2.x + u2.y};
    if (st.s != 0.0f && m != st.m) ts_shift(ts_gap<T>(m, mb, st.m, ts_base<T>(st.m)), st.s, st.u);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
      st.u += __shfl_xor_sync(0xffffffffu, st.u, o);
    }
    if (k > 0) {
      const float bound = ts_value(ts_bound(sm, ts_ordered(m), group, wpr, k));
      // A lane that reaches it: its vectors, read again, 32 at a time.
      const uint32_t reach = __ballot_sync(0xffffffffu, m >= bound);
      const int own = first < vectors ? (vectors - first + step - 1) / step * TS_UNR : 0;
      auto again = [&](auto use) {
        for (int i0 = 0; i0 < own; i0 += 32) {
          const int i = i0 + lane;
          const int at = first + i / TS_UNR * step + 32 * (i % TS_UNR);
          for (uint32_t lanes = reach; lanes;) {
            uint4 raw[TS_AGAIN];
            int v[TS_AGAIN];
#pragma unroll
            for (int n = 0; n < TS_AGAIN; ++n) {
              v[n] = i < own && lanes ? at + __ffs(lanes) - 1 : vectors;
              lanes &= lanes - 1;
              raw[n] = TsTile<T, 1>::vector(base, skew, columns, v[n], vectors);
            }
#pragma unroll
            for (int n = 0; n < TS_AGAIN; ++n) use(raw[n], v[n] * VEC - skew);
          }
        }
      };
      again([&](const uint4& raw, int c0) {
        if (TsTile<T, 1>::largest(&raw, 1) >= bound) {
          const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if ((float)e[j] >= bound) offer((float)e[j], c0 + j);
        }
      });
      if (ts_overflow(sm, group, wpr)) {
        again([&](const uint4& raw, int c0) {
          const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            ts_offer(list, (float)e[j] >= bound ? ts_key((float)e[j], (uint32_t)(c0 + j)) : 0, k, lane);
        });
        overflow = true;
      }
    }
  }
  if (CLUSTER || wpr > 1) {
    if (lane == 0) sm.stat[warp] = st;
  }
  if (k > 0) {
    // This CTA's K best, in order, to `final` (or the first CTA's clist).
    auto put = [&](int place, uint64_t key) {
      if (place >= k) return;
      if constexpr (CLUSTER) {
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_addr(&sm.clist[rank][place]), 0)), "l"(key)
                     : "memory");
      } else {
        sm.final[group][place] = key;
      }
    };
    if constexpr (CLUSTER) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (overflow) {
      ts_row_sync(group, wpr);
      uint64_t* lists = sm.pool + group * wpr * TS_POOL;
      if (lane < k) lists[wig * TS_MAXK + lane] = list;
      ts_row_sync(group, wpr);
      if (lane < k) put(ts_rank(lists, TS_MAXK, wpr, k, wig, lane), list);
    } else {
      const int n = sm.count[group];
      const uint64_t* pool = sm.pool + group * wpr * TS_POOL;
      for (int i = wig * 32 + lane; i < n; i += wpr * 32) {
        const uint64_t key = pool[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += pool[j] > key ? 1 : 0;
        put(place, key);
      }
      for (int i = n + wig * 32 + lane; i < k; i += wpr * 32) put(i, 0);
    }
  } else if constexpr (CLUSTER) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
  if constexpr (CLUSTER) {
    __syncthreads();  // the warps' sums
    if (tid == 0) {
      st = ts_join<T>(sm.stat, TS_WARPS);
      const uint32_t cs = mapa_shared(smem_addr(&sm.cstat[rank]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs), "f"(st.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs + 4), "f"(st.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs + 8), "f"(st.u) : "memory");
    }
    __syncwarp();
    cluster_sync();
    if (rank != 0) return;
    if (lane < k && warp < ranks) {
      const uint64_t key = sm.clist[warp][lane];
      const int place = ts_rank(&sm.clist[0][0], TS_MAXK, ranks, k, warp, lane);
      if (place < k) sm.final[0][place] = key;
    }
  }
  if (k > 0 || wpr > 1) ts_row_sync(group, wpr);
  if (!live || wig != 0) return;
  if constexpr (CLUSTER) st = ts_join<T>(sm.cstat, ranks);
  else if (wpr > 1) st = ts_join<T>(sm.stat + group * wpr, wpr);
  const bool empty = st.s == 0.0f;
  const float r = ts_rest<T>(st.m) * TS_LN2;  // the base's rounding
  const float log_s = empty ? 0.0f : logf(st.s) - r;
  if (lane == 0) {
    if (p.log_probs) p.log_probs[slot] = empty ? (given == given ? -INFINITY : NAN) : (given - st.m) - log_s;
    if (p.log_sums) p.log_sums[slot] = empty ? -INFINITY : st.m + log_s;
    if (p.entropies) p.entropies[slot] = empty ? 0.0f : log_s - (st.u / st.s * TS_LN2 - r);
  }
  if (k == 0) return;
  const uint64_t key = lane < k ? sm.final[group][lane] : 0;
  uint32_t id = ~(uint32_t)key;
  const float v = key ? ts_value((uint32_t)(key >> 32)) : -INFINITY;
  const int left = __popc(__ballot_sync(0xffffffffu, key != 0));
  if (left < k) {
    // Fewer unmasked columns than places: the lowest ids that are not among them.
    uint64_t missing = columns >= 64 ? ~0ull : (1ull << columns) - 1;
    for (int i = 0; i < left; ++i) {
      const uint32_t taken = __shfl_sync(0xffffffffu, id, i);
      if (taken < 64) missing &= ~(1ull << taken);
    }
    for (int i = left; i < lane; ++i) missing &= missing - 1;
    if (lane >= left) id = (uint32_t)__ffsll((long long)missing) - 1;
  }
  if (lane < k) {
    if (p.top_ids) p.top_ids[slot * k + lane] = id;
    if (p.top_log_probs) p.top_log_probs[slot * k + lane] = empty ? -INFINITY : (v - st.m) - log_s;
  }
}

template <typename T, int NV>
int launch_route(const TsParams& p, int wpr, int cluster, cudaStream_t stream) {
  if (cluster > 1) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)cluster, (unsigned)p.rows);
    cfg.blockDim = dim3(TS_THREADS);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cuda_error(cudaLaunchKernelEx(&cfg, token_scores_kernel<T, NV, true>, p, (int)TS_WARPS), "token_scores launch");
  }
  const int64_t per = TS_WARPS / wpr;
  return cuda_error(launch_kernel(token_scores_kernel<T, NV, false>, dim3((unsigned)((p.rows + per - 1) / per)),
                                  dim3(TS_THREADS), 0, stream, p, wpr),
                    "token_scores launch");
}

template <typename T>
int launch_typed(const DeviceCtx& dev, const TsParams& p, cudaStream_t stream) {
  constexpr int64_t vec = 16 / sizeof(T);
  const int64_t vectors = (p.columns + 2 * vec - 2) / vec;  // of the row with the worst start
  auto warps_for = [&](int nv) {
    int64_t w = 1;
    while (w * 32 * nv < vectors) w *= 2;
    return w;
  };
  // More alternatives than half a warp's lanes: one warp's 32 lane maxima would bound them too loosely.
  const int64_t least = p.k > 16 ? 2 : 1;
  // Few rows: every warp holds little, over as many SMs as there are (1x32000 f16
  // 5.7 us against 6.5 with TS_HELD vectors a lane and 7.7 streamed; 1x131072 8.4,
  // 14.4 without a cluster).
  const int64_t few = std::max(warps_for(TS_HELD_FEW), least);
  if (few <= TS_WARPS * TS_CLUSTER && p.rows * few <= (int64_t)dev.sm_count * TS_WARPS)
    return launch_route<T, TS_HELD_FEW>(p, (int)std::min<int64_t>(few, TS_WARPS), (int)std::max<int64_t>(1, few / TS_WARPS),
                                        stream);
  // Rows that all run at once (two CTAs an SM): held, one round trip to memory
  // (1000x4096 f16 8.1 us against 12.3 streamed, 1953x1025 f32 6.4 against 10.2).
  // More rows are streamed, by warps that come and go with more of them on an SM
  // (16384x4096 f16 50 us against 98 held, 4096x8192 22 against 51).
  const int64_t held = std::max(warps_for(TS_HELD), least);
  if (held <= TS_WARPS && p.rows * held <= 2 * (int64_t)dev.sm_count * TS_WARPS) return launch_route<T, TS_HELD>(p, (int)held, 1, stream);
  if (held <= TS_WARPS * TS_CLUSTER && p.rows * held <= (int64_t)dev.sm_count * TS_WARPS)
    return launch_route<T, TS_HELD>(p, TS_WARPS, (int)(held / TS_WARPS), stream);
  // Streamed: a warp per row costs least (4096x8192 f16 22 us, 30 with two, 41 with
  // four, 46 with eight), as long as the rows fill the SMs and those under way
  // stay in L2, from where candidates are read again (4096x50257: 133, 128, 114, 102).
  int cluster = 1;
  while (cluster < TS_CLUSTER && p.rows * cluster * 2 <= dev.sm_count) cluster *= 2;
  const int64_t warps = (int64_t)dev.sm_count * 4 * TS_WARPS;  // at once
  int wpr = cluster > 1 ? TS_WARPS : (int)least;
  while (wpr < TS_WARPS && (p.rows * wpr * 2 <= warps || warps / wpr * p.columns * (int64_t)sizeof(T) > TS_LIVE)) wpr *= 2;
  return launch_route<T, 0>(p, wpr, cluster, stream);
}

}  // namespace

int launch_token_scores(const DeviceCtx& dev, const pk_token_scores_desc& d, cudaStream_t stream) {
  TsParams p;
  p.logits = d.logits;
  p.targets = d.log_probs ? d.targets : nullptr;
  p.row_count = d.row_count;
  p.row_map = d.row_map;
  p.log_probs = d.log_probs;
  p.log_sums = d.log_sums;
  p.entropies = d.entropies;
  p.top_ids = d.top_ids;
  p.top_log_probs = d.top_log_probs;
  p.rows = d.rows;
  p.stride = d.row_stride;
  p.slots = d.slots;
  p.columns = (int)d.columns;
  p.k = d.top_k;
  return d.precision == PK_FP16 ? launch_typed<__half>(dev, p, stream) : launch_typed<float>(dev, p, stream);
}

}  // namespace pk
