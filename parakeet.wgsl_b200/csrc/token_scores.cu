// token_scores.cu -- what a row of logits says about a given token: its log
// probability, the log of the normaliser, the entropy and the best
// alternatives, in one pass over the row.
//
// With m the row's maximum, d_j = x_j - m, s = sum e^{d_j}, u = sum e^{d_j} d_j:
//   log_sum = m + log s,  log_prob(t) = d_t - log s,  entropy = log s - u / s,
// and the K best (value, then lower index) with their d - log s.  A thread
// keeps a running (m, s, u): when its maximum grows by g, s becomes s e^{-g}
// and u becomes (u - g s) e^{-g}.  Statistics are f32 whatever the logits' type
// and use x - m itself (exact near the maximum), not x log2(e) - m log2(e).
// A masked (-inf) logit has d clamped to -200, where e^d is zero, so that it
// adds 0 to u and not 0 * -inf; the clamp passes NaN on.  A row with a NaN or a
// +inf has no distribution: its numbers are NaN, its alternatives still rank
// (NaN as -inf).  A row of -inf alone scores -inf with entropy 0.
//
// Alternatives: a warp keeps its K best in registers, lane i the i-th, and
// inserts a candidate with one ballot and two shuffles.  Few values get that
// far: a tile is looked at only if some lane's maximum reaches the K-th best
// value any warp of the row has seen (one shared word, only ever raised), and
// the first tile starts from the K-th largest of the warp's 32 lane maxima.
// Joining lists counts, for every entry, how many entries beat it: its rank.
//
// Bound by reading the logits once.  A row is read by one warp, several warps
// of a CTA or a cluster of CTAs (joined through distributed shared memory: no
// workspace, no atomics on results, so results do not depend on timing).
#include <algorithm>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int TS_WARPS = 8;              // warps per CTA
constexpr int TS_THREADS = TS_WARPS * 32;
constexpr int TS_MAXK = 32;              // one alternative per lane
constexpr int TS_UNR = 4;                // 16-byte vectors per lane and tile
constexpr int TS_CLUSTER = 8;            // CTAs that share a row, at most
constexpr float TS_LOG2E = 1.4426950408889634f;

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

struct TsStat {
  float m, s, u;
};

struct TsSmem {
  alignas(16) unsigned char stage[TS_WARPS][32 * 16];  // one lane's tile, or the warp's lane maxima
  float lv[TS_WARPS][TS_MAXK];                         // the warps' lists
  uint32_t li[TS_WARPS][TS_MAXK];
  float cv[TS_CLUSTER][TS_MAXK];                       // the cluster's lists (rank 0 holds them all)
  uint32_t ci[TS_CLUSTER][TS_MAXK];
  TsStat stat[TS_WARPS];
  TsStat cstat[TS_CLUSTER];
  uint32_t bound[TS_WARPS];                            // per row of the CTA: ordered bits of the K-th best value seen
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
// Order-preserving bits of a float (its own zero: -0 counts as 0).
__device__ __forceinline__ uint32_t ts_ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ bool ts_beats(float av, uint32_t ai, float bv, uint32_t bi) {
  return av > bv || (av == bv && ai < bi);
}

// (m, s, u) of two parts of a row.
__device__ __forceinline__ TsStat ts_join(TsStat a, TsStat b) {
  const float m = fmaxf(a.m, b.m);
  TsStat r{m, 0.0f, 0.0f};
  auto add = [&](const TsStat& p) {
    if (p.s == 0.0f) return;  // nothing but masked logits
    const float g = p.m == m ? 0.0f : p.m - m;
    const float c = ts_ex2(g * TS_LOG2E);
    r.s = fmaf(p.s, c, r.s);
    // The part's share after rescaling; e^g g is 0 once e^g is.
    r.u = fmaf(c, c > 0.0f || c != c ? fmaf(g, p.s, p.u) : 0.0f, r.u);
  };
  add(a);
  add(b);
  return r;
}

template <typename T>
struct TsTile {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr uint32_t NEG = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u;  // -inf
  uint4 raw[TS_UNR];

  // Vectors v0, v0 + 32, ... of the row, which starts `skew` elements into its
  // first 16-byte vector; a vector that is not whole is read element by element.
  __device__ __forceinline__ void load(const T* base, int skew, int columns, int v0, int vectors) {
#pragma unroll
    for (int q = 0; q < TS_UNR; ++q) {
      const int v = v0 + 32 * q;
      const int c0 = v * VEC - skew;
      raw[q] = make_uint4(NEG, NEG, NEG, NEG);
      if (v < vectors) {
        if (c0 >= 0 && c0 + VEC <= columns) {
          raw[q] = __ldcs(reinterpret_cast<const uint4*>(base + c0));
        } else {
          T* e = reinterpret_cast<T*>(&raw[q]);
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (c0 + j >= 0 && c0 + j < columns) e[j] = base[c0 + j];
        }
      }
    }
  }
  __device__ __forceinline__ float maximum() const {
    if constexpr (sizeof(T) == 2) {
      __half2 mx = *reinterpret_cast<const __half2*>(&raw[0].x);
#pragma unroll
      for (int q = 0; q < TS_UNR; ++q) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[q]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = __hmax2(mx, h[j]);
      }
      const float2 f = __half22float2(mx);
      return fmaxf(fmaxf(f.x, f.y), -INFINITY);
    } else {
      float mx = -INFINITY;
#pragma unroll
      for (int q = 0; q < TS_UNR; ++q) {
        const float* f = reinterpret_cast<const float*>(&raw[q]);
        mx = fmaxf(mx, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
      }
      return mx;
    }
  }
  template <typename F>
  __device__ __forceinline__ void pairs(F f) const {
#pragma unroll
    for (int q = 0; q < TS_UNR; ++q) {
      if constexpr (sizeof(T) == 2) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[q]);
#pragma unroll
        for (int j = 0; j < 4; ++j) f(__half22float2(h[j]));
      } else {
        const float2* h = reinterpret_cast<const float2*>(&raw[q]);
        f(h[0]);
        f(h[1]);
      }
    }
  }
};

// A warp's K best: lane i holds the i-th (value, index); an empty place is
// (-inf, ~0).
struct TsList {
  float v = -INFINITY;
  uint32_t i = 0xffffffffu;

  // Inserts (cv, ci), the same in all lanes.
  __device__ __forceinline__ void insert(float cv, uint32_t ci, int k, int lane) {
    const int pos = __popc(__ballot_sync(0xffffffffu, ts_beats(v, i, cv, ci)));
    const float pv = __shfl_up_sync(0xffffffffu, v, 1);
    const uint32_t pi = __shfl_up_sync(0xffffffffu, i, 1);
    if (pos >= k) return;
    if (lane == pos) {
      v = cv;
      i = ci;
    } else if (lane > pos) {
      v = pv;
      i = pi;
    }
  }
};

// Looks at the tile's lanes whose maximum reaches `bound`: each such lane's
// values are spread over the warp through `stage`, and those that reach the
// bound are inserted.  Returns the raised bound.
template <typename T>
__device__ __forceinline__ uint32_t ts_candidates(const TsTile<T>& tile, TsList& list, unsigned char* stage, uint32_t mine,
                                               uint32_t bound, int v0, int skew, int columns, int k, int lane) {
  constexpr int VEC = TsTile<T>::VEC;
  constexpr int EPL = VEC * TS_UNR;
  uint32_t lanes = __ballot_sync(0xffffffffu, mine >= bound);
  while (lanes) {
    const int src = __ffs(lanes) - 1;
    lanes &= lanes - 1;
    if (__shfl_sync(0xffffffffu, mine, src) < bound) continue;  // the bound rose meanwhile
    __syncwarp();
    if (lane == src) {
#pragma unroll
      for (int q = 0; q < TS_UNR; ++q) reinterpret_cast<uint4*>(stage)[q] = tile.raw[q];
    }
    __syncwarp();
    float v = -INFINITY;
    uint32_t id = 0xffffffffu;
    if (lane < EPL) {
      v = (float)reinterpret_cast<const T*>(stage)[lane];
      if (v != v) v = -INFINITY;
      const int c = (v0 - lane + src + 32 * (lane / VEC)) * VEC - skew + lane % VEC;
      if (c >= 0 && c < columns) id = (uint32_t)c;
    }
    uint32_t cand = __ballot_sync(0xffffffffu, id != 0xffffffffu && ts_ordered(v) >= bound);
    while (cand) {
      const int from = __ffs(cand) - 1;
      cand &= cand - 1;
      list.insert(__shfl_sync(0xffffffffu, v, from), __shfl_sync(0xffffffffu, id, from), k, lane);
    }
    // The K-th best so far, once there are K.
    const uint32_t last = __shfl_sync(0xffffffffu, list.i, k - 1);
    if (last != 0xffffffffu) bound = max(bound, ts_ordered(__shfl_sync(0xffffffffu, list.v, k - 1)));
  }
  return bound;
}

// Ranks `n` entries (value, index; ties of empty places by position) and hands
// each of the best `k` to out(rank, value, index).
template <typename Out>
__device__ __forceinline__ void ts_rank(const float* v, const uint32_t* id, int lists, int k, int t, int threads, Out out) {
  const int n = lists * k;
  for (int e = t; e < n; e += threads) {
    const float ev = v[e / k * TS_MAXK + e % k];
    const uint32_t ei = id[e / k * TS_MAXK + e % k];
    int rank = e % k;  // a list is in order
    for (int l = 0; l < lists; ++l) {
      if (l == e / k) continue;
      for (int j = 0; j < k; ++j) {
        const float ov = v[l * TS_MAXK + j];
        const uint32_t oi = id[l * TS_MAXK + j];
        // Equal entries are empty places: the earlier list's come first.
        const bool beats = ts_beats(ov, oi, ev, ei) || (ov == ev && oi == ei && l < e / k);
        if (!beats) break;
        ++rank;
      }
    }
    if (rank < k) out(rank, ev, ei);
  }
}

// `wpr` warps of the CTA read one row (8 / wpr rows per CTA); with CLUSTER the
// CTAs of a cluster share one row.
template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(TS_THREADS) token_scores_kernel(const TsParams p, int wpr) {
  pdl_entry();
  // Distributed shared memory is written only after this barrier's wait: by
  // then every CTA of the cluster runs.
  if constexpr (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  __shared__ TsSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = warp / wpr, wig = warp % wpr;  // row of the CTA, warp of the row
  const int ranks = CLUSTER ? (int)gridDim.x : 1;  // the grid is (cluster, rows) then
  const int rank = CLUSTER ? (int)blockIdx.x : 0;
  const int64_t row = CLUSTER ? (int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y
                              : (int64_t)blockIdx.x * (TS_WARPS / wpr) + group;
  const int64_t rows = p.row_count ? min(p.rows, (int64_t)*p.row_count) : p.rows;
  int64_t slot = row;
  bool live = row < rows;
  if (live && p.row_map) {
    slot = p.row_map[row];
    live = slot < p.slots;
  }
  const int k = p.k;
  const T* base = static_cast<const T*>(p.logits) + (live ? row : 0) * p.stride;
  uint32_t target = 0;
  float given = -INFINITY;
  if (live && p.targets && wig == 0 && lane == 0 && rank == 0) {
    target = p.targets[slot];
    given = target < (uint32_t)p.columns ? (float)base[target] : NAN;  // an id outside the row has no probability
  }
  if (tid < TS_WARPS) sm.bound[tid] = 0;
  __syncthreads();

  TsList list;
  TsStat st{-INFINITY, 0.0f, 0.0f};
  if (live) {
    const int skew = (int)((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
    const int vectors = (int)(((int64_t)skew + p.columns + TsTile<T>::VEC - 1) / TsTile<T>::VEC);
    const int step = wpr * ranks * 32 * TS_UNR;
    int v0 = (rank * wpr + wig) * 32 * TS_UNR + lane;
    float2 s2 = make_float2(0.0f, 0.0f), u2 = make_float2(0.0f, 0.0f);
    float m = -INFINITY;
    TsTile<T> tile, next;
    const int first = v0 - lane;
    tile.load(base, skew, p.columns, v0, vectors);
    for (; v0 - lane < vectors; v0 += step) {
      if (v0 - lane + step < vectors) next.load(base, skew, p.columns, v0 + step, vectors);
      const float tm = tile.maximum();
      if (tm > m) {
        if (m > -INFINITY) {
          const float g = m - tm;
          const float c = ts_ex2(g * TS_LOG2E);
          // Once e^g is 0 nothing of the old sums is left.
          u2.x = c > 0.0f ? fmaf(g, s2.x, u2.x) * c : 0.0f;
          u2.y = c > 0.0f ? fmaf(g, s2.y, u2.y) * c : 0.0f;
          s2.x *= c;
          s2.y *= c;
        }
        m = tm;
      }
      const float neg = m > -INFINITY ? -m : 0.0f;
      tile.pairs([&](float2 x) {
        float2 d = ffma2(x, make_float2(1.0f, 1.0f), make_float2(neg, neg));
        d.x = ts_max_nan(d.x, -200.0f);
        d.y = ts_max_nan(d.y, -200.0f);
        const float2 t = ffma2(d, make_float2(TS_LOG2E, TS_LOG2E), make_float2(0.0f, 0.0f));
        const float2 e = make_float2(ts_ex2(t.x), ts_ex2(t.y));
        s2 = ffma2(e, make_float2(1.0f, 1.0f), s2);
        u2 = ffma2(e, d, u2);
      });
      if (k > 0) {
        const uint32_t mine = ts_ordered(tm);
        uint32_t bound = *(volatile uint32_t*)&sm.bound[group];
        if (v0 - lane == first) {
          // The K-th largest lane maximum: K values of the tile reach it.
          float* mx = reinterpret_cast<float*>(sm.stage[warp]);
          mx[lane] = tm;
          __syncwarp();
          int above = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 o = reinterpret_cast<const float4*>(mx)[j];
            above += (o.x > tm) + (o.y > tm) + (o.z > tm) + (o.w > tm);
          }
          bound = max(bound, __reduce_min_sync(0xffffffffu, above < k ? mine : 0xffffffffu));
          __syncwarp();
        }
        if (__any_sync(0xffffffffu, mine >= bound)) {
          const uint32_t raised =
              ts_candidates<T>(tile, list, sm.stage[warp], mine, bound, v0, skew, p.columns, k, lane);
          if (lane == 0) atomicMax(&sm.bound[group], raised);
        }
      }
#pragma unroll
      for (int q = 0; q < TS_UNR; ++q) tile.raw[q] = next.raw[q];
    }
    st = TsStat{m, s2.x + s2.y, u2.x + u2.y};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const TsStat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                         __shfl_xor_sync(0xffffffffu, st.u, o)};
      // Both lanes of a pair join in the same order.
      st = (lane & o) ? ts_join(other, st) : ts_join(st, other);
    }
  }
  if (lane == 0) sm.stat[warp] = st;
  sm.lv[warp][lane] = list.v;
  sm.li[warp][lane] = list.i;
  __syncthreads();
  // Every thread of the row joins the warps' sums (the same numbers in all).
  st = sm.stat[group * wpr];
  for (int w = 1; w < wpr; ++w) st = ts_join(st, sm.stat[group * wpr + w]);
  const float* lv = sm.lv[group * wpr];
  const uint32_t* li = sm.li[group * wpr];
  int lists = wpr;
  if constexpr (CLUSTER) {
    // This CTA's list and sums go to the first CTA's shared memory.
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const uint32_t cv = mapa_shared(smem_addr(&sm.cv[rank][0]), 0), ci = mapa_shared(smem_addr(&sm.ci[rank][0]), 0);
    ts_rank(lv, li, lists, k, tid, TS_THREADS, [&](int r, float v, uint32_t id) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cv + 4 * r), "f"(v) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ci + 4 * r), "r"(id) : "memory");
    });
    if (tid == 0) {
      const uint32_t cs = mapa_shared(smem_addr(&sm.cstat[rank]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs), "f"(st.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs + 4), "f"(st.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cs + 8), "f"(st.u) : "memory");
    }
    __syncthreads();
    cluster_sync();
    if (rank != 0) return;
    st = sm.cstat[0];
    for (int r = 1; r < ranks; ++r) st = ts_join(st, sm.cstat[r]);
    lv = sm.cv[0];
    li = sm.ci[0];
    lists = ranks;
  }
  if (!live) return;
  const bool empty = st.s == 0.0f;
  const float log_s = empty ? 0.0f : logf(st.s);
  if (wig == 0 && lane == 0) {
    if (p.log_probs) p.log_probs[slot] = empty ? (given == given ? -INFINITY : NAN) : (given - st.m) - log_s;
    if (p.log_sums) p.log_sums[slot] = empty ? -INFINITY : st.m + log_s;
    if (p.entropies) p.entropies[slot] = empty ? 0.0f : log_s - st.u / st.s;
  }
  ts_rank(lv, li, lists, k, tid - group * wpr * 32, wpr * 32, [&](int r, float v, uint32_t id) {
    if (p.top_ids) p.top_ids[slot * k + r] = id;
    if (p.top_log_probs) p.top_log_probs[slot * k + r] = empty ? -INFINITY : (v - st.m) - log_s;
  });
}

template <typename T>
int launch_typed(const DeviceCtx& dev, const TsParams& p, cudaStream_t stream) {
  // Tiles of the longest row.
  const int64_t vec = 16 / sizeof(T);
  const int64_t tiles = (p.columns + 2 * vec - 2) / vec / (32 * TS_UNR) + 1;
  int wpr = 1;
  while (wpr < TS_WARPS && wpr < tiles) wpr *= 2;
  int cluster = 1;
  if (wpr == TS_WARPS)
    while (cluster < TS_CLUSTER && p.rows * cluster * 2 <= dev.sm_count && tiles >= (int64_t)cluster * 2 * TS_WARPS)
      cluster *= 2;
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
    return cuda_error(cudaLaunchKernelEx(&cfg, token_scores_kernel<T, true>, p, (int)TS_WARPS), "token_scores launch");
  }
  const int64_t per = TS_WARPS / wpr;
  return cuda_error(launch_kernel(token_scores_kernel<T, false>, dim3((unsigned)((p.rows + per - 1) / per)),
                                  dim3(TS_THREADS), 0, stream, p, wpr),
                    "token_scores launch");
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
