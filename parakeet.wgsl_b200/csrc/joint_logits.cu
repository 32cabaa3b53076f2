// joint_logits.cu -- the transducer's joint for the emitted tokens of a batch
// of windows (the logits that token_scores reads):
//
//   hidden[r] = max(encoder[w, joint_frames[w, u]] + predictor[w, u], 0)
//   logits[r] = hidden[r] . weight + bias,   r = u plus the counts of the windows before w
//
// for u < counts[w].  The rows are ragged and their number is known on the
// device alone: every CTA sums the counts, and a persistent grid walks the
// tiles that exist.  Rows behind the last window's are not written; row_map
// gives each row's place [w, u] and row_count their number.
//
// Both precisions run on the tensor cores (tcgen05, f32 accumulators in TMEM).
// A tile is 128 rows times up to 256 (FP32: 128) columns, whose width follows
// from the number of row tiles, so that few rows still fill the SMs.  For every
// 128 bytes of inputs the threads gather, add, clamp and lay out their rows in
// shared memory (K-major, 128-byte swizzle), three steps ahead of the MMAs.
//
// FP16: hidden is rounded to f16, as the decoder rounds its joint inputs; the
// weight [inner, columns] arrives by TMA as it lies (the MN-major operand).
// FP32: an f32 is the sum of two tf32 values up to 2^-22 of itself, so logits
// are three tf32 products, hi hi + hi lo + lo hi (what is left out is 2^-22 of
// a product).  The threads split the weights too, and lay them out K-major.
// The MMA cuts its f32 sums, always towards zero, so one accumulator over all
// 3 inner / 8 products drifts (4e-5 in logits of 12 at inner 640): the two
// small products have an accumulator of their own, and the steps of the large
// one take turns on as many as TMEM's 512 columns hold.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int JL_THREADS = 512;
constexpr int JL_M = 128;          // rows per tile
constexpr int JL_STAGES = 3;
constexpr int JL_AHEAD = 3;        // steps whose inputs are on their way to a thread's registers
constexpr int JL_STAGE = 64 * 1024;  // FP16: A 16 KB, weights 32 KB; FP32: hi and lo of both, 16 KB each
constexpr int JL_B = 32 * 1024;    // the weights of a stage (FP16: at 16 KB)
constexpr int JL_BAR = JL_STAGES * JL_STAGE;  // full[stages], empty[stages], done
constexpr int JL_MISC = JL_BAR + 128;
constexpr int JL_SMEM = JL_MISC + 64 + 1024;  // + alignment slack
static_assert(JL_SMEM <= 232448, "shared memory budget");
template <typename T>
constexpr int jl_k() { return 128 / (int)sizeof(T); }  // inputs per step: 128 bytes
constexpr int JL_TMEM = 512;       // TMEM columns: FP32's accumulators (FP16: 256 are enough)
template <typename T>
constexpr int jl_n() { return sizeof(T) == 2 ? 256 : 128; }  // columns per tile, at most

struct JlParams {
  CUtensorMap tmap_w;  // weight [inner][columns] f16, box {64, 64}, 128-byte swizzle (reads past the edge are 0)
  const void* encoder;
  const float* predictor;
  const uint32_t* joint_frames;
  const uint32_t* counts;
  const void* weight;
  const float* bias;
  void* logits;
  uint32_t* row_map;
  uint32_t* row_count;
  unsigned int* status;
  int batch, frames, max_tokens, inner, columns;
};

struct JlRows {
  int place[JL_M];  // w * max_tokens + u of the tile's rows, -1 behind the last
  int frame[JL_M];  // w * frames + the token's frame
  int warp_sum[JL_THREADS / 32];
};

// The rows of window `w` start at `start`; `all` rows come before the next
// JL_THREADS windows.  Called by all threads, with consecutive windows.
struct JlSpan {
  int start, count, all;
};
__device__ __forceinline__ JlSpan jl_scan(const JlParams& p, JlRows& rows, int w, int base) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = w < p.batch ? (int)min(p.counts[w], (uint32_t)p.max_tokens) : 0;
  int incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) rows.warp_sum[warp] = incl;
  __syncthreads();
  int sum = lane < JL_THREADS / 32 ? rows.warp_sum[lane] : 0;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0);
  const int all = __reduce_add_sync(0xffffffffu, sum);
  __syncthreads();
  return JlSpan{base + before + incl - n, n, base + all};
}

// Fills the places and frames of rows [r0, r0 + JL_M); `span` holds the first
// JL_THREADS windows' rows.
__device__ __forceinline__ void jl_fill(const JlParams& p, JlRows& rows, int r0, JlSpan span) {
  const int tid = threadIdx.x;
  __syncthreads();  // the previous tile's places are read
  if (tid < JL_M) rows.place[tid] = -1;
  __syncthreads();
  for (int w0 = 0;; w0 += JL_THREADS) {
    const int w = w0 + tid;
    for (int r = max(span.start, r0); r < min(span.start + span.count, r0 + JL_M); ++r)
      rows.place[r - r0] = w * p.max_tokens + r - span.start;
    if (w0 + JL_THREADS >= p.batch) break;
    span = jl_scan(p, rows, w + JL_THREADS, span.all);
  }
  __syncthreads();
  if (tid < JL_M) {
    const int place = rows.place[tid];
    if (place >= 0)
      rows.frame[tid] = place / p.max_tokens * p.frames + (int)min(p.joint_frames[place], (uint32_t)(p.frames - 1));
  }
  __syncthreads();
}

__device__ __forceinline__ float jl_relu(float v) { return v < 0.0f ? 0.0f : v; }  // keeps NaN
__device__ __forceinline__ uint32_t jl_hidden2(uint32_t e, float p0, float p1) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&e));
  const __half2 h = __floats2half2_rn(jl_relu(f.x + p0), jl_relu(f.y + p1));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The leading 11 bits of v (a tf32 value), and the rest.  An infinite v has no rest.
__device__ __forceinline__ void jl_split(float v, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(v) & 0xffffe000u;
  if (v != v) hi = 0x7fc00000u;
  const float d = v - __uint_as_float(hi);
  lo = d == d ? __float_as_uint(d) : 0u;
}
__device__ __forceinline__ void jl_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, __half) {
  tc_mma_f16(d, a, b, idesc, accumulate);
}
__device__ __forceinline__ void jl_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, float) {
  tc_mma_tf32(d, a, b, idesc, accumulate);
}
// 16-byte chunk `c` of row `r` in a K-major block of 128-byte rows, swizzled.
__device__ __forceinline__ uint32_t jl_at(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}

// What a thread gathers for one step: chunk tid % 8 of rows tid / 8 + 64 i, and
// (FP32) inputs 4 (tid / 128) + 16 i .. + 3 of column tid % 128 of the weights.
template <typename T>
struct JlSlot;
template <>
struct JlSlot<__half> {
  uint4 e[2];
  float4 p[2][2];
};
template <>
struct JlSlot<float> {
  float4 e[2], p[2];
  float w[2][4];
};

template <typename T>
__global__ void __launch_bounds__(JL_THREADS, 1) joint_logits_kernel(const __grid_constant__ JlParams p) {
  pdl_entry();
  extern __shared__ uint8_t jl_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(jl_raw) + 1023) & ~uintptr_t(1023));
  __shared__ JlRows rows;
  constexpr bool F16 = sizeof(T) == 2;
  constexpr int K = jl_k<T>(), N = jl_n<T>(), EPC = 16 / sizeof(T);  // elements per chunk
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + JL_BAR);  // FP16: the stage's weights have landed
  uint64_t* empty = full + JL_STAGES;                         // the stage's MMAs have read it
  uint64_t* done = empty + JL_STAGES;                         // the tile's MMAs are complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + JL_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + JL_MISC + 4);
  if (tid == 0) {
    for (int i = 0; i < 2 * JL_STAGES + 1; ++i) mbar_init(&full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    if constexpr (F16) tma_prefetch_desc(&p.tmap_w);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, F16 ? N : JL_TMEM);
    tmem_relinquish();
  }
  JlSpan span = jl_scan(p, rows, tid, 0);
  int total = span.all;
  for (int w0 = JL_THREADS; w0 < p.batch; w0 += JL_THREADS) total = jl_scan(p, rows, w0 + tid, total).all;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (blockIdx.x == 0 && tid == 0) *p.row_count = (uint32_t)total;

  const int mtiles = (total + JL_M - 1) / JL_M;
  // Columns per tile: as few tiles as N columns allow, more while SMs are idle.
  int ntiles = max((p.columns + N - 1) / N, min((p.columns + 63) / 64, (int)gridDim.x / max(mtiles, 1)));
  const int bn = ((p.columns + ntiles - 1) / ntiles + 15) / 16 * 16;
  ntiles = (p.columns + bn - 1) / bn;
  const int boxes = (bn + 63) / 64;
  const uint32_t idesc = (F16 ? umma_idesc_f16(JL_M, 0, 0, /*weight, MN-major*/ 1) : umma_idesc_tf32(JL_M, 0)) |
                         ((uint32_t)(bn >> 3) << 17);
  const int steps = (p.inner + K - 1) / K;
  // FP32: accumulators, `pitch` columns apart; the first is the small products'.
  const int pitch = (bn + 31) / 32 * 32;
  const int turns = F16 ? 1 : min(min(8, JL_TMEM / pitch) - 1, steps);
  const int chunk = tid & 7, rbase = tid >> 3;
  const T* enc = static_cast<const T*>(p.encoder);

  uint32_t used = 0, tiles_done = 0;  // stages used, tiles finished (the same in all threads)
  // `good`: this thread's waits ended in time; `ok`: all threads' did, as of the
  // last barrier (the same in all threads, so all meet at the same barriers).
  bool ok = true, good = true;
  for (int tile = blockIdx.x; tile < mtiles * ntiles && ok; tile += gridDim.x) {
    const int r0 = tile / ntiles * JL_M, n0 = tile % ntiles * bn;
    jl_fill(p, rows, r0, span);
    if (n0 == 0 && tid < JL_M && rows.place[tid] >= 0) p.row_map[r0 + tid] = (uint32_t)rows.place[tid];
    const T* es[2];
    const float* ps[2];
    bool live[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int place = rows.place[rbase + 64 * i];
      live[i] = place >= 0;
      es[i] = enc + (size_t)(live[i] ? rows.frame[rbase + 64 * i] : 0) * p.inner + chunk * EPC;
      ps[i] = p.predictor + (size_t)(live[i] ? place : 0) * p.inner + chunk * EPC;
    }
    const int wn = tid & 127, wk = tid >> 7;  // FP32: this thread's column and inputs of a step's weights
    const float* ws = static_cast<const float*>(p.weight) + (size_t)(4 * wk) * p.columns + n0 + wn;
    const bool wlive = wn < bn && n0 + wn < p.columns;
    auto fetch = [&](JlSlot<T>& s, int kb) {
      const int k = kb * K;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = live[i] && k + chunk * EPC < p.inner;
        if constexpr (F16) {
          s.e[i] = make_uint4(0u, 0u, 0u, 0u);
          s.p[i][0] = s.p[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (in) {
            s.e[i] = *reinterpret_cast<const uint4*>(es[i] + k);
            s.p[i][0] = reinterpret_cast<const float4*>(ps[i] + k)[0];
            s.p[i][1] = reinterpret_cast<const float4*>(ps[i] + k)[1];
          }
        } else {
          s.e[i] = s.p[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (in) {
            s.e[i] = *reinterpret_cast<const float4*>(es[i] + k);
            s.p[i] = *reinterpret_cast<const float4*>(ps[i] + k);
          }
          // inner is a multiple of 32, a step's inputs are all inside
#pragma unroll
          for (int j = 0; j < 4; ++j) s.w[i][j] = wlive ? __ldg(ws + (size_t)(k + 16 * i + j) * p.columns) : 0.0f;
        }
      }
    };
    JlSlot<T> slot[JL_AHEAD];
#pragma unroll
    for (int d = 0; d < JL_AHEAD; ++d)
      if (d < steps) fetch(slot[d], d);
    for (int kb0 = 0; kb0 < steps && ok; kb0 += JL_AHEAD) {
#pragma unroll
      for (int d = 0; d < JL_AHEAD; ++d) {
        const int kb = kb0 + d;
        if (kb >= steps || !ok) break;
        const uint32_t st = used % JL_STAGES, use = used / JL_STAGES;
        uint8_t* stage = sm + st * JL_STAGE;
        if (use > 0 && good) good = mbar_wait(&empty[st], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
        if constexpr (F16) {
          if (tid == 0 && good) {
            mbar_arrive_expect_tx(&full[st], (uint32_t)boxes * K * 128);
            for (int b = 0; b < boxes; ++b)
              tma_load_2d(stage + JL_B / 2 + b * K * 128, &p.tmap_w, &full[st], n0 + 64 * b, kb * K);
          }
        }
        JlSlot<T>& s = slot[d];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t at = jl_at(rbase + 64 * i, chunk);
          if constexpr (F16) {
            uint4 o;
            o.x = jl_hidden2(s.e[i].x, s.p[i][0].x, s.p[i][0].y);
            o.y = jl_hidden2(s.e[i].y, s.p[i][0].z, s.p[i][0].w);
            o.z = jl_hidden2(s.e[i].z, s.p[i][1].x, s.p[i][1].y);
            o.w = jl_hidden2(s.e[i].w, s.p[i][1].z, s.p[i][1].w);
            *reinterpret_cast<uint4*>(stage + at) = o;
          } else {
            uint4 hi, lo;
            jl_split(jl_relu(s.e[i].x + s.p[i].x), hi.x, lo.x);
            jl_split(jl_relu(s.e[i].y + s.p[i].y), hi.y, lo.y);
            jl_split(jl_relu(s.e[i].z + s.p[i].z), hi.z, lo.z);
            jl_split(jl_relu(s.e[i].w + s.p[i].w), hi.w, lo.w);
            *reinterpret_cast<uint4*>(stage + at) = hi;
            *reinterpret_cast<uint4*>(stage + JL_M * 128 + at) = lo;
            if (wn < bn) {
              const uint32_t wat = jl_at(wn, wk + 4 * i);
              jl_split(s.w[i][0], hi.x, lo.x);
              jl_split(s.w[i][1], hi.y, lo.y);
              jl_split(s.w[i][2], hi.z, lo.z);
              jl_split(s.w[i][3], hi.w, lo.w);
              *reinterpret_cast<uint4*>(stage + JL_B + wat) = hi;
              *reinterpret_cast<uint4*>(stage + JL_B + N * 128 + wat) = lo;
            }
          }
        }
        if (kb + JL_AHEAD < steps) fetch(s, kb + JL_AHEAD);
        fence_proxy_async_smem();
        ++used;
        ok = __syncthreads_and(good) != 0;
        if (tid == 0 && ok) {
          if constexpr (F16) good = mbar_wait(&full[st], use & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_TMA);
          if (good) {
            tc_fence_after();
            const uint32_t a = smem_addr(stage), b = smem_addr(stage + (F16 ? JL_B / 2 : JL_B));
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {  // 32 bytes of inputs each
              const uint64_t ah = umma_smem_desc(a + ks * 32, 16, 1024, 2);
              if constexpr (F16) {
                jl_mma(tmem, ah, umma_smem_desc(b + ks * 2048, K * 128, 1024, 2), idesc, kb > 0 || ks > 0 ? 1u : 0u, T());
              } else {
                const uint64_t al = umma_smem_desc(a + JL_M * 128 + ks * 32, 16, 1024, 2);
                const uint64_t bh = umma_smem_desc(b + ks * 32, 16, 1024, 2);
                const uint64_t bl = umma_smem_desc(b + N * 128 + ks * 32, 16, 1024, 2);
                jl_mma(tmem, al, bh, idesc, kb > 0 || ks > 0 ? 1u : 0u, T());
                jl_mma(tmem, ah, bl, idesc, 1u, T());
                jl_mma(tmem + (uint32_t)((1 + kb % turns) * pitch), ah, bh, idesc, kb >= turns || ks > 0 ? 1u : 0u, T());
              }
            }
            tc_commit(&empty[st]);
            if (kb + 1 == steps) tc_commit(done);
          }
        }
      }
    }
    if (ok && good) good = mbar_wait(done, tiles_done & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_EPILOGUE);
    ok = __syncthreads_and(good) != 0;
    if (!ok) break;
    ++tiles_done;
    tc_fence_after();
    // Warp w reads TMEM lanes 32 (w % 4) .. + 31, columns 32 (w / 4) + 128 i .. + 31.
    const int r = (warp & 3) * 32 + lane;
    const bool mine = rows.place[r] >= 0;
    T* out = static_cast<T*>(p.logits) + (size_t)(r0 + r) * p.columns;
    for (int c = (warp >> 2) * 32; c < bn; c += 128) {
      uint32_t v[32];
      const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c;
      tc_ld_32x32b_x32(at, v);
      tc_wait_ld();
      if constexpr (!F16) {
        for (int a = 1; a <= turns; ++a) {
          uint32_t u[32];
          tc_ld_32x32b_x32(at + (uint32_t)(a * pitch), u);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + c + 8 * q;
        if (mine && c + 8 * q < bn && n < p.columns) {  // columns are a multiple of 8
          float b[8] = {};
          if (p.bias) {
            *reinterpret_cast<float4*>(b) = __ldg(reinterpret_cast<const float4*>(p.bias + n));
            *reinterpret_cast<float4*>(b + 4) = __ldg(reinterpret_cast<const float4*>(p.bias + n + 4));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) b[j] += __uint_as_float(v[8 * q + j]);
          if constexpr (F16) {
            __half2 h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(b[2 * j], b[2 * j + 1]);
            *reinterpret_cast<uint4*>(out + n) = *reinterpret_cast<const uint4*>(h);
          } else {
            *reinterpret_cast<float4*>(out + n) = make_float4(b[0], b[1], b[2], b[3]);
            *reinterpret_cast<float4*>(out + n + 4) = make_float4(b[4], b[5], b[6], b[7]);
          }
        }
      }
    }
    tc_fence_before();
    __syncthreads();  // the accumulators are read
    tc_fence_after();
  }
  // Unwind: the loads and MMAs that this CTA issued are complete before shared
  // memory and TMEM are released (at once, unless a wait expired).
  __syncthreads();
  if (tid == 0 && *abort_flag) {
    for (uint32_t s = 0; s < JL_STAGES; ++s) {
      const uint32_t uses = used > s ? (used - s + JL_STAGES - 1) / JL_STAGES : 0;
      if (F16 && uses > 0) mbar_wait_drain(&full[s], (uses - 1) & 1, p.status);
      if (uses > 1) mbar_wait_drain(&empty[s], (uses - 2) & 1, p.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, F16 ? N : JL_TMEM);
  }
}

template <typename T>
int launch_typed(const DeviceCtx& dev, const JlParams& p, cudaStream_t stream) {
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(joint_logits_kernel<T>), JL_SMEM);
  if (st != PK_OK) return st;
  const int64_t tiles = ((int64_t)p.batch * p.max_tokens + JL_M - 1) / JL_M * ((p.columns + 63) / 64);
  return cuda_error(launch_kernel(joint_logits_kernel<T>, dim3((unsigned)std::min<int64_t>(tiles, dev.sm_count)),
                                  dim3(JL_THREADS), JL_SMEM, stream, p),
                    "joint_logits launch");
}

}  // namespace

int launch_joint_logits(const DeviceCtx& dev, const pk_joint_logits_desc& d, cudaStream_t stream) {
  JlParams p;
  p.encoder = d.encoder_projected;
  p.predictor = d.predictor;
  p.joint_frames = d.joint_frames;
  p.counts = d.counts;
  p.weight = d.weight;
  p.bias = d.bias;
  p.logits = d.logits;
  p.row_map = d.row_map;
  p.row_count = d.row_count;
  p.status = dev.status;
  p.batch = d.batch;
  p.frames = d.frames;
  p.max_tokens = d.max_tokens;
  p.inner = (int)d.inner;
  p.columns = (int)d.columns;
  if (d.precision == PK_FP32) return launch_typed<float>(dev, p, stream);
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(dev.encode_tiled);
  const cuuint64_t dims[2] = {(cuuint64_t)p.columns, (cuuint64_t)p.inner};
  const cuuint64_t strides[1] = {(cuuint64_t)p.columns * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)jl_k<__half>()}, unit[2] = {1, 1};
  if (!encode ||
      encode(&p.tmap_w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(d.weight), dims, strides, box, unit,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return set_error(PK_E_CUDA, "cuTensorMapEncodeTiled failed (joint weight)");
  return launch_typed<__half>(dev, p, stream);
}

}  // namespace pk
