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
// from the number of row tiles, so that few rows still fill the SMs.  16 warps
// gather, add, clamp and lay out 128 bytes of inputs a step in shared memory
// (K-major, 128-byte swizzle), their loads a step ahead; one warp issues the
// MMAs, one the weights' loads, so that none of the three waits for another's
// instructions (with one thread doing both between barriers a step took 2400
// cycles, 900 of them the MMAs' issue and 800 the loads').
//
// 30 rows (1 window; 640 x 1032) f16 8.4 us: 33 tiles, latency from start to end.
// 1531 rows (32 windows) f16 10.9 us: 144 tiles, one per SM, of which 12 gather the
// same rows each; reading everything once takes 1.6.  3584 rows (40 windows) f32 48 us, bound by shared memory: a step of 32 inputs
// writes 64 KB of split operands there, reads 96 KB of them for its MMAs and
// moves 32 KB of weights in and out, 1540 of its 2100 cycles.
//
// FP16: hidden is rounded to f16, as the decoder rounds its joint inputs; the
// weight [inner, columns] arrives by TMA as it lies (the MN-major operand).
// FP32: an f32 is the sum of two tf32 values up to 2^-22 of itself, so logits
// are three tf32 products, hi hi + hi lo + lo hi (what is left out is 2^-22 of
// a product).  The threads split the weights too, from a TMA copy of them, and
// lay them out K-major.
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

constexpr int JL_ROWS = 512;       // threads that lay out rows and store logits
constexpr int JL_M = 128;          // rows per tile
constexpr int JL_BAR = 192 * 1024;  // after the stages: the barriers
constexpr int JL_MISC = JL_BAR + 256;
constexpr int JL_SMEM = JL_MISC + 64 + 1024;  // + alignment slack
static_assert(JL_SMEM <= 232448, "shared memory budget");
// A stage: FP16 the rows (16 KB) and the weights (32 KB), FP32 hi and lo of both (16 KB each).
template <typename T>
constexpr int jl_stages() { return sizeof(T) == 2 ? 4 : 2; }
template <typename T>
constexpr int jl_stage() { return sizeof(T) == 2 ? 48 * 1024 : 64 * 1024; }
template <typename T>
constexpr int jl_b() { return sizeof(T) == 2 ? 16 * 1024 : 32 * 1024; }  // the weights of a stage
// FP32: the weights as they lie, [32 inputs][128 columns], behind the stages.
constexpr int JL_RAW = 128 * 1024, JL_RAW_STAGES = 4, JL_RAW_STAGE = 16 * 1024;
static_assert(JL_RAW == jl_stages<float>() * jl_stage<float>() && JL_RAW + JL_RAW_STAGES * JL_RAW_STAGE <= JL_BAR &&
              jl_stages<__half>() * jl_stage<__half>() <= JL_BAR, "stages fit");
template <typename T>
constexpr int jl_k() { return 128 / (int)sizeof(T); }  // inputs per step: 128 bytes
constexpr int JL_TMEM = 512;       // TMEM columns: FP32's accumulators (FP16: 256 are enough)
// Row threads.  A warp each for the MMAs and the weights' loads comes after them.
template <typename T>
constexpr int jl_n() { return sizeof(T) == 2 ? 256 : 128; }  // columns per tile, at most

struct JlParams {
  // weight [inner][columns]; reads past the edge are 0.  FP16: box {64, 64},
  // 128-byte swizzle; FP32: box {128, 32}, as it lies.
  CUtensorMap tmap_w;
  const void* encoder;
  const float* predictor;
  const uint32_t* joint_frames;
  const uint32_t* counts;
  const float* bias;
  void* logits;
  uint32_t* row_map;
  uint32_t* row_count;
  unsigned int* status;
  int batch, frames, max_tokens, inner, columns;
};

struct JlRows {
  int place[JL_M];     // w * max_tokens + u of the tile's rows, -1 behind the last
  int frame[JL_M];     // w * frames + the token's frame
  int start[JL_ROWS];  // the first row of each of JL_ROWS consecutive windows
  alignas(16) float bias[JL_ROWS];  // of the tile's columns
  int warp_sum[JL_ROWS / 32];
};

template <int ROWS>
__device__ __forceinline__ void jl_rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(ROWS) : "memory"); }

// The row threads: windows w0 + tid, whose rows come after `base` others.  Fills
// rows.start and returns the number of rows up to the last of these windows.
template <int ROWS>
__device__ __forceinline__ int jl_scan(const JlParams& p, JlRows& rows, int w0, int base) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = w0 + tid < p.batch ? (int)min(p.counts[w0 + tid], (uint32_t)p.max_tokens) : 0;
  int incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) rows.warp_sum[warp] = incl;
  jl_rows_sync<ROWS>();
  const int sum = lane < ROWS / 32 ? rows.warp_sum[lane] : 0;
  rows.start[tid] = base + __reduce_add_sync(0xffffffffu, lane < warp ? sum : 0) + incl - n;
  jl_rows_sync<ROWS>();
  return base + __reduce_add_sync(0xffffffffu, sum);
}

// The row threads: places and frames of rows [r0, r0 + JL_M) and the bias from
// column n0 on.  `all`: rows of the first ROWS windows, whose starts
// are in rows.start where they are all the windows.
template <int ROWS>
__device__ __forceinline__ void jl_fill(const JlParams& p, JlRows& rows, int r0, int n0, int all) {
  const int tid = threadIdx.x;
  jl_rows_sync<ROWS>();  // the previous tile's are read
  rows.bias[tid] = p.bias && n0 + tid < p.columns ? __ldg(p.bias + n0 + tid) : 0.0f;
  int place = -1;
  int base = 0;
  if (p.batch > ROWS) all = jl_scan<ROWS>(p, rows, 0, 0);
  for (int w0 = 0;; w0 += ROWS) {
    const int r = r0 + tid;
    if (tid < JL_M && r >= base && r < all) {
      // The last window that starts at or before r (windows without rows start where the next does).
      int w = 0;
#pragma unroll
      for (int step = ROWS / 2; step > 0; step >>= 1)
        if (rows.start[w + step] <= r) w += step;
      place = (w0 + w) * p.max_tokens + r - rows.start[w];
    }
    if (w0 + ROWS >= p.batch) break;
    jl_rows_sync<ROWS>();
    base = all;
    all = jl_scan<ROWS>(p, rows, w0 + ROWS, base);
  }
  if (tid < JL_M) {
    rows.place[tid] = place;
    if (place >= 0)
      rows.frame[tid] = place / p.max_tokens * p.frames + (int)min(p.joint_frames[place], (uint32_t)(p.frames - 1));
  }
  jl_rows_sync<ROWS>();
}

__device__ __forceinline__ float jl_relu(float v) { return v < 0.0f ? 0.0f : v; }  // keeps NaN
__device__ __forceinline__ uint32_t jl_hidden2(uint32_t e, float p0, float p1) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&e));
  const __half2 h = __floats2half2_rn(jl_relu(f.x + p0), jl_relu(f.y + p1));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The leading 11 bits of v (a tf32 value), and the rest (NaN for an infinite v).
__device__ __forceinline__ void jl_split(float v, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(v) & 0xffffe000u;
  lo = __float_as_uint(v - __uint_as_float(hi));
}
// 16-byte chunk `c` of row `r` in a K-major block of 128-byte rows, swizzled.
__device__ __forceinline__ uint32_t jl_at(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}

// What a thread gathers for one step: chunk tid % 8 of every 64th row.
constexpr int JL_TASKS = JL_M * 8 / JL_ROWS;
template <typename T>
struct JlSlot;
template <>
struct JlSlot<__half> {
  uint4 e[JL_TASKS];
  float4 p[JL_TASKS][2];
};
template <>
struct JlSlot<float> {
  float4 e[JL_TASKS], p[JL_TASKS];
};

template <typename T>
__global__ void __launch_bounds__(JL_ROWS + 64, 1) joint_logits_kernel(const __grid_constant__ JlParams p) {
  pdl_entry();
  extern __shared__ uint8_t jl_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(jl_raw) + 1023) & ~uintptr_t(1023));
  __shared__ JlRows rows;
  constexpr bool F16 = sizeof(T) == 2;
  constexpr int ROWS = JL_ROWS, TASKS = JL_TASKS;
  constexpr int K = jl_k<T>(), N = jl_n<T>(), EPC = 16 / sizeof(T);  // elements per chunk
  constexpr int STAGES = jl_stages<T>(), STAGE = jl_stage<T>(), B = jl_b<T>();
  constexpr int RAW = F16 ? STAGES : JL_RAW_STAGES;  // the weights' stages (FP16: the MMAs')
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + JL_BAR);  // the stage's rows are laid out
  uint64_t* weights = full + STAGES;                          // the weights' stage has landed
  uint64_t* unpacked = weights + RAW;                         // FP32: the row threads have read it
  uint64_t* empty = unpacked + RAW;                           // the stage's MMAs have read it
  uint64_t* done = empty + STAGES;                            // the tile's MMAs are complete
  uint64_t* taken = done + 1;                                 // the tile's accumulators are read
  uint64_t* drain = taken + 1;                                // every MMA issued is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + JL_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + JL_MISC + 4);
  int* totals = reinterpret_cast<int*>(sm + JL_MISC + 8);
  if (tid == ROWS) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], ROWS / 32);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&weights[i], 1);
      mbar_init(&unpacked[i], ROWS / 32);
    }
    mbar_init(done, 1);
    mbar_init(taken, ROWS / 32);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_w);
  }
  if (warp == ROWS / 32 + 1) {
    tmem_alloc(tmem_slot, F16 ? N : JL_TMEM);
    tmem_relinquish();
  }
  if (tid < ROWS) {
    const int all = jl_scan<ROWS>(p, rows, 0, 0);
    int total = all;
    for (int w0 = ROWS; w0 < p.batch; w0 += ROWS) total = jl_scan<ROWS>(p, rows, w0, total);
    if (tid == 0) {
      totals[0] = total;
      totals[1] = all;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = totals[0];
  if (blockIdx.x == 0 && tid == 0) *p.row_count = (uint32_t)total;

  const int mtiles = (total + JL_M - 1) / JL_M;
  // Columns per tile, in units of 16: as few tiles as N columns allow, more while
  // SMs are idle.  FP16 shares the units out evenly.  FP32 fills its tiles: the 8
  // columns that 1032 leave to a ninth one cost less there than nine equal tiles
  // (and less than a 144-column tile among eight: 40 windows 54 against 51 us).
  const int units = (p.columns + 15) / 16;
  int ntiles = max((units + N / 16 - 1) / (N / 16), min((p.columns + 31) / 32, (int)gridDim.x / max(mtiles, 1)));
  const int even = units / ntiles, rest = units % ntiles, most = even + (rest > 0 ? 1 : 0);
  if (!F16) ntiles = (units + most - 1) / most;
  auto tile_start = [&](int t) { return 16 * (F16 ? t * even + min(t, rest) : t * most); };
  auto tile_width = [&](int t) { return 16 * (F16 ? t < rest ? most : even : min(most, units - t * most)); };
  const int tiles = mtiles * ntiles;
  const int steps = (p.inner + K - 1) / K;
  // FP32: accumulators, `pitch` columns apart; the first is the small products'.
  const int pitch = (16 * most + 31) / 32 * 32;
  const int turns = F16 ? 1 : min(min(8, JL_TMEM / pitch) - 1, steps);

  // Every role walks the same tiles and steps; step number `used` has stage
  // used % STAGES.  A wait that expires raises the abort flag and ends the
  // roles' loops; they meet again behind them.
  uint32_t used = 0;
  if (warp == ROWS / 32) {
    // ------------------------------------------------------------ MMAs
    if (elect_one()) {
      uint32_t turn = 0;
      bool good = true;
      for (int tile = blockIdx.x; tile < tiles && good; tile += gridDim.x, ++turn) {
        const uint32_t idesc = (F16 ? umma_idesc_f16(JL_M, 0, 0, /*weight, MN-major*/ 1) : umma_idesc_tf32(JL_M, 0)) |
                               ((uint32_t)(tile_width(tile % ntiles) >> 3) << 17);
        if (turn > 0) good = mbar_wait(taken, (turn - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
        for (int kb = 0; kb < steps && good; ++kb, ++used) {
          const uint32_t st = used % STAGES, use = used / STAGES;
          good = mbar_wait(&full[st], use & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_DECODE);
          if (F16 && good) good = mbar_wait(&weights[st], use & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_TMA);
          if (!good) break;
          tc_fence_after();
          // 32 bytes of inputs an MMA: 2 in a K-major descriptor's address, 128 (16 rows) in an MN-major one's.
          const uint8_t* stage = sm + st * STAGE;
          const uint64_t ah = umma_smem_desc(smem_addr(stage), 16, 1024, 2);
          const uint64_t bh = F16 ? umma_smem_desc(smem_addr(stage + B), K * 128, 1024, 2)
                                  : umma_smem_desc(smem_addr(stage + B), 16, 1024, 2);
          const uint32_t first = kb > 0 ? 1u : 0u;
          if constexpr (F16) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) tc_mma_f16(tmem, ah + 2 * ks, bh + 128 * ks, idesc, ks > 0 ? 1u : first);
          } else {
            const uint64_t al = ah + JL_M * 128 / 16, bl = bh + N * 128 / 16;
            const uint32_t large = tmem + (uint32_t)((1 + kb % turns) * pitch);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              tc_mma_tf32(tmem, al + 2 * ks, bh + 2 * ks, idesc, ks > 0 ? 1u : first);
              tc_mma_tf32(tmem, ah + 2 * ks, bl + 2 * ks, idesc, 1u);
              tc_mma_tf32(large, ah + 2 * ks, bh + 2 * ks, idesc, kb >= turns || ks > 0 ? 1u : 0u);
            }
          }
          tc_commit(&empty[st]);
        }
        if (good) tc_commit(done);
      }
      // The MMAs issued are complete before the roles meet and TMEM is given back, whoever gave up on them: a row
      // warp's wait may expire where none of this thread's did.
      tc_commit(drain);
      mbar_wait_drain(drain, 0, p.status);
    }
  } else if (warp == ROWS / 32 + 1) {
    // ------------------------------------------------------------ weights
    if (elect_one()) {
      uint64_t* read = F16 ? empty : unpacked;
      bool good = true;
      for (int tile = blockIdx.x; tile < tiles && good; tile += gridDim.x) {
        const int n0 = tile_start(tile % ntiles), boxes = F16 ? (tile_width(tile % ntiles) + 63) / 64 : 1;
        for (int kb = 0; kb < steps; ++kb, ++used) {
          const uint32_t st = used % RAW, use = used / RAW;
          if (use > 0) good = mbar_wait(&read[st], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
          if (!good) break;
          mbar_arrive_expect_tx(&weights[st], (uint32_t)(F16 ? boxes * K * 128 : JL_RAW_STAGE));
          uint8_t* dst = F16 ? sm + st * STAGE + B : sm + JL_RAW + st * JL_RAW_STAGE;
          for (int b = 0; b < boxes; ++b) tma_load_2d(dst + b * K * 128, &p.tmap_w, &weights[st], n0 + 64 * b, kb * K);
        }
      }
      // Unwind: the loads issued have landed before the roles meet.
      for (uint32_t s = 0; s < RAW; ++s)
        if (used > s) mbar_wait_drain(&weights[s], (used - s - 1) / RAW & 1, p.status);
    }
  } else {
    // ------------------------------------------------------------ rows and logits
    const int chunk = tid & 7, rbase = tid >> 3;
    const T* enc = static_cast<const T*>(p.encoder);
    const int all = totals[1];
    uint32_t turn = 0;
    bool good = true;  // of this warp
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
      const int r0 = tile / ntiles * JL_M, n0 = tile_start(tile % ntiles), bn = tile_width(tile % ntiles);
      jl_fill<ROWS>(p, rows, r0, n0, all);
      if (n0 == 0 && tid < JL_M && rows.place[tid] >= 0) p.row_map[r0 + tid] = (uint32_t)rows.place[tid];
      const T* es[TASKS];
      const float* ps[TASKS];
      bool live[TASKS];
#pragma unroll
      for (int i = 0; i < TASKS; ++i) {
        const int place = rows.place[rbase + ROWS / 8 * i];
        live[i] = place >= 0;
        es[i] = enc + (size_t)(live[i] ? rows.frame[rbase + ROWS / 8 * i] : 0) * p.inner + chunk * EPC;
        ps[i] = p.predictor + (size_t)(live[i] ? place : 0) * p.inner + chunk * EPC;
      }
      const int wn = tid & 127, wk = tid >> 7;  // FP32: this thread's column and inputs of a step's weights
      auto fetch = [&](JlSlot<T>& s, int kb) {
        const int k = kb * K;
#pragma unroll
        for (int i = 0; i < TASKS; ++i) {
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
          }
        }
      };
      // One step ahead: with the loads of two in registers a step waits for the
      // younger ones too (32 windows f16 10.9 us, with two 12.0).
      JlSlot<T> s;
      fetch(s, 0);
      for (int kb = 0; kb < steps; ++kb) {
        const uint32_t st = used % STAGES, use = used / STAGES;
        uint8_t* stage = sm + st * STAGE;
        if (use > 0 && good) good = mbar_wait(&empty[st], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
        if (!F16 && good) good = mbar_wait(&weights[used % RAW], used / RAW & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_TMA);
        good = __all_sync(0xffffffffu, good);
        if (good) {
#pragma unroll
          for (int i = 0; i < TASKS; ++i) {
            const uint32_t at = jl_at(rbase + ROWS / 8 * i, chunk);
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
            }
          }
          if constexpr (!F16) {
            const float* raw = reinterpret_cast<const float*>(sm + JL_RAW + used % RAW * JL_RAW_STAGE) + wn;
            if (wn < bn) {
#pragma unroll
              for (int i = 0; i < K / 16; ++i) {  // 16 inputs at a time over the row threads
                float w[4];
                uint4 hi, lo;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = raw[(4 * wk + 16 * i + j) * N];
                jl_split(w[0], hi.x, lo.x);
                jl_split(w[1], hi.y, lo.y);
                jl_split(w[2], hi.z, lo.z);
                jl_split(w[3], hi.w, lo.w);
                const uint32_t wat = jl_at(wn, wk + 4 * i);
                *reinterpret_cast<uint4*>(stage + B + wat) = hi;
                *reinterpret_cast<uint4*>(stage + B + N * 128 + wat) = lo;
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&unpacked[used % RAW]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[st]);
        }
        if (kb + 1 < steps) fetch(s, kb + 1);
        ++used;
      }
      if (good) good = mbar_wait(done, turn & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_EPILOGUE);
      good = __all_sync(0xffffffffu, good);
      if (good) {
        tc_fence_after();
        // Warp w reads TMEM lanes 32 (w % 4) .. + 31, columns 16 (w / 4) + ROWS / 8 i .. + 15.
        const int r = (warp & 3) * 32 + lane;
        const bool mine = rows.place[r] >= 0;
        T* out = static_cast<T*>(p.logits) + (size_t)(r0 + r) * p.columns;
        for (int c = (warp >> 2) * 16; c < bn; c += ROWS / 8) {
          uint32_t v[16];
          const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c;
          tc_ld_32x32b_x16(at, v);
          tc_wait_ld();
          if constexpr (!F16) {
            for (int a = 1; a <= turns; ++a) {
              uint32_t u[16];
              tc_ld_32x32b_x16(at + (uint32_t)(a * pitch), u);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
            }
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int n = n0 + c + 8 * q;
            if (mine && n < p.columns) {  // columns are a multiple of 8, a tile's of 16
              float b[8];
              *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(rows.bias + c + 8 * q);
              *reinterpret_cast<float4*>(b + 4) = *reinterpret_cast<const float4*>(rows.bias + c + 8 * q + 4);
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
        __syncwarp();
        if (lane == 0) mbar_arrive(taken);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ROWS / 32 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, F16 ? N : JL_TMEM);
  }
}

template <typename T>
int launch_typed(const DeviceCtx& dev, const JlParams& p, cudaStream_t stream) {
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(joint_logits_kernel<T>), JL_SMEM);
  if (st != PK_OK) return st;
  const int64_t tiles = ((int64_t)p.batch * p.max_tokens + JL_M - 1) / JL_M * ((p.columns + 31) / 32);
  return cuda_error(launch_kernel(joint_logits_kernel<T>, dim3((unsigned)std::min<int64_t>(tiles, dev.sm_count)),
                                  dim3(JL_ROWS + 64), JL_SMEM, stream, p),
                    "joint_logits launch");
}

}  // namespace

int launch_joint_logits(const DeviceCtx& dev, const pk_joint_logits_desc& d, cudaStream_t stream) {
  JlParams p;
  p.encoder = d.encoder_projected;
  p.predictor = d.predictor;
  p.joint_frames = d.joint_frames;
  p.counts = d.counts;
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
  const bool f16 = d.precision == PK_FP16;
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(dev.encode_tiled);
  const cuuint64_t dims[2] = {(cuuint64_t)p.columns, (cuuint64_t)p.inner};
  const cuuint64_t strides[1] = {(cuuint64_t)p.columns * (f16 ? 2 : 4)};
  const cuuint32_t box16[2] = {64, (cuuint32_t)jl_k<__half>()}, box32[2] = {(cuuint32_t)jl_n<float>(), (cuuint32_t)jl_k<float>()};
  const cuuint32_t unit[2] = {1, 1};
  if (!encode ||
      encode(&p.tmap_w, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2,
             const_cast<void*>(d.weight), dims, strides, f16 ? box16 : box32, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
             f16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return set_error(PK_E_CUDA, "cuTensorMapEncodeTiled failed (joint weight)");
  if (!f16) return launch_typed<float>(dev, p, stream);
  return launch_typed<__half>(dev, p, stream);
}

}  // namespace pk
