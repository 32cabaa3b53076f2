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
// FP16: hidden is rounded to f16 (as the decoder rounds its joint inputs) and
// multiplied on the tensor cores (tcgen05, f32 accumulators in TMEM).  A tile
// is 128 rows times at most 256 columns: the threads gather, add, clamp and
// round 64 inputs of the rows into shared memory (K-major, 128-byte swizzle)
// while the previous 64 are multiplied; the weight [inner, columns] arrives by
// TMA as it lies (the MN-major operand).  The column width follows from the
// number of row tiles, so that few rows still fill the SMs.  FP32: FMA chains
// on the CUDA cores, 128 x 64 outputs per CTA.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int JL_THREADS = 256;
constexpr int JL_M = 128;          // rows per tile
constexpr int JL_K = 64;           // inputs per stage
constexpr int JL_N = 256;          // columns per tile, at most
constexpr int JL_STAGES = 3;
constexpr int JL_A = 0;                                    // [stage][128 rows x 128 B]
constexpr int JL_B = JL_STAGES * JL_M * 128;               // [stage][column block of 64][64 inputs x 128 B]
constexpr int JL_BSTAGE = JL_N / 64 * JL_K * 128;
constexpr int JL_BAR = JL_B + JL_STAGES * JL_BSTAGE;       // full[stages], empty[stages], done
constexpr int JL_MISC = JL_BAR + 128;
constexpr int JL_SMEM = JL_MISC + 64 + 1024;               // + alignment slack
static_assert(JL_SMEM <= 232448, "shared memory budget");

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

// Sums the counts (all threads; returns the number of rows) and, where r0 >= 0,
// fills the places of rows [r0, r0 + JL_M).
__device__ int jl_rows(const JlParams& p, JlRows& rows, int r0) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __syncthreads();  // the previous tile's places are read
  if (r0 >= 0 && tid < JL_M) rows.place[tid] = -1;
  int base = 0;
  for (int w0 = 0; w0 < p.batch; w0 += JL_THREADS) {
    const int w = w0 + tid;
    const int n = w < p.batch ? (int)min(p.counts[w], (uint32_t)p.max_tokens) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) rows.warp_sum[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < JL_THREADS / 32; ++i) {
      if (i < warp) before += rows.warp_sum[i];
      all += rows.warp_sum[i];
    }
    const int start = base + before + incl - n;
    if (r0 >= 0)
      for (int r = max(start, r0); r < min(start + n, r0 + JL_M); ++r) rows.place[r - r0] = w * p.max_tokens + r - start;
    base += all;
    __syncthreads();
  }
  if (r0 >= 0 && tid < JL_M) {
    const int place = rows.place[tid];
    if (place >= 0)
      rows.frame[tid] =
          place / p.max_tokens * p.frames + (int)min(p.joint_frames[place], (uint32_t)(p.frames - 1));
  }
  __syncthreads();
  return base;
}

__device__ __forceinline__ uint32_t jl_hidden2(uint32_t e, float p0, float p1) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&e));
  const float a = f.x + p0, b = f.y + p1;
  const __half2 h = __floats2half2_rn(a < 0.0f ? 0.0f : a, b < 0.0f ? 0.0f : b);  // keeps NaN
  return *reinterpret_cast<const uint32_t*>(&h);
}

__global__ void __launch_bounds__(JL_THREADS, 1) joint_logits_umma_kernel(const __grid_constant__ JlParams p) {
  pdl_entry();
  extern __shared__ uint8_t jl_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(jl_raw) + 1023) & ~uintptr_t(1023));
  __shared__ JlRows rows;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + JL_BAR);  // the stage's weights have landed
  uint64_t* empty = full + JL_STAGES;                         // the stage's MMAs have read it
  uint64_t* done = empty + JL_STAGES;                         // the tile's MMAs are complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + JL_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + JL_MISC + 4);
  if (tid == 0) {
    for (int i = 0; i < 2 * JL_STAGES + 1; ++i) mbar_init(&full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_w);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, JL_N);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int total = jl_rows(p, rows, -1);
  if (blockIdx.x == 0 && tid == 0) *p.row_count = (uint32_t)total;
  const int mtiles = (total + JL_M - 1) / JL_M;
  // Columns per tile: as few tiles as 256 columns allow, more while SMs are idle.
  int ntiles = max((p.columns + JL_N - 1) / JL_N, min((p.columns + 63) / 64, (int)gridDim.x / max(mtiles, 1)));
  const int bn = ((p.columns + ntiles - 1) / ntiles + 15) / 16 * 16;
  ntiles = (p.columns + bn - 1) / bn;
  const int boxes = (bn + 63) / 64;
  const uint32_t idesc = umma_idesc_f16(JL_M, 0, 0, /*weight, MN-major*/ 1) | ((uint32_t)(bn >> 3) << 17);
  const int kblocks = (p.inner + JL_K - 1) / JL_K;
  // This thread's part of a stage: 16-byte chunk tid % 8 of rows tid / 8 + 32 i.
  const int chunk = tid & 7, rbase = tid >> 3;
  const __half* enc = static_cast<const __half*>(p.encoder);

  uint32_t loads = 0, tiles_done = 0;  // stages used, tiles finished (the same in all threads)
  bool ok = true;
  for (int tile = blockIdx.x; tile < mtiles * ntiles && ok; tile += gridDim.x) {
    const int r0 = tile / ntiles * JL_M, n0 = tile % ntiles * bn;
    jl_rows(p, rows, r0);
    if (n0 == 0 && tid < JL_M && rows.place[tid] >= 0) p.row_map[r0 + tid] = (uint32_t)rows.place[tid];
    uint4 ev[4];
    float4 pv[4][2];
    auto fetch = [&](int kb) {
      const int k = kb * JL_K + chunk * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int place = rows.place[rbase + 32 * i];
        if (place >= 0 && k < p.inner) {
          ev[i] = *reinterpret_cast<const uint4*>(enc + (size_t)rows.frame[rbase + 32 * i] * p.inner + k);
          const float4* src = reinterpret_cast<const float4*>(p.predictor + (size_t)place * p.inner + k);
          pv[i][0] = src[0];
          pv[i][1] = src[1];
        } else {
          ev[i] = make_uint4(0u, 0u, 0u, 0u);
          pv[i][0] = pv[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
    };
    fetch(0);
    for (int kb = 0; kb < kblocks; ++kb, ++loads) {
      const uint32_t st = loads % JL_STAGES, use = loads / JL_STAGES;
      if (use > 0) ok = mbar_wait(&empty[st], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
      if (!__syncthreads_and(ok)) {
        ok = false;
        break;
      }
      if (tid == 0) {
        mbar_arrive_expect_tx(&full[st], (uint32_t)boxes * JL_K * 128);
        for (int b = 0; b < boxes; ++b)
          tma_load_2d(sm + JL_B + st * JL_BSTAGE + b * JL_K * 128, &p.tmap_w, &full[st], n0 + 64 * b, kb * JL_K);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = rbase + 32 * i;
        uint4 o;
        o.x = jl_hidden2(ev[i].x, pv[i][0].x, pv[i][0].y);
        o.y = jl_hidden2(ev[i].y, pv[i][0].z, pv[i][0].w);
        o.z = jl_hidden2(ev[i].z, pv[i][1].x, pv[i][1].y);
        o.w = jl_hidden2(ev[i].w, pv[i][1].z, pv[i][1].w);
        *reinterpret_cast<uint4*>(sm + JL_A + st * JL_M * 128 + (r >> 3) * 1024 + (r & 7) * 128 +
                                  ((chunk ^ (r & 7)) << 4)) = o;
      }
      if (kb + 1 < kblocks) fetch(kb + 1);
      fence_proxy_async_smem();
      __syncthreads();
      if (tid == 0) {
        ok = mbar_wait(&full[st], use & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_TMA);
        if (ok) {
          tc_fence_after();
          const uint32_t a = smem_addr(sm + JL_A + st * JL_M * 128), b = smem_addr(sm + JL_B + st * JL_BSTAGE);
#pragma unroll
          for (int ks = 0; ks < JL_K / 16; ++ks)
            tc_mma_f16(tmem, umma_smem_desc(a + ks * 32, 16, 1024, 2), umma_smem_desc(b + ks * 2048, JL_K * 128, 1024, 2),
                       idesc, kb > 0 || ks > 0 ? 1u : 0u);
          tc_commit(&empty[st]);
          if (kb + 1 == kblocks) tc_commit(done);
        }
      }
    }
    if (ok) ok = mbar_wait(done, tiles_done & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_EPILOGUE);
    ok = __syncthreads_and(ok) != 0;
    if (!ok) break;
    ++tiles_done;
    tc_fence_after();
    // Warps w and w + 4 read TMEM lanes 32 (w % 4) .. + 31, every other 32 columns each.
    const int r = (warp & 3) * 32 + lane;
    const bool live = rows.place[r] >= 0;
    __half* out = static_cast<__half*>(p.logits) + (size_t)(r0 + r) * p.columns;
    for (int c = (warp >> 2) * 32; c < bn; c += 64) {
      uint32_t v[32];
      tc_ld_32x32b_x32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, v);
      tc_wait_ld();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + c + 8 * q;
        if (live && c + 8 * q < bn && n < p.columns) {  // columns are a multiple of 8
          float b[8] = {};
          if (p.bias) {
            *reinterpret_cast<float4*>(b) = __ldg(reinterpret_cast<const float4*>(p.bias + n));
            *reinterpret_cast<float4*>(b + 4) = __ldg(reinterpret_cast<const float4*>(p.bias + n + 4));
          }
          __half2 h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            h[j] = __floats2half2_rn(__uint_as_float(v[8 * q + 2 * j]) + b[2 * j],
                                     __uint_as_float(v[8 * q + 2 * j + 1]) + b[2 * j + 1]);
          *reinterpret_cast<uint4*>(out + n) = *reinterpret_cast<const uint4*>(h);
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
      const uint32_t uses = loads > s ? (loads - s + JL_STAGES - 1) / JL_STAGES : 0;
      if (uses > 0) mbar_wait_drain(&full[s], (uses - 1) & 1, p.status);
      if (uses > 1) mbar_wait_drain(&empty[s], (uses - 2) & 1, p.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, JL_N);
  }
}

// FP32: 128 rows x 64 columns per CTA, 16 inputs a step; a thread owns 8 rows
// and 4 columns, its FMA chains in increasing input order.
constexpr int JF_N = 64;
constexpr int JF_K = 16;

__global__ void __launch_bounds__(JL_THREADS) joint_logits_fp32_kernel(const __grid_constant__ JlParams p) {
  pdl_entry();
  __shared__ JlRows rows;
  __shared__ __align__(16) float sa[2][JF_K][JL_M + 4], sb[2][JF_K][JF_N];
  const int tid = threadIdx.x;
  const int total = jl_rows(p, rows, -1);
  if (blockIdx.x == 0 && tid == 0) *p.row_count = (uint32_t)total;
  const int mtiles = (total + JL_M - 1) / JL_M, ntiles = (p.columns + JF_N - 1) / JF_N;
  const float* enc = static_cast<const float*>(p.encoder);
  const float* weight = static_cast<const float*>(p.weight);
  const int tm = tid >> 4, tn = tid & 15;  // rows 8 tm .. + 7, columns 4 tn .. + 3
  const int steps = p.inner / JF_K;        // inner is a multiple of 32
  for (int tile = blockIdx.x; tile < mtiles * ntiles; tile += gridDim.x) {
    const int r0 = tile / ntiles * JL_M, n0 = tile % ntiles * JF_N;
    jl_rows(p, rows, r0);
    if (n0 == 0 && tid < JL_M && rows.place[tid] >= 0) p.row_map[r0 + tid] = (uint32_t)rows.place[tid];
    // Gather: row tid / 2, inputs 8 (tid % 2) .. + 7 of a step; weights: input tid / 16, columns 4 (tid % 16) .. + 3.
    const int gr = tid >> 1, gk = (tid & 1) * 8;
    const int place = rows.place[gr];
    const float* es = enc + (size_t)(place >= 0 ? rows.frame[gr] : 0) * p.inner + gk;
    const float* ps = p.predictor + (size_t)(place >= 0 ? place : 0) * p.inner + gk;
    const bool wlive = n0 + 4 * tn < p.columns;
    const float* ws = weight + (size_t)(tid >> 4) * p.columns + n0 + 4 * tn;
    float4 e0, e1, q0, q1, w;
    auto fetch = [&](int s) {
      if (place >= 0) {
        e0 = *reinterpret_cast<const float4*>(es + s * JF_K);
        e1 = *reinterpret_cast<const float4*>(es + s * JF_K + 4);
        q0 = *reinterpret_cast<const float4*>(ps + s * JF_K);
        q1 = *reinterpret_cast<const float4*>(ps + s * JF_K + 4);
      } else {
        e0 = e1 = q0 = q1 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      w = wlive ? *reinterpret_cast<const float4*>(ws + (size_t)s * JF_K * p.columns) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    auto relu = [](float v) { return v < 0.0f ? 0.0f : v; };
    auto store = [&](int b) {
      const float h[8] = {e0.x + q0.x, e0.y + q0.y, e0.z + q0.z, e0.w + q0.w,
                          e1.x + q1.x, e1.y + q1.y, e1.z + q1.z, e1.w + q1.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) sa[b][gk + j][gr] = relu(h[j]);
      *reinterpret_cast<float4*>(&sb[b][tid >> 4][4 * tn]) = w;
    };
    float2 acc[4][4] = {};  // [row pair][column]
    fetch(0);
    store(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
      if (s + 1 < steps) fetch(s + 1);
#pragma unroll
      for (int k = 0; k < JF_K; ++k) {
        const float4 a0 = *reinterpret_cast<const float4*>(&sa[s & 1][k][8 * tm]);
        const float4 a1 = *reinterpret_cast<const float4*>(&sa[s & 1][k][8 * tm + 4]);
        const float4 b = *reinterpret_cast<const float4*>(&sb[s & 1][k][4 * tn]);
        const float2 a[4] = {make_float2(a0.x, a0.y), make_float2(a0.z, a0.w), make_float2(a1.x, a1.y),
                             make_float2(a1.z, a1.w)};
        const float bc[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = ffma2(a[i], make_float2(bc[j], bc[j]), acc[i][j]);
      }
      if (s + 1 < steps) store((s + 1) & 1);
      __syncthreads();
    }
    if (wlive) {
      float4 b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p.bias) b = __ldg(reinterpret_cast<const float4*>(p.bias + n0 + 4 * tn));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 8 * tm + i;
        if (rows.place[r] < 0) continue;
        const float2* c = acc[i / 2];
        const float4 o = i & 1 ? make_float4(c[0].y + b.x, c[1].y + b.y, c[2].y + b.z, c[3].y + b.w)
                               : make_float4(c[0].x + b.x, c[1].x + b.y, c[2].x + b.z, c[3].x + b.w);
        *reinterpret_cast<float4*>(static_cast<float*>(p.logits) + (size_t)(r0 + r) * p.columns + n0 + 4 * tn) = o;
      }
    }
  }
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
  const int64_t most = ((int64_t)d.batch * d.max_tokens + JL_M - 1) / JL_M;  // row tiles
  if (d.precision == PK_FP32) {
    const int64_t tiles = most * ((p.columns + JF_N - 1) / JF_N);
    return cuda_error(launch_kernel(joint_logits_fp32_kernel, dim3((unsigned)std::min<int64_t>(tiles, 2 * dev.sm_count)),
                                    dim3(JL_THREADS), 0, stream, p),
                      "joint_logits launch");
  }
  auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(dev.encode_tiled);
  const cuuint64_t dims[2] = {(cuuint64_t)p.columns, (cuuint64_t)p.inner};
  const cuuint64_t strides[1] = {(cuuint64_t)p.columns * 2};
  const cuuint32_t box[2] = {64, JL_K}, unit[2] = {1, 1};
  if (!encode ||
      encode(&p.tmap_w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(d.weight), dims, strides, box, unit,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return set_error(PK_E_CUDA, "cuTensorMapEncodeTiled failed (joint weight)");
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(joint_logits_umma_kernel), JL_SMEM);
  if (st != PK_OK) return st;
  const int64_t tiles = most * ((p.columns + 63) / 64);
  return cuda_error(launch_kernel(joint_logits_umma_kernel, dim3((unsigned)std::min<int64_t>(tiles, dev.sm_count)),
                                  dim3(JL_THREADS), JL_SMEM, stream, p),
                    "joint_logits launch");
}

}  // namespace pk
