// residual_norm.cu -- what stands between two blocks of a network, in one pass:
//
//   u = post(block)                     the norm after the block
//   y = input + scale * gate * u        its gate and residual scale; the residual stream
//   h = pre(y)                          the next block's norm
//
// post and pre are LayerNorm ((v - mean) rstd gamma + beta), RMS norm
// (v rrms gamma) or absent; the gate is absent, one row of channels, or one
// row for every `gate_rows` rows.  y and h are each rounded once: h is the
// norm of y before its rounding.  Means and variances are f32, the variance
// from the centred values (a second sum over registers costs no memory, and
// E[v^2] - mean^2 loses what a large mean hides).
//
// Bound by memory: two reads and two writes of every element, nothing in
// between reaches memory.  16384x4096 f32 175 us, 6.1 TB/s or 94% of a copy's
// rate; 16384x2048 f16 46 us, 5.9 TB/s; 6016x1024 f16 12.0 us; 1x640 f16 2.7 us
// in a graph of such calls, 3.2 launched one by one: a launch and one round trip.
//
// Rows of up to 512 vectors of 16 bytes: a thread owns a vector's channels, keeps
// their parameters in registers and takes four rows of its CTA at a time.  Longer
// or unaligned rows: a row lives in the registers of 32 to 1024 threads; all its
// loads are issued before the first is used, and gamma, beta and gate come from
// L1 after the first rows.
#include <algorithm>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

struct RnParams {
  const void* x;
  const void* f;
  const float* post_gamma;
  const float* post_beta;
  const float* pre_gamma;
  const float* pre_beta;
  const float* gate;
  void* y;
  void* h;
  int64_t rows, gate_rows;
  int channels, post, pre;
  float scale, eps;
};

// VEC elements of T as one load or store.
template <int BYTES>
struct RnWord;
template <>
struct RnWord<16> { using type = uint4; };
template <>
struct RnWord<8> { using type = uint2; };
template <>
struct RnWord<4> { using type = uint32_t; };
template <>
struct RnWord<2> { using type = uint16_t; };

template <typename T, int VEC>
__device__ __forceinline__ void rn_unpack(const typename RnWord<VEC * sizeof(T)>::type& raw, float (&v)[VEC]) {
  const T* e = reinterpret_cast<const T*>(&raw);
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    const __half2* e2 = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const float2 f = __half22float2(e2[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)e[j];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ typename RnWord<VEC * sizeof(T)>::type rn_pack(const float (&v)[VEC]) {
  typename RnWord<VEC * sizeof(T)>::type raw;
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    __half2* e2 = reinterpret_cast<__half2*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) e2[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
  } else {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int j = 0; j < VEC; ++j) e[j] = (T)v[j];
  }
  return raw;
}
template <int VEC>
__device__ __forceinline__ void rn_params(const float* src, float (&v)[VEC]) {
  if constexpr (VEC >= 4) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) *reinterpret_cast<float4*>(v + j) = __ldg(reinterpret_cast<const float4*>(src + j));
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = __ldg(src + j);
  }
}

// 1 / sqrt(v): the hardware's estimate (2 ulp) and one Newton step, where neither
// v nor the result is infinite (the step would meet inf * 0).
__device__ __forceinline__ float rn_rsqrt(float v) {
  const float r = rsqrtf(v);
  return r > 0.0f && r < INFINITY ? fmaf(r * 0.5f, fmaf(-v * r, r, 1.0f), r) : r;
}

// Sum over the G threads of a row.  Rows of more than a warp meet in shared
// memory; `turn` alternates the two halves of `red`, so one barrier a sum is enough.
template <int G>
__device__ __forceinline__ float rn_sum(float v, float* red, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (G > 32) {
    float* mine = red + 32 * turn;
    turn ^= 1;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) mine[warp] = v;
    __syncthreads();
    const int w0 = (int)threadIdx.x / G * (G / 32);
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) v += mine[w0 + w];
  }
  return v;
}

// G threads per row, NV vectors of VEC elements per thread, blockDim / G rows per CTA.
template <typename T, int VEC, int G, int NV>
__global__ void __launch_bounds__(G > 256 ? G : 256) residual_norm_kernel(const RnParams p) {
  pdl_entry();
  using Word = typename RnWord<VEC * sizeof(T)>::type;
  __shared__ float red[64];
  int turn = 0;
  const int t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
  const bool live = row < p.rows;
  const int C = p.channels;
  const int words = C / VEC;
  const Word* fx = reinterpret_cast<const Word*>(static_cast<const T*>(p.f) + (live ? row : 0) * C);
  const Word* xx = reinterpret_cast<const Word*>(static_cast<const T*>(p.x) + (live ? row : 0) * C);
  // With 1024 threads and more than 16 elements each, the residual's words do
  // not fit beside the block's values: they are read when they are used.
  constexpr bool EARLY = G < 1024 || VEC * NV <= 16;
  Word fr[NV], xr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (live && t + i * G < words) fr[i] = fx[t + i * G];
  if constexpr (EARLY) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (live && t + i * G < words) xr[i] = xx[t + i * G];
  }
  float v[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (live && t + i * G < words) {
      rn_unpack<T, VEC>(fr[i], v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
    }
  }
  const float inv = 1.0f / (float)C;
  // Mean and 1 / deviation (RMS: 0 and 1 / root mean square) of the row in v.
  auto stats = [&](int kind, float& mean, float& rstd) {
    float s = 0.0f;
    mean = 0.0f;
    if (kind == PK_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[i][j];
      mean = rn_sum<G>(s, red, turn) * inv;
    }
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t + i * G < words) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = v[i][j] - mean;
          s = fmaf(d, d, s);
        }
      }
    }
    rstd = rn_rsqrt(rn_sum<G>(s, red, turn) * inv + p.eps);
  };
  float mean = 0.0f, rstd = 1.0f;
  if (p.post != PK_NORM_NONE) stats(p.post, mean, rstd);
  const float* gate = p.gate ? p.gate + (p.gate_rows > 0 ? (live ? row : 0) / p.gate_rows : 0) * C : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * G) * VEC;
    if (live && t + i * G < words) {
      float g[VEC], x[VEC];
      if (p.post != PK_NORM_NONE) {
        rn_params<VEC>(p.post_gamma + c, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = (v[i][j] - mean) * rstd * g[j];
        if (p.post == PK_NORM_LAYER) {
          rn_params<VEC>(p.post_beta + c, g);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += g[j];
        }
      }
      if (gate) {
        rn_params<VEC>(gate + c, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] *= g[j];
      }
      if constexpr (!EARLY) xr[i] = xx[t + i * G];
      rn_unpack<T, VEC>(xr[i], x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = fmaf(p.scale, v[i][j], x[j]);
    }
  }
  // The row is in registers, whole: where y or h takes the place of x or f,
  // every thread has read its elements, and it writes only those.
  Word* yo = reinterpret_cast<Word*>(static_cast<T*>(p.y) + (live ? row : 0) * C);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (live && t + i * G < words) yo[t + i * G] = rn_pack<T, VEC>(v[i]);
  if (p.pre == PK_NORM_NONE) return;
  stats(p.pre, mean, rstd);
  Word* ho = reinterpret_cast<Word*>(static_cast<T*>(p.h) + (live ? row : 0) * C);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * G) * VEC;
    if (live && t + i * G < words) {
      float g[VEC];
      rn_params<VEC>(p.pre_gamma + c, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = (v[i][j] - mean) * rstd * g[j];
      if (p.pre == PK_NORM_LAYER) {
        rn_params<VEC>(p.pre_beta + c, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] += g[j];
      }
      ho[t + i * G] = rn_pack<T, VEC>(v[i]);
    }
  }
}

// Many rows of at most 512 vectors: a thread keeps one vector of channels for
// every row that its CTA takes, so the parameters stay in its registers (a gate
// that all rows share folded with the scale into gamma and beta), and the CTA
// takes R rows at a time: their sums meet at the same barriers, and the next R
// rows are on their way meanwhile.
constexpr int RN_R = 4;
constexpr int RN_COLS = 512;  // threads per CTA, at most

// Sums the CTA's R values per thread; all threads receive last(total) of each.  The
// warp's butterfly halves what a lane holds as long as it holds more than one
// value, so R sums cost R + 2 exchanges, not 5 R.  `turn` alternates two halves
// of `red`: one barrier a sum is enough.
template <typename Last>
__device__ __forceinline__ void rn_sums(float (&v)[RN_R], float (*red)[RN_COLS / 32][RN_R], int& turn, Last last) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool b4 = lane & 16, b3 = lane & 8;
  float k0 = b4 ? v[2] : v[0], k1 = b4 ? v[3] : v[1];
  k0 += __shfl_xor_sync(0xffffffffu, b4 ? v[0] : v[2], 16);
  k1 += __shfl_xor_sync(0xffffffffu, b4 ? v[1] : v[3], 16);
  float k = b3 ? k1 : k0;
  k += __shfl_xor_sync(0xffffffffu, b3 ? k0 : k1, 8);
  k += __shfl_xor_sync(0xffffffffu, k, 4);
  k += __shfl_xor_sync(0xffffffffu, k, 2);
  k += __shfl_xor_sync(0xffffffffu, k, 1);
  float(*mine)[RN_R] = red[turn];
  turn ^= 1;
  if ((lane & 7) == 0) mine[warp][lane >> 3] = k;
  __syncthreads();
  // Lane (w, r): the sums of row r in warps w, w + 8.
  const int w = lane >> 2, r = lane & 3;
  k = w < warps ? mine[w][r] : 0.0f;
  if (w + 8 < warps) k += mine[w + 8][r];
  k += __shfl_xor_sync(0xffffffffu, k, 4);
  k += __shfl_xor_sync(0xffffffffu, k, 8);
  k = last(k + __shfl_xor_sync(0xffffffffu, k, 16));
#pragma unroll
  for (int i = 0; i < RN_R; ++i) v[i] = __shfl_sync(0xffffffffu, k, i);
}

template <typename T, bool BY_ROWS>
__global__ void __launch_bounds__(RN_COLS, 1) residual_norm_rows_kernel(const RnParams p) {
  pdl_entry();
  constexpr int VEC = 16 / sizeof(T), P = VEC / 2;
  __shared__ float red[2][RN_COLS / 32][RN_R];
  const int C = p.channels;
  const int c = threadIdx.x * VEC;
  const bool in = c < C;  // the last warp may reach past the row
  const uint32_t gate_rows = (uint32_t)min(p.gate_rows, p.rows);  // rows are below 2^31
  const float2 one = make_float2(1.0f, 1.0f), zero = make_float2(0.0f, 0.0f);
  uint4 fr[RN_R], xr[RN_R];
  // Rows left from the batch's first, and its first element of this thread.
  const int step = (int)gridDim.x * RN_R;
  int left = (int)(p.rows - (int64_t)blockIdx.x * RN_R);
  int64_t at = (int64_t)blockIdx.x * RN_R * C + c;
  auto fetch = [&](const void* src, int64_t from, int rows, uint4 (&raw)[RN_R]) {
    const T* s = static_cast<const T*>(src) + from;
#pragma unroll
    for (int i = 0; i < RN_R; ++i)
      raw[i] = in && i < rows ? *reinterpret_cast<const uint4*>(s + (size_t)(uint32_t)(i * C)) : make_uint4(0u, 0u, 0u, 0u);
  };
  fetch(p.f, at, left, fr);
  fetch(p.x, at, left, xr);
  float2 sg[P], sb[P], hg[P], hb[P];  // post and pre gamma and beta
#pragma unroll
  for (int j = 0; j < P; ++j) sg[j] = hg[j] = one, sb[j] = hb[j] = zero;
  if (in) {
    auto take = [&](const float* src, float2 (&dst)[P]) {
#pragma unroll
      for (int j = 0; j < P; j += 2) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(src + c + 2 * j));
        dst[j] = make_float2(v.x, v.y);
        dst[j + 1] = make_float2(v.z, v.w);
      }
    };
    if (p.post != PK_NORM_NONE) take(p.post_gamma, sg);
    if (p.post == PK_NORM_LAYER) take(p.post_beta, sb);
    if (p.pre != PK_NORM_NONE) take(p.pre_gamma, hg);
    if (p.pre == PK_NORM_LAYER) take(p.pre_beta, hb);
    if constexpr (!BY_ROWS) {
      float2 g[P];
#pragma unroll
      for (int j = 0; j < P; ++j) g[j] = one;
      if (p.gate) take(p.gate, g);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        g[j] = make_float2(g[j].x * p.scale, g[j].y * p.scale);
        sg[j] = ffma2(sg[j], g[j], zero);
        sb[j] = ffma2(sb[j], g[j], zero);
      }
    }
  }
  const float inv = 1.0f / (float)C;
  int turn = 0;
  float2 v[RN_R][P];
  float rstd[RN_R];
  // Centres the rows in v (LayerNorm) and sets rstd = 1 / deviation; threads
  // past the row hold zeros.
  auto normalize = [&](int kind) {
    float s[RN_R];
    if (kind == PK_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < RN_R; ++i) {
        float2 a = v[i][0];
#pragma unroll
        for (int j = 1; j < P; ++j) a = ffma2(v[i][j], one, a);
        s[i] = a.x + a.y;
      }
      rn_sums(s, red, turn, [&](float k) { return -k * inv; });
#pragma unroll
      for (int i = 0; i < RN_R; ++i) {
        const float m = in ? s[i] : 0.0f;
#pragma unroll
        for (int j = 0; j < P; ++j) v[i][j] = ffma2(v[i][j], one, make_float2(m, m));
      }
    }
#pragma unroll
    for (int i = 0; i < RN_R; ++i) {
      float2 a = ffma2(v[i][0], v[i][0], zero);
#pragma unroll
      for (int j = 1; j < P; ++j) a = ffma2(v[i][j], v[i][j], a);
      s[i] = a.x + a.y;
    }
    rn_sums(s, red, turn, [&](float k) { return rn_rsqrt(fmaf(k, inv, p.eps)); });
#pragma unroll
    for (int i = 0; i < RN_R; ++i) rstd[i] = s[i];
  };
  for (; left > 0; left -= step, at += (int64_t)step * C) {
#pragma unroll
    for (int i = 0; i < RN_R; ++i) {
      float e[VEC];
      rn_unpack<T, VEC>(fr[i], e);
#pragma unroll
      for (int j = 0; j < P; ++j) v[i][j] = make_float2(e[2 * j], e[2 * j + 1]);
      rstd[i] = 1.0f;
    }
    const int64_t next = at + (int64_t)step * C;
    if (left > step) fetch(p.f, next, left - step, fr);
    if (p.post != PK_NORM_NONE) normalize(p.post);
#pragma unroll
    for (int i = 0; i < RN_R; ++i) {
      float e[VEC], y[VEC];
      rn_unpack<T, VEC>(xr[i], e);
      float2 w[P];  // the row's gate times the scale
#pragma unroll
      for (int j = 0; j < P; ++j) w[j] = one;
      if constexpr (BY_ROWS) {
        if (in && i < left) {
          const float* gate = p.gate + (size_t)((uint32_t)(p.rows - left + i) / gate_rows) * C + c;
#pragma unroll
          for (int j = 0; j < P; j += 2) {
            const float4 g = __ldg(reinterpret_cast<const float4*>(gate + 2 * j));
            w[j] = make_float2(g.x * p.scale, g.y * p.scale);
            w[j + 1] = make_float2(g.z * p.scale, g.w * p.scale);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 x = make_float2(e[2 * j], e[2 * j + 1]);
        float2 u = ffma2(v[i][j], make_float2(rstd[i], rstd[i]), zero);
        if constexpr (BY_ROWS) {
          u = ffma2(ffma2(u, sg[j], sb[j]), w[j], x);
        } else {
          u = ffma2(u, sg[j], ffma2(sb[j], one, x));
        }
        v[i][j] = u;
        y[2 * j] = u.x;
        y[2 * j + 1] = u.y;
      }
      if (in && i < left)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.y) + at + (size_t)(uint32_t)(i * C)) = rn_pack<T, VEC>(y);
    }
    if (left > step) fetch(p.x, next, left - step, xr);
    if (p.pre == PK_NORM_NONE) continue;
    normalize(p.pre);
#pragma unroll
    for (int i = 0; i < RN_R; ++i) {
      float h[VEC];
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 u = ffma2(ffma2(v[i][j], make_float2(rstd[i], rstd[i]), zero), hg[j], hb[j]);
        h[2 * j] = u.x;
        h[2 * j + 1] = u.y;
      }
      if (in && i < left)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.h) + at + (size_t)(uint32_t)(i * C)) = rn_pack<T, VEC>(h);
    }
  }
}

template <typename T, int VEC, int G, int NV>
int launch_one(const RnParams& p, cudaStream_t stream) {
  constexpr int threads = G > 256 ? G : 256;
  const int64_t per = threads / G;
  return cuda_error(launch_kernel(residual_norm_kernel<T, VEC, G, NV>, dim3((unsigned)((p.rows + per - 1) / per)),
                                  dim3(threads), 0, stream, p),
                    "residual_norm launch");
}

// The fewest threads that hold a row at NV vectors each.
template <typename T, int VEC>
int launch_vec(const RnParams& p, cudaStream_t stream) {
  const int words = p.channels / VEC;
  if (words <= 32) return launch_one<T, VEC, 32, 1>(p, stream);
  if (words <= 128) return launch_one<T, VEC, 32, 4>(p, stream);
  if (words <= 256) return launch_one<T, VEC, 64, 4>(p, stream);
  if (words <= 512) return launch_one<T, VEC, 128, 4>(p, stream);
  if (words <= 1024) return launch_one<T, VEC, 256, 4>(p, stream);
  if (words <= 2048) return launch_one<T, VEC, 512, 4>(p, stream);
  // Rows of at most 32768 channels: 4096 words of 8, 8192 of 4, 32768 single
  // elements (a row whose start is not aligned).
  if constexpr (VEC < 8) {
    if (words > 4096) return launch_one<T, VEC, 1024, VEC == 1 ? 32 : 8>(p, stream);
  }
  return launch_one<T, VEC, 1024, 4>(p, stream);
}

template <typename T>
int launch_rows(const DeviceCtx& dev, const RnParams& p, cudaStream_t stream) {
  const int threads = (p.channels * (int)sizeof(T) / 16 + 31) / 32 * 32;
  const int64_t ctas = std::min<int64_t>((p.rows + RN_R - 1) / RN_R, (int64_t)dev.sm_count * (RN_COLS / threads));
  auto kernel = p.gate && p.gate_rows > 0 ? residual_norm_rows_kernel<T, true> : residual_norm_rows_kernel<T, false>;
  return cuda_error(launch_kernel(kernel, dim3((unsigned)ctas), dim3((unsigned)threads), 0, stream, p),
                    "residual_norm launch");
}

template <typename T>
int launch_typed(const DeviceCtx& dev, const RnParams& p, cudaStream_t stream) {
  const uintptr_t data = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.f) |
                         reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.h) |
                         (uintptr_t)p.channels * sizeof(T);
  const uintptr_t params = reinterpret_cast<uintptr_t>(p.post_gamma) | reinterpret_cast<uintptr_t>(p.post_beta) |
                           reinterpret_cast<uintptr_t>(p.pre_gamma) | reinterpret_cast<uintptr_t>(p.pre_beta) |
                           reinterpret_cast<uintptr_t>(p.gate);
  if ((data & 15) == 0 && (params & 15) == 0) {
    const int64_t vectors = p.channels * (int64_t)sizeof(T) / 16;
    // A thread per vector of the row where a CTA has so many: its parameters are
    // loaded beside the row and not behind the sums (1x1024 f16 2.8 us against 4.5,
    // 1000x1024 4.3 against 7.3, 6016x1024 12.0 against 19.8).
    if (vectors <= RN_COLS) return launch_rows<T>(dev, p, stream);
    return launch_vec<T, 16 / sizeof(T)>(p, stream);
  }
  if (sizeof(T) == 2 && (data & 7) == 0 && (params & 15) == 0) return launch_vec<T, 8 / sizeof(T)>(p, stream);
  return launch_vec<T, 1>(p, stream);
}

}  // namespace

int launch_residual_norm(const DeviceCtx& dev, const pk_residual_norm_desc& d, cudaStream_t stream) {
  RnParams p;
  p.x = d.input;
  p.f = d.block;
  p.post_gamma = d.post_gamma;
  p.post_beta = d.post_beta;
  p.pre_gamma = d.pre_gamma;
  p.pre_beta = d.pre_beta;
  p.gate = d.gate;
  p.y = d.output;
  p.h = d.normalized;
  p.rows = d.rows;
  p.gate_rows = d.gate_rows;
  p.channels = (int)d.channels;
  p.post = d.post;
  p.pre = d.pre;
  p.scale = d.residual_scale;
  p.eps = d.epsilon;
  return d.precision == PK_FP16 ? launch_typed<__half>(dev, p, stream) : launch_typed<float>(dev, p, stream);
}

}  // namespace pk
