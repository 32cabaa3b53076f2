// int4_gemv.cu -- a few rows times a matrix held in 4 bits: the decode form of
// the palette GEMM, for weights with a scale per group of inputs.
//
//   c[r, n] = epilogue(sum_g scale[g, n] * sum_{k in g} (code[k, n] - 8) a[r, k])
//
// Bound by reading the codes once (half a byte a weight), so what matters is
// that the codes stream without a pause and that a weight costs few
// instructions.  The product runs on mma.sync m16n8k16 with the weights as the
// 16-row operand and the rows of A as the 8 columns: tcgen05 would have to
// take the weights through shared memory first, and its 128-row tiles would
// stay empty for the sake of a rate that this operator cannot use.
//
// Codes lie in tiles of 16 outputs x 128 inputs (1 KB) in the order in which a
// warp's lanes hold the matrix operand, so a lane reads two 16-byte words per
// tile and a warp 512 contiguous bytes at a time, four tiles ahead.  Word i of
// a lane holds inputs 32 i + 8 t .. + 7 (t = lane % 4) of outputs lane / 4 (+ 8
// in the second 16 bytes).  A code becomes f16 by placing its 4 bits in the
// mantissa of 1024 (or, 4 bits further up, as 16 times the code) and
// subtracting: 9 instructions for 8 weights, exact.  That makes pairs of inputs
// (0,4) (1,5) (2,6) (3,7); A's rows lie in shared memory in that order.
//
// The scale multiplies a group's f32 sum, not the weight: no weight is
// rounded.  FP32 rows are two f16 columns each, the leading 11 bits and the
// next 11, after a power-of-two scale per row and 128 inputs that brings the
// largest to [2^14, 2^15): 22 bits of every input, where the sum's own rounding
// is 24.  The warps of a CTA split outputs and inputs; the inputs' parts join
// in shared memory in a fixed order (no atomics).
#include <algorithm>

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {
namespace {

constexpr int I4_WARPS = 8;       // warps per CTA, at most
constexpr int I4_KT = 128;        // inputs per tile
constexpr int I4_DEPTH = 4;       // tiles in flight per warp
constexpr int I4_COLS = 64;       // columns of one pass, at most
constexpr int I4_STAGE_BYTES = 72 * 1024;  // shared memory for A's rows, about

struct I4Params {
  const void* a;
  const uint4* codes;
  const void* scales;
  const float* bias;
  const void* residual;
  void* c;
  int rows, inner, columns, ktiles, group, groups;
  int wm, wk;        // warps over outputs, over inputs
  int chunk;         // tiles of A staged at a time (a multiple of wk * I4_DEPTH, or all)
  int rows_per_pass;
  int act;
  float residual_scale;
};

__device__ __forceinline__ uint32_t i4_lop(uint32_t a, uint32_t b, uint32_t c) {  // (a & b) | c
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t i4_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 i4_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// Eight codes -> four pairs (0,4) (1,5) (2,6) (3,7) of code - 8.
__device__ __forceinline__ void i4_expand(uint32_t w, uint32_t (&p)[4]) {
  const __half2 one = __float2half2_rn(1032.0f), sixteenth = __float2half2_rn(0.0625f), off = __float2half2_rn(-72.0f);
  const uint32_t w8 = w >> 8;
  p[0] = i4_bits(__hsub2(i4_h2(i4_lop(w, 0x000f000fu, 0x64006400u)), one));
  p[1] = i4_bits(__hfma2(i4_h2(i4_lop(w, 0x00f000f0u, 0x64006400u)), sixteenth, off));
  p[2] = i4_bits(__hsub2(i4_h2(i4_lop(w8, 0x000f000fu, 0x64006400u)), one));
  p[3] = i4_bits(__hfma2(i4_h2(i4_lop(w8, 0x00f000f0u, 0x64006400u)), sixteenth, off));
}

__device__ __forceinline__ void i4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 i4_load(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

// Bytes of one column of staged inputs: the columns of a quarter warp's loads
// fall on different banks.
__host__ __device__ inline int i4_col_bytes(int chunk) { return chunk * I4_KT * 2 + 64; }

// Stages tiles [kt0, kt0 + tiles) of `rows` rows of A: 16 lanes per row and
// tile, eight inputs each, in the order 0 4 1 5 2 6 3 7.
template <typename T>
__device__ __forceinline__ void i4_stage(const I4Params& p, unsigned char* xs, float* xscale, int row0, int rows, int kt0,
                                         int tiles) {
  const int lane16 = threadIdx.x & 15;
  const int jobs = rows * tiles;
  const int stride = i4_col_bytes(p.chunk);
  for (int j0 = (threadIdx.x >> 5) * 2; j0 < jobs; j0 += (blockDim.x >> 5) * 2) {
    const int j = j0 + ((threadIdx.x >> 4) & 1);  // the two halves of a warp
    const int r = min(j, jobs - 1) / tiles, kt = min(j, jobs - 1) % tiles;
    const int k = (kt0 + kt) * I4_KT + 8 * lane16;
    const T* src = static_cast<const T*>(p.a) + (size_t)(row0 + r) * p.inner + k;
    const bool in = k < p.inner;  // inner is a multiple of 32: eight at once
    if constexpr (sizeof(T) == 2) {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (in) v = *reinterpret_cast<const uint4*>(src);
      const uint4 o = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                 __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
      if (j < jobs) *reinterpret_cast<uint4*>(xs + (size_t)r * stride + kt * (I4_KT * 2) + lane16 * 16) = o;
    } else {
      float v[8] = {};
      if (in) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(src + 4);
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      // 2^s with the largest magnitude in [2^14, 2^15); s <= 126 keeps 2^s and 2^-s normal.
      const int s = min(141 - (int)(top >> 23), 126);
      const float up = __uint_as_float((uint32_t)(s + 127) << 23), down = __uint_as_float((uint32_t)(127 - s) << 23);
      __half hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = v[i] * up;
        hi[i] = __float2half_rn(y);
        const float h = __half2float(hi[i]);
        // An infinite or NaN input stands in the first column alone.
        lo[i] = __float2half_rn(fabsf(h) <= 65504.0f ? y - h : 0.0f);
      }
      if (j < jobs) {
        const int at[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        uint4 a, b;
        __half* ha = reinterpret_cast<__half*>(&a);
        __half* hb = reinterpret_cast<__half*>(&b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ha[i] = hi[at[i]];
          hb[i] = lo[at[i]];
        }
        unsigned char* dst = xs + (size_t)(2 * r) * stride + kt * (I4_KT * 2) + lane16 * 16;
        *reinterpret_cast<uint4*>(dst) = a;
        *reinterpret_cast<uint4*>(dst + stride) = b;
        if (lane16 == 0) xscale[r * p.chunk + kt] = down;
      }
    }
  }
}

// NT tiles of 8 columns, MT tiles of 16 outputs per warp, GB blocks of 32
// inputs per scale within a tile (1, 2, or 4: groups of whole tiles).
template <typename T, int NT, int MT, int GB>
__global__ void __launch_bounds__(I4_WARPS * 32) int4_gemv_kernel(const I4Params p) {
  extern __shared__ __align__(128) unsigned char i4_smem[];
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 2;  // columns per row
  constexpr int SPT = 4 / GB;                    // scales per tile and output
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wm = warp % p.wm, wk = warp / p.wm;
  const int row0 = blockIdx.y * p.rows_per_pass;
  const int rows = min(p.rows - row0, p.rows_per_pass);
  const int cols = rows * PARTS;
  const int mtile0 = (blockIdx.x * p.wm + wm) * MT;  // this warp's first tile of 16 outputs
  const int mtiles = (p.columns + 15) / 16;
  unsigned char* xs = i4_smem;
  const int stride = i4_col_bytes(p.chunk);
  float* xscale = reinterpret_cast<float*>(i4_smem + (size_t)cols * stride);

  struct Slot {
    uint4 code[MT][2];
    T scale[MT][2][SPT];
  };
  Slot ring[I4_DEPTH];
  auto load = [&](Slot& s, int kt) {
    if (kt >= p.ktiles) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int mt = min(mtile0 + m, mtiles - 1);
      const uint4* src = p.codes + ((size_t)mt * p.ktiles + kt) * 64 + lane;
      s.code[m][0] = i4_load(src);
      s.code[m][1] = i4_load(src + 32);
#pragma unroll
      for (int b = 0; b < SPT; ++b) {
        const int gi = min((kt * I4_KT + b * GB * 32) / p.group, p.groups - 1);
        const T* sc = static_cast<const T*>(p.scales) + (size_t)gi * p.columns;
        s.scale[m][0][b] = __ldg(sc + min(mt * 16 + g, p.columns - 1));
        s.scale[m][1][b] = __ldg(sc + min(mt * 16 + g + 8, p.columns - 1));
      }
    }
  };
  // The weights too may be the previous kernel's work (a pack, a load): nothing
  // is read before it is done.
  pdl_entry();
#pragma unroll
  for (int d = 0; d < I4_DEPTH; ++d) load(ring[d], wk + d * p.wk);

  float total[MT][NT][4] = {};
  const unsigned char* xcol[NT];
  int xrow[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    xcol[n] = xs + (size_t)min(n * 8 + g, cols - 1) * stride + t * 16;
    xrow[n][0] = min((n * 8 + 2 * t) / PARTS, rows - 1) * p.chunk;
    xrow[n][1] = min((n * 8 + 2 * t + 1) / PARTS, rows - 1) * p.chunk;
  }
  for (int kt0 = 0; kt0 < p.ktiles; kt0 += p.chunk) {
    const int tiles = min(p.chunk, p.ktiles - kt0);
    if (kt0) __syncthreads();
    i4_stage<T>(p, xs, xscale, row0, rows, kt0, tiles);
    __syncthreads();
    for (int k1 = wk; k1 < tiles; k1 += I4_DEPTH * p.wk) {
#pragma unroll
      for (int d = 0; d < I4_DEPTH; ++d) {
        const int kl = k1 + d * p.wk;  // tile of the chunk
        if (kl < tiles) {
          Slot& s = ring[d];
#pragma unroll
          for (int b = 0; b < SPT; ++b) {
            float acc[MT][NT][4] = {};
#pragma unroll
            for (int i = b * GB; i < (b + 1) * GB; ++i) {
              uint4 x[NT];
#pragma unroll
              for (int n = 0; n < NT; ++n)
                x[n] = *reinterpret_cast<const uint4*>(xcol[n] + kl * (I4_KT * 2) + i * 64);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                uint32_t w0[4], w1[4];
                i4_expand((&s.code[m][0].x)[i], w0);
                i4_expand((&s.code[m][1].x)[i], w1);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  i4_mma(acc[m][n], w0[0], w1[0], w0[1], w1[1], x[n].x, x[n].y);
                  i4_mma(acc[m][n], w0[2], w1[2], w0[3], w1[3], x[n].z, x[n].w);
                }
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float x0 = 1.0f, x1 = 1.0f;
              if constexpr (PARTS == 2) {
                x0 = xscale[xrow[n][0] + kl];
                x1 = xscale[xrow[n][1] + kl];
              }
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const float s0 = (float)s.scale[m][0][b], s1 = (float)s.scale[m][1][b];
                total[m][n][0] = fmaf(s0 * x0, acc[m][n][0], total[m][n][0]);
                total[m][n][1] = fmaf(s0 * x1, acc[m][n][1], total[m][n][1]);
                total[m][n][2] = fmaf(s1 * x0, acc[m][n][2], total[m][n][2]);
                total[m][n][3] = fmaf(s1 * x1, acc[m][n][3], total[m][n][3]);
              }
            }
          }
          load(s, kt0 + kl + I4_DEPTH * p.wk);
        }
      }
    }
  }
  // Parts of the inputs' split, [wk][column][output]: the staged rows are done with.
  __syncthreads();
  const int M = p.wm * MT * 16;
  constexpr int PC = NT * 8;
  float* part = reinterpret_cast<float*>(i4_smem);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[((size_t)wk * PC + n * 8 + 2 * t + (e & 1)) * (M + 4) + (wm * MT + m) * 16 + g + 8 * (e >> 1)] =
            total[m][n][e];
  __syncthreads();
  for (int i = tid; i < rows * M; i += blockDim.x) {
    const int r = i / M, m = i % M;
    const int n = blockIdx.x * M + m;
    if (n >= p.columns) continue;
    float v = 0.0f;
    for (int w = 0; w < p.wk; ++w)
#pragma unroll
      for (int q = 0; q < PARTS; ++q) v += part[((size_t)w * PC + r * PARTS + q) * (M + 4) + m];
    if (p.bias) v += __ldg(p.bias + n);
    if (p.act == PK_ACT_SILU) v = v / (1.0f + expf(-v));
    else if (p.act == PK_ACT_RELU) v = v < 0.0f ? 0.0f : v;
    const size_t at = (size_t)(row0 + r) * p.columns + n;
    if (p.residual) v = fmaf(p.residual_scale, v, (float)static_cast<const T*>(p.residual)[at]);
    static_cast<T*>(p.c)[at] = (T)v;
  }
}

template <typename T, int NT, int MT, int GB>
int launch_one(const I4Params& p, dim3 grid, int smem, cudaStream_t stream) {
  if (smem > 48 * 1024) {
    const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(int4_gemv_kernel<T, NT, MT, GB>), 200 * 1024);
    if (st != PK_OK) return st;
  }
  return cuda_error(launch_kernel(int4_gemv_kernel<T, NT, MT, GB>, grid, dim3((unsigned)(p.wm * p.wk * 32)),
                                  (size_t)smem, stream, p),
                    "int4_gemv launch");
}

template <typename T, int NT, int MT>
int launch_group(const I4Params& p, dim3 grid, int smem, cudaStream_t stream) {
  if (p.group == 32) return launch_one<T, NT, MT, 1>(p, grid, smem, stream);
  if (p.group == 64) return launch_one<T, NT, MT, 2>(p, grid, smem, stream);
  return launch_one<T, NT, MT, 4>(p, grid, smem, stream);
}

template <typename T>
int launch_typed(const DeviceCtx& dev, I4Params p, cudaStream_t stream) {
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 2;
  p.rows_per_pass = std::min(p.rows, I4_COLS / PARTS);
  const int passes = (p.rows + p.rows_per_pass - 1) / p.rows_per_pass;
  const int cols = p.rows_per_pass * PARTS;
  const int nt = cols <= 8 ? 1 : cols <= 16 ? 2 : cols <= 32 ? 4 : 8;
  const int mt = nt == 4 ? 2 : 1;
  const int mtiles = (p.columns + 15) / 16;
  // Warps over the inputs: as many as there are tiles for, and as the staged
  // rows leave room for with I4_DEPTH tiles each.
  int wk = 1;
  while (wk < I4_WARPS && 2 * wk <= p.ktiles && 2 * wk * I4_DEPTH * I4_KT * 2 * cols <= I4_STAGE_BYTES) wk *= 2;
  int wm = I4_WARPS / wk;
  // Outputs rather than inputs where there are enough of them for every SM.
  while (wk > 1 && (mtiles + 2 * wm * mt - 1) / (2 * wm * mt) >= 2 * dev.sm_count) wk /= 2, wm *= 2;
  while (wm > 1 && (mtiles + wm * mt - 1) / (wm * mt) < dev.sm_count) wm /= 2;
  p.wm = wm;
  p.wk = wk;
  const int step = wk * I4_DEPTH;
  p.chunk = std::max(step, I4_STAGE_BYTES / (cols * I4_KT * 2) / step * step);
  if (p.chunk >= p.ktiles) p.chunk = p.ktiles;
  const int stage = cols * i4_col_bytes(p.chunk) + (PARTS == 2 ? p.rows_per_pass * p.chunk * 4 : 0);
  const int parts = wk * nt * 8 * (wm * mt * 16 + 4) * 4;
  const int smem = std::max(stage, parts);
  const dim3 grid((unsigned)((mtiles + wm * mt - 1) / (wm * mt)), (unsigned)passes);
  if (nt == 1) return launch_group<T, 1, 1>(p, grid, smem, stream);
  if (nt == 2) return launch_group<T, 2, 1>(p, grid, smem, stream);
  if (nt == 4) return launch_group<T, 4, 2>(p, grid, smem, stream);
  return launch_group<T, 8, 1>(p, grid, smem, stream);
}

}  // namespace

int launch_int4_gemv(const DeviceCtx& dev, const pk_int4_gemv_desc& d, cudaStream_t stream) {
  I4Params p{};
  p.a = d.a;
  p.codes = reinterpret_cast<const uint4*>(d.codes);
  p.scales = d.scales;
  p.bias = d.bias;
  p.residual = d.residual;
  p.c = d.c;
  p.rows = (int)d.rows;
  p.inner = (int)d.inner;
  p.columns = (int)d.columns;
  p.ktiles = (int)((d.inner + I4_KT - 1) / I4_KT);
  p.group = (int)d.group;
  p.groups = (int)(d.inner / d.group);
  p.act = d.activation;
  p.residual_scale = d.residual_scale;
  return d.precision == PK_FP16 ? launch_typed<__half>(dev, p, stream) : launch_typed<float>(dev, p, stream);
}

}  // namespace pk
