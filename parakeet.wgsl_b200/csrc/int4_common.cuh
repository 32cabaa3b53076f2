// int4_common.cuh -- what the two kernels of the int4 product share: the call's
// parameters, how rows of A become f16 columns, the products of infinite inputs
// and the epilogue.
#pragma once

#include "pk_common.cuh"
#include "pk_internal.h"

namespace pk {

constexpr int I4_KT = 128;        // inputs per tile of codes
constexpr int I4_CLUSTER = 8;     // CTAs that share the inputs, at most
constexpr int I4_SMEM = 220 * 1024;

struct I4Params {
  const void* a;
  const uint4* codes;
  const void* scales;
  const float* bias;
  const void* residual;
  void* c;
  int rows, inner, columns, ktiles;
  int groups;           // scales per output
  uint32_t group_inv;   // 2^32 / (tiles per group), rounded up (groups of whole tiles)
  int wm, wk;           // warps over outputs, over inputs
  int ktiles_cta;       // tiles of inputs per CTA of a cluster
  int cluster;
  int rows_per_pass;
  int part_offset;      // bytes of shared memory before the parts
  int act;
  float residual_scale;
  unsigned int* status;
};

// Clusters of `cluster` CTAs that run at once with one CTA per SM.
int int4_clusters(const DeviceCtx& dev, int cluster, int* out);
int launch_int4_umma(const DeviceCtx& dev, const I4Params& p, int precision, int group, cudaStream_t stream);

__device__ __forceinline__ uint32_t i4_lop(uint32_t a, uint32_t b, uint32_t c) {  // (a & b) | c
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t i4_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 i4_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

__device__ __forceinline__ uint4 i4_load(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 i4_lds(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float i4_lds_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Eight inputs of a row as f16 columns, in the order 0 4 1 5 2 6 3 7 in which a
// word of codes gives its pairs; 16 lanes (`mask`) hold a tile's 128.  FP32: two
// columns and the factor `down` that undoes their scale where it is applied
// twice, once to the weights' scale and once to the sum: the whole of it would
// take either out of f32's range where the product is well inside.  Returns
// whether an input was infinite or NaN; it becomes 0.
template <typename T>
__device__ __forceinline__ bool i4_columns(const uint4 (&raw)[sizeof(T) / 2], uint32_t mask, uint4 (&col)[sizeof(T) / 2],
                                           float& down) {
  bool special = false;
  if constexpr (sizeof(T) == 2) {
    uint4 v = raw[0];
    auto over = [](uint32_t w) { return (w & 0x7fff7fffu) + 0x04000400u; };  // bit 15 of a half: its exponent is all ones
    if (((over(v.x) | over(v.y) | over(v.z) | over(v.w)) & 0x80008000u) != 0) {
      special = true;
      uint32_t* w = &v.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t o = over(w[i]);
        w[i] &= (o & 0x8000u ? 0u : 0xffffu) | (o & 0x80000000u ? 0u : 0xffff0000u);
      }
    }
    col[0] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                        __byte_perm(v.y, v.w, 0x7632));
  } else {
    float v[8];
    *reinterpret_cast<uint4*>(v) = raw[0];
    *reinterpret_cast<uint4*>(v + 4) = raw[1];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    if (top >= 0x7f800000u) {
      special = true;
      top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if ((__float_as_uint(v[i]) & 0x7fffffffu) >= 0x7f800000u) v[i] = 0.0f;
        top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
    // 2^s with the largest magnitude in [2^13, 2^15), s even; s <= 126 keeps 2^s normal.
    const int s = min(141 - (int)(top >> 23), 126) & ~1;
    const float up = __uint_as_float((uint32_t)(s + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - s / 2) << 23);
    __half hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = v[i] * up;
      hi[i] = __float2half_rn(y);
      lo[i] = __float2half_rn(y - __half2float(hi[i]));
    }
    const int at[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    __half* ha = reinterpret_cast<__half*>(&col[0]);
    __half* hb = reinterpret_cast<__half*>(&col[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ha[i] = hi[at[i]];
      hb[i] = lo[at[i]];
    }
  }
  return special;
}

// The products of row r's infinite and NaN inputs of tiles [kt0, kt0 + tiles) with output n.
template <typename T>
__device__ float i4_special(const I4Params& p, int r, int n, int kt0, int tiles) {
  const T* a = static_cast<const T*>(p.a) + (size_t)r * p.inner;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(p.codes) + ((size_t)(n >> 4) * p.ktiles) * 256;
  const T* scales = static_cast<const T*>(p.scales) + (size_t)(n >> 4) * p.groups * 16 + (n & 15);
  const int group = p.inner / p.groups;
  const int end = min((kt0 + tiles) * I4_KT, p.inner);
  float v = 0.0f;
#pragma unroll 1
  for (int k = kt0 * I4_KT; k < end; ++k) {
    const float x = (float)a[k];
    if (fabsf(x) < INFINITY) continue;
    const uint32_t w = words[(size_t)(k >> 7) * 256 + (n & 15) * 16 + ((k >> 3) + (n >> 1) & 3) * 4 + (k >> 5 & 3)];
    v += x * (((float)(w >> 4 * (k & 7) & 15) - 8.0f) * (float)scales[(size_t)(k / group) * 16]);
  }
  return v;
}

// The epilogue behind the bias, of element `at` of the output.
template <typename T>
__device__ __forceinline__ void i4_finish(const I4Params& p, size_t at, float v) {
  if (p.act == PK_ACT_SILU) v = v / (1.0f + expf(-v));
  else if (p.act == PK_ACT_RELU) v = v < 0.0f ? 0.0f : v;
  if (p.residual) v = fmaf(p.residual_scale, v, (float)static_cast<const T*>(p.residual)[at]);
  static_cast<T*>(p.c)[at] = (T)v;
}

}  // namespace pk
