// int4_gemv.cu -- a few rows times a matrix held in 4 bits: the decode form of
// the palette GEMM, for weights with a scale per group of inputs.
//
//   c[r, n] = epilogue(sum_g scale[g, n] * sum_{k in g} (code[k, n] - 8) a[r, k])
//
// Bound by reading the codes once (half a byte a weight), so what matters is
// that the codes stream without a pause and that a weight costs few
// instructions.  Here, for up to 16 columns and for small matrices, the product
// runs on mma.sync m16n8k16 with the weights as the 16-row operand and the rows
// of A as the 8 columns: its operand is expanded in the registers that it is
// loaded to, a warp needs no other, and no tile is larger than the work.
// int4_umma.cu has the rest.
//
// Codes lie in tiles of 16 outputs x 128 inputs (1 KB), 64 bytes an output, so a
// lane reads two 16-byte words per tile and a warp 512 contiguous bytes at a
// time.  Word i of a lane holds inputs 32 i + 8 t .. + 7 (t = lane % 4) of
// outputs lane / 4 (+ 8 in the second 16 bytes); the four t of an output are
// turned by output / 2, so that a thread per output reads them from shared
// memory without bank conflicts too.  A code becomes f16 by placing its 4 bits in a
// mantissa: 1024 + code where they are the lowest, less 1032 in one more
// instruction; 64 + code where they are the next four, which stays as it is --
// the sums of a group begin at -72 times the sum of those inputs instead (the
// first product's addend).  7 instructions for 8 weights; the second form adds
// values 16 times the weights' size to the f32 sums, 2^-20 of a product's size.
// That makes pairs of inputs (0,4) (1,5) (2,6) (3,7); A's rows lie in shared
// memory in that order.
//
// The scale multiplies a group's f32 sum, not the weight: no weight is
// rounded.  FP32 rows are two f16 columns each, the leading 11 bits and the
// next 11, after a power-of-two scale per row and 128 inputs that brings the
// largest to [2^13, 2^15): 22 bits of every input, where the sum's own rounding
// is 24.  An infinite or NaN input is laid out as 0 and its row marked; the
// thread that joins such a row's sum adds those products itself, from A.
//
// 1x4096x65536 f16 26.7 us, 5.2 TB/s or 80% of a copy's rate; 8 rows 29.9 us (72%);
// 1x4096x16384 f16 10.1 us and 1x640x640 f16 3.0 us (3.2 launched one by one),
// where start and join show.  FP32: 1x4096x65536 27.4 us (80%), 4 rows 29.5, 8 rows
// 46; 1x4096x16384 10.4 us.  16 columns (16 rows f16 51 us): two MMAs a weight
// tile, and twice the columns to read from shared memory.  (What marks infinite inputs costs 0.1 to 0.4 us of these.)
//
// One CTA per SM walks the output tiles; A's rows are laid out in its shared
// memory once.  Its warps split outputs (wm) and inputs (wk), so that the
// outputs of an SM come out even: 1024 tiles on 148 SMs are 7 a SM, at once.
// Where the rows are more than shared memory holds, or the outputs are fewer
// than the SMs, a cluster of CTAs splits the inputs and joins through
// distributed shared memory.  Parts join in a fixed order: no workspace, no
// atomics.
#include <algorithm>
#include <map>
#include <mutex>
#include <utility>

#include "int4_common.cuh"

namespace pk {
namespace {

constexpr int I4_COLS = 32;       // columns of one pass, at most (more rows: the codes again, from L2)

// Warps per CTA (registers: 72, 128, 128 a thread), tiles of outputs a warp takes
// at a time and tiles in flight per warp, by column tiles.  With two output
// tiles a column leaves shared memory half as often: 16x4096x65536 f16 53 -> 48
// us; with 32 columns their sums leave room for 12 warps alone, 86 -> 92 us.
__host__ __device__ constexpr int i4_warps(int nt) { return nt == 1 ? 28 : 16; }
__host__ __device__ constexpr int i4_mt(int nt) { return nt == 2 ? 2 : 1; }
__host__ __device__ constexpr int i4_depth(int nt) { return nt == 4 ? 3 : 2; }

// Eight codes -> the pairs (0,4) (2,6) of code - 8 and (1,5) (3,7) of code + 64.
__device__ __forceinline__ void i4_expand(uint32_t w, uint32_t (&p)[4]) {
  const __half2 off = __float2half2_rn(1032.0f);
  const uint32_t w8 = w >> 8;
  p[0] = i4_bits(__hsub2(i4_h2(i4_lop(w, 0x000f000fu, 0x64006400u)), off));
  p[1] = i4_lop(w, 0x00f000f0u, 0x54005400u);
  p[2] = i4_bits(__hsub2(i4_h2(i4_lop(w8, 0x000f000fu, 0x64006400u)), off));
  p[3] = i4_lop(w8, 0x00f000f0u, 0x54005400u);
}

__device__ __forceinline__ void i4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B + C: the first product of a group's sum.
__device__ __forceinline__ void i4_mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, uint4 c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(__uint_as_float(c.x)), "f"(__uint_as_float(c.y)), "f"(__uint_as_float(c.z)), "f"(__uint_as_float(c.w)));
}

// Bytes of one column of staged inputs: the columns of a quarter warp's loads
// fall on different banks.
__host__ __device__ inline int i4_col_bytes(int ktiles) { return ktiles * I4_KT * 2 + 64; }

// The addend of a group's first product, as a lane holds it: -72 times the
// sums of the inputs that meet code + 64, columns 2 t and 2 t + 1 twice.
// [tile of inputs][scale of the tile][column / 2] float4.
template <int NT>
__device__ __forceinline__ float* i4_addend(float* base, int block, int col) {
  return base + (size_t)(block * NT * 4 + (col >> 1)) * 4 + (col & 1);
}

// Lays out tiles [kt0, kt0 + tiles) of `rows` rows of A: 16 lanes per row and
// tile, eight inputs each, in the order 0 4 1 5 2 6 3 7.
template <typename T, int NT, int GB>
__device__ __forceinline__ void i4_stage(const I4Params& p, unsigned char* xs, float* xscale, float* addend, int* special,
                                         int row0, int rows, int kt0, int tiles) {
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 2;
  constexpr int SPT = 4 / GB;
  constexpr int AHEAD = NT == 1 ? (PARTS == 1 ? 4 : 2) : 4;  // loads in flight per lane: the rows come from L2 or beyond
  const int lane16 = threadIdx.x & 15;
  const uint32_t mask = 0xffffu << (threadIdx.x & 16);  // this half of the warp
  const int stride = i4_col_bytes(p.ktiles_cta);
  // A half warp keeps its tile and walks the rows (or, with more tiles than
  // half warps, walks the tiles too).
  const int halves = blockDim.x >> 4, half = threadIdx.x >> 4;
  const int side = max(1, halves / max(tiles, 1));  // half warps per tile
  for (int kt = tiles <= halves ? (half < side * tiles ? half % max(tiles, 1) : tiles) : half; kt < tiles; kt += halves) {
    const int k = (kt0 + kt) * I4_KT + 8 * lane16;
    const bool in = k < p.inner;  // inner is a multiple of 32: eight at once
    const T* src = static_cast<const T*>(p.a) + (size_t)row0 * p.inner + k;
    for (int r0 = tiles <= halves ? half / tiles : 0; r0 < rows; r0 += side * AHEAD) {
      uint4 raw[AHEAD][PARTS];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
          raw[u][q] = in && r0 + u * side < rows ? reinterpret_cast<const uint4*>(src + (size_t)(r0 + u * side) * p.inner)[q]
                                                 : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int r = r0 + u * side;
        if (r >= rows) break;
        uint4 col[PARTS];
        float down = 1.0f;
        if (i4_columns<T>(raw[u], mask, col, down)) special[r] = 1;
        if (PARTS == 2 && lane16 == 0) xscale[r * p.ktiles_cta + kt] = down;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          *reinterpret_cast<uint4*>(xs + (size_t)(r * PARTS + q) * stride + kt * (I4_KT * 2) + lane16 * 16) = col[q];
          // The second and fourth pairs of the eight; four lanes hold 32 inputs.
          const float2 b = __half22float2(i4_h2(col[q].y)), d = __half22float2(i4_h2(col[q].w));
          float sum = (b.x + b.y) + (d.x + d.y);
#pragma unroll
          for (int o = 1; o < 4 * GB; o <<= 1) sum += __shfl_xor_sync(mask, sum, o);
          if (lane16 % (4 * GB) == 0) {
            float* dst = i4_addend<NT>(addend, kt * SPT + lane16 / (4 * GB), r * PARTS + q);
            dst[0] = -72.0f * sum;
            dst[2] = -72.0f * sum;
          }
        }
      }
    }
  }
}

// NT tiles of 8 columns, MT tiles of 16 outputs a warp at a time, GB blocks of
// 32 inputs per scale within a tile (1, 2, or 4: groups of whole tiles).
template <typename T, int NT, int GB>
__global__ void __launch_bounds__(i4_warps(NT) * 32, 1) int4_gemv_kernel(const I4Params p) {
  constexpr int MT = i4_mt(NT);
  extern __shared__ __align__(128) unsigned char i4_smem[];
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 2;  // columns per row
  constexpr int SPT = 4 / GB;                    // scales per tile and output
  constexpr int DEPTH = i4_depth(NT);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same in all lanes, and known to be
  const int g = lane >> 2, t = lane & 3;
  const int wm = warp / p.wk, wk = warp % p.wk;
  const int rank = p.cluster > 1 ? (int)cluster_ctarank() : 0;
  const int row0 = blockIdx.y * p.rows_per_pass;
  const int rows = min(p.rows - row0, p.rows_per_pass);
  const int cols = rows * PARTS;
  const int mtiles = (p.columns + 15) / 16;
  const int mgroups = (mtiles + MT - 1) / MT;           // a warp's outputs, MT tiles each
  const int walk = (int)gridDim.x / p.cluster * p.wm;  // groups of outputs between a warp's
  const int k0 = rank * p.ktiles_cta;                  // this CTA's tiles of inputs
  const int ktiles = max(0, min(p.ktiles_cta, p.ktiles - k0));
  unsigned char* xs = i4_smem;
  const int stride = i4_col_bytes(p.ktiles_cta);
  float* addend = reinterpret_cast<float*>(i4_smem + (size_t)cols * stride);
  float* xscale = addend + (size_t)p.ktiles_cta * SPT * NT * 16;
  int* special = reinterpret_cast<int*>(i4_smem + p.part_offset - I4_COLS * 4);  // rows with infinite or NaN inputs

  struct Slot {
    uint4 code[MT][2];
    T scale[MT][2];  // of the tile's scale t % SPT; lanes exchange them when they are used
  };
  Slot ring[DEPTH];
  // What is loaded next: this warp's tile `lk` of inputs (of the CTA's) for
  // output tile `lm`.  A warp's tiles come in rounds of DEPTH, the last of them
  // perhaps empty.
  const int rounds = (p.ktiles_cta + p.wk * DEPTH - 1) / (p.wk * DEPTH);
  const int round_end = wk + rounds * DEPTH * p.wk;
  const int first = (int)blockIdx.x / p.cluster * p.wm + wm;
  int lm = first, lk = wk, lend = first < mgroups ? ktiles : 0;
  const uint4* lcode[MT];
  const T* lscale[MT];
  auto aim = [&]() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int mt = min(lm * MT + m, mtiles - 1);
      lcode[m] = p.codes + ((size_t)mt * p.ktiles + k0 + lk) * 64 + 4 * g + ((t + (g >> 1)) & 3);
      lscale[m] = static_cast<const T*>(p.scales) + (size_t)mt * p.groups * 16 + g;
    }
  };
  aim();
  auto load = [&](Slot& s) {
    if (lk < lend) {
      const int kt = k0 + lk;
      const int gi = GB == 4 ? (p.group_inv ? (int)__umulhi((uint32_t)kt, p.group_inv) : kt)
                             : min(kt * SPT + (t & (SPT - 1)), p.groups - 1);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        s.code[m][0] = i4_load(lcode[m]);
        s.code[m][1] = i4_load(lcode[m] + 32);
        s.scale[m][0] = __ldg(lscale[m] + gi * 16);
        s.scale[m][1] = __ldg(lscale[m] + gi * 16 + 8);
      }
    }
    lk += p.wk;
#pragma unroll
    for (int m = 0; m < MT; ++m) lcode[m] += p.wk * 64;
    if (lk == round_end) {
      lk = wk;
      lm += walk;
      if (lm >= mgroups) lend = 0;
      aim();
    }
  };
  // The weights too may be the previous kernel's work (a pack, a load): nothing
  // is read before it is done.
  if (tid < I4_COLS) special[tid] = 0;
  __syncthreads();
  pdl_entry();
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(ring[d]);
  i4_stage<T, NT, GB>(p, xs, xscale, addend, special, row0, rows, k0, ktiles);
  __syncthreads();

  uint32_t xcol[NT], xsc[NT];  // shared memory addresses
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    xcol[n] = smem_addr(xs + (size_t)min(n * 8 + g, cols - 1) * stride + t * 16);
    xsc[n] = smem_addr(xscale + min(n * 4 + t, rows - 1) * p.ktiles_cta);  // FP32: columns 2 t and 2 t + 1 are one row
  }
  const uint32_t xadd = smem_addr(addend) + t * 16;
  const int M = p.wm * MT * 16;
  constexpr int PC = NT * 8;
  float* part = reinterpret_cast<float*>(i4_smem + p.part_offset);  // [wk][column][output]
  float* sums = part + (size_t)p.wk * PC * (M + 4);                 // cluster: [parity][row][output]
  const int pm = tid % M, pr = tid / M;  // the output and first row that this thread joins
  const int rstep = (int)blockDim.x / M;   // threads per output
  int parity = 0;
  for (int m0 = (int)blockIdx.x / p.cluster * p.wm; m0 < mgroups; m0 += walk, parity ^= 1) {
    float total[MT][NT][4] = {};
    for (int r = 0; r < rounds; ++r) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int kl = wk + (r * DEPTH + d) * p.wk;
        Slot& s = ring[d];
        if (kl < ktiles && m0 + wm < mgroups) {
#pragma unroll
          for (int b = 0; b < SPT; ++b) {
            float acc[MT][NT][4];
#pragma unroll
            for (int i = b * GB; i < (b + 1) * GB; ++i) {
              uint4 x[NT];
#pragma unroll
              for (int n = 0; n < NT; ++n) x[n] = i4_lds(xcol[n] + kl * (I4_KT * 2) + i * 64);
              uint32_t w0[MT][4], w1[MT][4];
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                i4_expand((&s.code[m][0].x)[i], w0[m]);
                i4_expand((&s.code[m][1].x)[i], w1[m]);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (i == b * GB) {
                  const uint4 c = i4_lds(xadd + (kl * SPT + b) * (NT * 64) + n * 64);
#pragma unroll
                  for (int m = 0; m < MT; ++m) i4_mma_first(acc[m][n], w0[m][0], w1[m][0], w0[m][1], w1[m][1], x[n].x, x[n].y, c);
                } else {
#pragma unroll
                  for (int m = 0; m < MT; ++m) i4_mma(acc[m][n], w0[m][0], w1[m][0], w0[m][1], w1[m][1], x[n].x, x[n].y);
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) i4_mma(acc[m][n], w0[m][2], w1[m][2], w0[m][3], w1[m][3], x[n].z, x[n].w);
              }
            }
            float s0[MT], s1[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              s0[m] = (float)s.scale[m][0];
              s1[m] = (float)s.scale[m][1];
              if constexpr (SPT > 1) {
                s0[m] = __shfl_sync(0xffffffffu, s0[m], (lane & ~3) | b);
                s1[m] = __shfl_sync(0xffffffffu, s1[m], (lane & ~3) | b);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float f = 1.0f;
              if constexpr (PARTS == 2) f = i4_lds_f32(xsc[n] + 4 * kl);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const float f0 = PARTS == 2 ? s0[m] * f : s0[m], f1 = PARTS == 2 ? s1[m] * f : s1[m];
                if constexpr (PARTS == 2) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[m][n][e] *= f;
                }
                total[m][n][0] = fmaf(f0, acc[m][n][0], total[m][n][0]);
                total[m][n][1] = fmaf(f0, acc[m][n][1], total[m][n][1]);
                total[m][n][2] = fmaf(f1, acc[m][n][2], total[m][n][2]);
                total[m][n][3] = fmaf(f1, acc[m][n][3], total[m][n][3]);
              }
            }
          }
        }
        load(s);
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[((size_t)wk * PC + n * 8 + 2 * t + (e & 1)) * (M + 4) + (wm * MT + m) * 16 + g + 8 * (e >> 1)] = total[m][n][e];
    __syncthreads();
    auto finish = [&](int r, float v) {
      const int n = m0 * MT * 16 + pm;
      if (n >= p.columns) return;
      if (p.bias) v += __ldg(p.bias + n);
      i4_finish<T>(p, (size_t)(row0 + r) * p.columns + n, v);
    };
    for (int r = pr; r < rows; r += rstep) {
      float v = 0.0f;
      const float* src = part + (size_t)r * PARTS * (M + 4) + pm;
      for (int w = 0; w < p.wk; ++w, src += PC * (M + 4)) {
        v += src[0];
        if constexpr (PARTS == 2) v += src[M + 4];
      }
      if (special[r] && m0 * MT * 16 + pm < p.columns) v += i4_special<T>(p, row0 + r, m0 * MT * 16 + pm, k0, ktiles);
      if (p.cluster == 1) finish(r, v);
      else sums[(size_t)(parity * rows + r) * M + pm] = v;
    }
    __syncthreads();  // the parts are read (and the sums written)
    if (p.cluster > 1) {
      // Each CTA finishes its share of the rows.  The sums of this parity are
      // written again two tiles on, behind the next tile's barrier.
      cluster_sync();
      for (int r = pr * p.cluster + rank; r < rows; r += rstep * p.cluster) {
        const uint32_t at = smem_addr(sums + (size_t)(parity * rows + r) * M + pm);
        float u[I4_CLUSTER];
#pragma unroll
        for (int c = 0; c < I4_CLUSTER; ++c)
          if (c < p.cluster) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u[c]) : "r"(mapa_shared(at, (uint32_t)c)));
        float v = 0.0f;
#pragma unroll
        for (int c = 0; c < I4_CLUSTER; ++c)
          if (c < p.cluster) v += u[c];
        finish(r, v);
      }
    }
  }
  if (p.cluster > 1) {
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its sums
  }
}

template <typename T, int NT, int GB>
int launch_one(const I4Params& p, dim3 grid, int smem, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(int4_gemv_kernel<T, NT, GB>);
  const int st = set_max_dynamic_smem(kernel, I4_SMEM);
  if (st != PK_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)(p.wm * p.wk * 32));
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cuda_error(cudaLaunchKernelEx(&cfg, int4_gemv_kernel<T, NT, GB>, p), "int4_gemv launch");
}

template <typename T, int NT>
int launch_group(const I4Params& p, int group, dim3 grid, int smem, cudaStream_t stream) {
  if (group == 32) return launch_one<T, NT, 1>(p, grid, smem, stream);
  if (group == 64) return launch_one<T, NT, 2>(p, grid, smem, stream);
  return launch_one<T, NT, 4>(p, grid, smem, stream);
}

template <typename T>
int launch_typed(const DeviceCtx& dev, I4Params p, int group, cudaStream_t stream) {
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 2;
  const int mtiles = (p.columns + 15) / 16;
  int cols = std::min(p.rows * PARTS, I4_COLS);
  int nt = 0, smem = 0, clusters = 0, mgroups = 0;
  // Columns per pass, then CTAs per cluster: the least that fit.
  for (;; cols = std::max(PARTS, cols / 2 / PARTS * PARTS)) {
    p.rows_per_pass = cols / PARTS;
    nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
    const int mt = i4_mt(nt);
    mgroups = (mtiles + mt - 1) / mt;
    // Few tiles per SM: fewer warps to start and to join.  With 4096 inputs 20 warps
    // gain up to 138 tiles per SM (8x4096xN f16: 55 tiles 7.1 us against 7.8 with 28,
    // 111 9.2 against 9.5, 138 9.9 against 10.7) and lose from 166 on (11.9 against
    // 10.8; 221 18.3 against 11.9); with few inputs they lose earlier (8x640x32768, 69
    // tiles, 8.3 against 7.0; 8x1024x32768, 111, 10.5 against 8.0).
    const int warps = nt == 1 && (int64_t)mgroups * p.ktiles < 100 * dev.sm_count ? 20 : i4_warps(nt);
    for (p.cluster = 1; p.cluster <= I4_CLUSTER; p.cluster *= 2) {
      // Few outputs: the inputs over more SMs, while each has a tile for every warp of 4.
      if (mgroups * p.cluster * 2 <= dev.sm_count && p.cluster < I4_CLUSTER && p.ktiles >= p.cluster * 2 * 4) continue;
      p.ktiles_cta = (p.ktiles + p.cluster - 1) / p.cluster;
      const int st = int4_clusters(dev, p.cluster, &clusters);
      if (st != PK_OK) return st;
      const int q = (mgroups + clusters - 1) / clusters;  // groups of outputs of a cluster
      const int turns = (q + warps - 1) / warps;
      p.wm = (q + turns - 1) / turns;
      p.wk = std::max(1, std::min(p.ktiles_cta, warps / p.wm));
      const int spt = group == 32 ? 4 : group == 64 ? 2 : 1;
      p.part_offset = cols * i4_col_bytes(p.ktiles_cta) + p.ktiles_cta * spt * nt * 64;
      p.part_offset = (p.part_offset + (PARTS == 2 ? p.rows_per_pass * p.ktiles_cta * 4 : 0) + I4_COLS * 4 + 127) / 128 * 128;
      smem = p.part_offset + p.wk * nt * 8 * (p.wm * mt * 16 + 4) * 4 +
             (p.cluster > 1 ? 2 * p.rows_per_pass * p.wm * mt * 16 * 4 : 0);
      if (smem <= I4_SMEM) break;
    }
    if (p.cluster <= I4_CLUSTER || cols == PARTS) break;
  }
  if (smem > I4_SMEM) return set_error(PK_E_SHAPE, "int4 products of K=%d do not fit shared memory", p.inner);
  const int passes = (p.rows + p.rows_per_pass - 1) / p.rows_per_pass;
  clusters = std::min(clusters, (mgroups + p.wm - 1) / p.wm);
  const dim3 grid((unsigned)(clusters * p.cluster), (unsigned)passes);
  if (nt == 1) return launch_group<T, 1>(p, group, grid, smem, stream);
  if (nt == 2) return launch_group<T, 2>(p, group, grid, smem, stream);
  return launch_group<T, 4>(p, group, grid, smem, stream);
}

// tcgen05 takes more than 16 columns, and five tiles of 128 x 128 weights per SM
// (counted once per 32 columns).  Below that its pipeline is not filled, and its
// tiles are too coarse to share out (32x1024x4096 f16: 8.3 us against 7.0 here);
// above it, 32x4096x8192 f16 takes 15.0 us against 22.3, 64x4096x4096 21.5
// against 27.1.  With 16 columns it is behind: 16x4096x65536 f16 55 us against 51.
bool umma_route(const DeviceCtx& dev, const I4Params& p, int parts) {
  const int64_t columns = (int64_t)p.rows * parts, tiles = (int64_t)((p.columns + 127) / 128) * p.ktiles;
  return columns > 16 && tiles * ((columns + I4_COLS - 1) / I4_COLS) >= 5 * dev.sm_count;
}

}  // namespace

// Fewer than SMs / cluster: a cluster stays within a GPC, and GPCs differ in size.
int int4_clusters(const DeviceCtx& dev, int cluster, int* out) {
  if (cluster == 1) {
    *out = dev.sm_count;
    return PK_OK;
  }
  static std::mutex mu;
  static std::map<std::pair<int, int>, int> known;
  std::lock_guard<std::mutex> lock(mu);
  int& n = known[{dev.ordinal, cluster}];
  if (n == 0) {
    const void* kernel = reinterpret_cast<const void*>(int4_gemv_kernel<__half, 1, 4>);
    const int st = set_max_dynamic_smem(kernel, I4_SMEM);
    if (st != PK_OK) return st;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)cluster);
    cfg.blockDim = dim3(i4_warps(1) * 32);
    cfg.dynamicSmemBytes = I4_SMEM;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int most = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
    if (e != cudaSuccess) return cuda_error(e, "occupancy query (int4 product)");
    n = std::max(1, most);
  }
  *out = n;
  return PK_OK;
}

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
  p.groups = (int)(d.inner / d.group);
  // Exact for fewer than 2^13 tiles; 0: one tile per group.
  const int per = (int)(d.group / I4_KT);
  p.group_inv = per > 1 ? (uint32_t)((((uint64_t)1 << 32) + per - 1) / per) : 0u;
  p.act = d.activation;
  p.residual_scale = d.residual_scale;
  p.status = dev.status;
  if (umma_route(dev, p, d.precision == PK_FP16 ? 1 : 2)) {
    const int st = launch_int4_umma(dev, p, d.precision, (int)d.group, stream);
    if (st != PK_E_SHAPE) return st;
  }
  return d.precision == PK_FP16 ? launch_typed<__half>(dev, p, (int)d.group, stream)
                                : launch_typed<float>(dev, p, (int)d.group, stream);
}

}  // namespace pk
