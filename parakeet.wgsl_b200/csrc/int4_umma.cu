// int4_umma.cu -- the int4 product on tcgen05, for more than 16 columns
// (int4_gemv.cu has the formula, the layouts, the kernel for few columns and
// the rule between the two).
//
// With 32 columns the mma.sync kernel is bound by its shared memory reads
// of A (once per 16 outputs) and its MMAs.  Here 128 outputs share a read, and
// the expanded weights never pass through shared memory: a decode thread owns
// an output, expands 128 codes of its row to f16 code - 8 and stores them to
// TMEM, the matrix operand of the MMA (M = 128 outputs, N = A's columns).  A's
// columns lie in shared memory (K-major, 128-byte swizzle), laid out once; they
// are split over a cluster's CTAs where they do not fit.
//
// The scale multiplies a group's f32 sum, so every group has an accumulator of
// its own: a ring of them in TMEM, which the epilogue warps read, scale and add
// up in registers, thread = output.  Codes arrive by bulk copies.  Everything is
// a pipeline of warps: two for the copies, 16 that expand, two that issue MMAs
// and four for the epilogue, each place of it owned by one of them.
//
// 16x4096x65536 f32 59 us (mma.sync 86), 32x4096x65536 f16 66 us (94); reading
// the codes takes 21.  No part of it alone is the bound: a tile of 128 x 128 takes
// about 1000 cycles, of which an SM sub-partition issues on 470 (a third of them
// expand), and neither copies nor MMAs nor the expansion hold it up (without the
// expansion 53 us where it takes 58, f32 54 of 59; with an eighth of the copies 57;
// with an eighth of the MMAs the same time).  What is left is the chain of
// hand-overs: a group of decode warps owns one stage of codes and one place in
// TMEM, so that a copy, a store, an MMA and a commit follow one another before its
// next tile.  Register loads instead of bulk copies kept one
// tile on the way whatever the depth asked for (58 us with two groups of
// decode warps); MMAs issued behind `lane == 0` instead of an elected lane took
// 85 cycles each instead of 20.
//
// A CTA has its SM to itself (24 warps of 80 registers, shared memory), so that no two
// clusters wait on each other's TMEM.
#include <algorithm>

#include "int4_common.cuh"

namespace pk {
namespace {

constexpr int IU_M = 128;          // outputs per tile
constexpr int IU_COLS = 32;        // columns of a pass, at most
constexpr int IU_GROUPS = 4;       // groups of four decode warps, a tile of inputs each in turn
constexpr int IU_A = 4;            // expanded tiles in TMEM, 64 columns each
constexpr int IU_STAGES = 4;       // tiles of codes on their way
constexpr int IU_PAIRS = 2;        // pairs of a warp for loads and one for MMAs, a tile each in turn
constexpr int IU_RING = 4;         // accumulators of a pair
// A place belongs to one warp or group, which waits for every use of it in turn.
static_assert(IU_A % IU_GROUPS == 0 && IU_STAGES % IU_GROUPS == 0 && IU_GROUPS % IU_PAIRS == 0, "owners of places");
constexpr int IU_DECODE = IU_GROUPS * 4, IU_EPI = 4;
constexpr int IU_MMA = IU_DECODE + IU_EPI, IU_LOAD = IU_MMA + IU_PAIRS;  // the first of the MMAs' and of the loads' warps
constexpr int IU_THREADS = (IU_LOAD + IU_PAIRS) * 32;
constexpr int IU_TMEM = 512;
static_assert(IU_A * 64 + IU_PAIRS * IU_RING * IU_COLS <= IU_TMEM, "TMEM columns");
constexpr int IU_MIN_SMEM = 120 * 1024;  // more than half an SM's
// Tiles whose scales are held.  Tile q + HELD is expanded when the MMAs of q +
// HELD - IU_A are done; the last of those waited until the epilogue had read the
// accumulator IU_RING before it, IU_RING / spt of the pair's tiles back.
constexpr int iu_held(int spt) { return IU_A + IU_PAIRS * IU_RING / spt; }

struct IuLayout {
  int xscale, codes, scales, sums, special, bars, bytes;
};
constexpr int IU_STAGE = IU_M * 64;  // bytes of 128 outputs' codes
__host__ __device__ inline IuLayout iu_layout(int np, int spt, int parts, int ktiles, int rows) {
  IuLayout l;
  l.xscale = ktiles * np * I4_KT * 2;
  l.codes = l.xscale + (parts == 2 ? ktiles * (np / 2) * 4 : 0);
  l.codes = (l.codes + 127) / 128 * 128;
  l.scales = l.codes + IU_STAGES * IU_STAGE;
  l.sums = l.scales + iu_held(spt) * spt * IU_M * 4;
  l.special = l.sums + 2 * rows * IU_M * 4;
  l.bars = l.special + IU_COLS * 4;
  l.bytes = l.bars + 512 + 1024;  // + alignment slack
  return l;
}

__device__ __forceinline__ void iu_cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void iu_cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// D (+)= A B with A in TMEM: lane = row, 16 f16 in eight columns.
__device__ __forceinline__ void iu_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// `bytes` of global memory to shared memory (16-byte aligned, a multiple of 16).
__device__ __forceinline__ void iu_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// Eight codes -> the pairs (0,4) (1,5) (2,6) (3,7) of code - 8.
__device__ __forceinline__ void iu_expand(uint32_t w, uint32_t* p) {
  auto sub = [](uint32_t u, float off) {
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&u), __float2half2_rn(off));
    return *reinterpret_cast<const uint32_t*>(&h);
  };
  const uint32_t w8 = w >> 8;
  p[0] = sub(i4_lop(w, 0x000f000fu, 0x64006400u), 1032.0f);
  p[1] = sub(i4_lop(w, 0x00f000f0u, 0x54005400u), 72.0f);
  p[2] = sub(i4_lop(w8, 0x000f000fu, 0x64006400u), 1032.0f);
  p[3] = sub(i4_lop(w8, 0x00f000f0u, 0x54005400u), 72.0f);
}

// Lays out tiles [kt0, kt0 + tiles) of `rows` rows of A as columns: blocks of 64
// inputs, NP columns of 128 bytes each.
template <typename T, int NP>
__device__ __forceinline__ void iu_stage(const I4Params& p, unsigned char* xs, float* xscale, int* special, int row0,
                                         int rows, int kt0, int tiles) {
  constexpr int PARTS = sizeof(T) / 2, AHEAD = 4;
  const int lane16 = threadIdx.x & 15;
  const uint32_t mask = 0xffffu << (threadIdx.x & 16);
  const int halves = IU_THREADS / 16, half = threadIdx.x >> 4;
  const int units = rows * tiles;  // a half warp's: (tile, row)
  for (int u0 = half; u0 < units; u0 += halves * AHEAD) {
    uint4 raw[AHEAD][PARTS];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int at = u0 + u * halves, r = at / tiles, k = (kt0 + at - r * tiles) * I4_KT + 8 * lane16;
      const bool in = at < units && k < p.inner;  // inner is a multiple of 32: eight at once
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.a) + (size_t)(row0 + r) * p.inner + k);
#pragma unroll
      for (int q = 0; q < PARTS; ++q) raw[u][q] = in ? src[q] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int at = u0 + u * halves, r = at / tiles, kt = at - r * tiles;
      if (at >= units) break;
      uint4 col[PARTS];
      float down = 1.0f;
      if (i4_columns<T>(raw[u], mask, col, down)) special[r] = 1;
      if (PARTS == 2 && lane16 == 0) xscale[kt * (NP / 2) + r] = down;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) {
        const int n = r * PARTS + q;
        *reinterpret_cast<uint4*>(xs + (size_t)(kt * 2 + (lane16 >> 3)) * (NP * 128) + (n >> 3) * 1024 + (n & 7) * 128 +
                                  (((lane16 & 7) ^ (n & 7)) << 4)) = col[q];
      }
    }
  }
}

// NP columns (16 or 32), GB blocks of 32 inputs per scale within a tile (1,
// 2, or 4: groups of whole tiles).
template <typename T, int NP, int GB>
__global__ void __launch_bounds__(IU_THREADS, 1) int4_umma_kernel(const I4Params p) {
  constexpr int PARTS = sizeof(T) / 2, RP = NP / PARTS;  // columns per row, rows
  constexpr int SPT = 4 / GB, HELD = iu_held(SPT);
  extern __shared__ unsigned char iu_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(iu_raw) + 1023) & ~uintptr_t(1023));
  const IuLayout at = iu_layout(NP, SPT, PARTS, p.ktiles_cta, p.rows_per_pass);
  float* xscale = reinterpret_cast<float*>(sm + at.xscale);
  float* scales = reinterpret_cast<float*>(sm + at.scales);  // [tile % HELD][group of the tile][output]
  float* sums = reinterpret_cast<float*>(sm + at.sums);      // [parity][row][output]
  int* special = reinterpret_cast<int*>(sm + at.special);
  uint64_t* c_full = reinterpret_cast<uint64_t*>(sm + at.bars);  // the stage's codes have landed
  uint64_t* c_empty = c_full + IU_STAGES;                        // and are in registers
  uint64_t* a_full = c_empty + IU_STAGES;                        // the expanded tile is in TMEM
  uint64_t* a_empty = a_full + IU_A;                             // its MMAs are done
  uint64_t* d_full = a_empty + IU_A;                             // the accumulator is complete
  uint64_t* d_empty = d_full + IU_PAIRS * IU_RING;              // and read
  uint64_t* drain = d_empty + IU_PAIRS * IU_RING;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + IU_PAIRS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int rank = p.cluster > 1 ? (int)cluster_ctarank() : 0;
  const int row0 = blockIdx.y * p.rows_per_pass;
  const int rows = min(p.rows - row0, p.rows_per_pass);
  const int mtiles = (p.columns + IU_M - 1) / IU_M;
  const int walk = (int)gridDim.x / p.cluster, first = (int)blockIdx.x / p.cluster;
  const int k0 = rank * p.ktiles_cta;
  const int ktiles = max(0, min(p.ktiles_cta, p.ktiles - k0));
  if (tid < IU_COLS) special[tid] = 0;
  if (tid == 0) {
    for (int i = 0; i < IU_STAGES; ++i) {
      mbar_init(&c_full[i], 1);
      mbar_init(&c_empty[i], 4);
    }
    for (int i = 0; i < IU_A; ++i) {
      mbar_init(&a_full[i], 4);
      mbar_init(&a_empty[i], 2);
    }
    for (int i = 0; i < IU_PAIRS * IU_RING; ++i) {
      mbar_init(&d_full[i], 2);
      mbar_init(&d_empty[i], IU_EPI);
    }
    for (int i = 0; i < IU_PAIRS; ++i) mbar_init(&drain[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // Nothing is read, and no TMEM taken, before the previous kernel is done.
  pdl_entry();

  // A walk over the CTA's tiles: of inputs, then of outputs.
  struct Cursor {
    int m, k, index;
    __device__ __forceinline__ void settle(int ktiles, int walk) {
      while (k >= ktiles) {
        k -= ktiles;
        m += walk;
        ++index;
      }
    }
  };
  auto begin = [&](int k) {
    Cursor c{first, k, 0};
    if (ktiles == 0) c.m = mtiles;
    else c.settle(ktiles, walk);
    return c;
  };
  const int quad = warp & 3, row = quad * 32 + lane;  // the TMEM lane: an output of the tile
  // The loads of tile `c` into stage s: eight tiles of 16 outputs.  One lane
  // issues them (lanes in turn took 120 cycles a copy, one takes 30).
  const bool leader = elect_one();
  const int last_m16 = (p.columns + 15) / 16 - 1;  // outputs behind it are not stored
  auto load = [&](const Cursor& c, uint32_t s) {
    if (leader) {
      mbar_arrive_expect_tx(&c_full[s], IU_STAGE);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int m16 = min(c.m * (IU_M / 16) + i, last_m16);
        iu_copy(sm + at.codes + s * IU_STAGE + i * 1024, p.codes + ((size_t)m16 * p.ktiles + k0 + c.k) * 64, 1024, &c_full[s]);
      }
    }
    __syncwarp();
  };
  Cursor next = begin(warp - IU_LOAD);
  uint32_t loaded = 0;  // of this warp's tiles
  constexpr uint32_t OWN = IU_STAGES / IU_PAIRS;
  if (warp >= IU_LOAD) {
    for (; loaded < OWN && next.m < mtiles; ++loaded) {
      load(next, loaded * IU_PAIRS + warp - IU_LOAD);
      next.k += IU_PAIRS;
      next.settle(ktiles, walk);
    }
  }
  if (warp == IU_MMA) {
    tmem_alloc(tmem_slot, IU_TMEM);
    tmem_relinquish();
  }
  iu_stage<T, NP>(p, sm, xscale, special, row0, rows, k0, ktiles);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, accs = tmem + IU_A * 64;
  const bool plain = __all_sync(0xffffffffu, special[lane] == 0);
  const int turns = first < mtiles ? (mtiles - first + walk - 1) / walk : 0;  // tiles of outputs of this cluster

  // The cluster's barrier has a phase per tile of outputs.  The epilogue joins
  // there; the other warps arrive when they are done with the tile and wait for
  // the phase before they arrive again.
  bool good = true;
  int ended = 0;
  auto end_tiles = [&](int n) {
    if (p.cluster == 1) return;
    for (; ended < n; ++ended) {
      if (ended > 0) iu_cluster_wait();
      iu_cluster_arrive();
    }
  };
  if (warp < IU_DECODE) {
    // ------------------------------------------------------------ codes to TMEM
    uint32_t q = warp >> 2;
    T scale[SPT];  // of the next tile
    auto fetch = [&](const Cursor& c) {
      if (c.m >= mtiles) return;
      const int kt = k0 + c.k;
      const T* src = static_cast<const T*>(p.scales) + (size_t)min(c.m * (IU_M / 16) + (row >> 4), last_m16) * p.groups * 16 + (row & 15);
#pragma unroll
      for (int b = 0; b < SPT; ++b) {
        const int gi = GB == 4 ? (p.group_inv ? (int)__umulhi((uint32_t)kt, p.group_inv) : kt) : min(kt * SPT + b, p.groups - 1);
        scale[b] = __ldg(src + gi * 16);
      }
    };
    Cursor now = begin(warp >> 2);
    fetch(now);
    for (; now.m < mtiles; q += IU_GROUPS) {
      end_tiles(now.index);
      const uint32_t cs = q % IU_STAGES, st = q % IU_A, use = q / IU_A;
      if (good) good = mbar_wait(&c_full[cs], q / IU_STAGES & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_TMA);
      good = __all_sync(0xffffffffu, good);
      if (good) {
        uint4 code[4];
        const unsigned char* stage = sm + at.codes + cs * IU_STAGE;
#pragma unroll
        for (int t = 0; t < 4; ++t) code[t] = i4_lds(smem_addr(stage + row * 64 + ((t + (row >> 1)) & 3) * 16));
        if (use > 0) good = mbar_wait(&a_empty[st], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
        good = __all_sync(0xffffffffu, good);
#pragma unroll
        for (int b = 0; b < SPT; ++b) scales[(q % HELD * SPT + b) * IU_M + row] = (float)scale[b];
        if (good) {
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int t = 0; t < 4; ++t) iu_expand((&code[t].x)[2 * h + i], v + (4 * i + t) * 4);
            tc_st_32x32b_x32(tmem + ((uint32_t)(quad * 32) << 16) + st * 64 + h * 32, v);
          }
          if (lane == 0) mbar_arrive(&c_empty[cs]);  // behind the warp's barrier above: all lanes have read
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&a_full[st]);
        }
      }
      now.k += IU_GROUPS;
      now.settle(ktiles, walk);
      fetch(now);
    }
  } else if (warp >= IU_LOAD) {
    // ------------------------------------------------------------ loads
    for (; next.m < mtiles; ++loaded) {
      end_tiles(next.index);
      const uint32_t s = loaded % OWN * IU_PAIRS + warp - IU_LOAD;
      if (good) good = mbar_wait(&c_empty[s], (loaded / OWN - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_DECODE);
      good = __all_sync(0xffffffffu, good);
      if (!good) break;
      load(next, s);
      next.k += IU_PAIRS;
      next.settle(ktiles, walk);
    }
    // The copies issued have landed before the CTA ends, whatever became of their readers.
    for (uint32_t s = 0; s < OWN; ++s)
      if (loaded > s) mbar_wait_drain(&c_full[s * IU_PAIRS + warp - IU_LOAD], (loaded - s - 1) / OWN & 1, p.status);
  } else if (warp >= IU_MMA) {
    // ------------------------------------------------------------ MMAs
    constexpr uint32_t idesc = umma_idesc_f16(IU_M, NP, 0, 0);
    constexpr uint32_t KT_DESC = 2 * NP * 128 / 16;  // a tile's columns, in a descriptor's address
    const int pair = warp - IU_MMA;
    const uint64_t columns = umma_smem_desc(smem_addr(sm), 16, 1024, 2);
    uint32_t q = pair, a = 0;  // the tile, the pair's accumulator
    for (Cursor now = begin(pair); now.m < mtiles; q += IU_PAIRS) {
      end_tiles(now.index);
      const uint32_t st = q % IU_A;
      if (good) good = mbar_wait(&a_full[st], q / IU_A & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_DECODE);
#pragma unroll
      for (int b = 0; b < SPT; ++b, ++a) {
        const uint32_t slot = pair * IU_RING + a % IU_RING, use = a / IU_RING;
        if (use > 0 && good) good = mbar_wait(&d_empty[slot], (use - 1) & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_EPILOGUE);
        good = __all_sync(0xffffffffu, good);
        if (good && leader) {
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 2 * GB; ++j) {
            const int ks = b * 2 * GB + j;  // of the tile's eight steps of 16 inputs
            iu_mma(accs + slot * NP, tmem + st * 64 + ks * 8, columns + now.k * KT_DESC + (ks >> 2) * (NP * 128 / 16) + 2 * (ks & 3),
                   idesc, j > 0 ? 1u : 0u);
          }
          // The plain arrivals hand on what the decode and epilogue warps wrote and read.
          tc_commit(&d_full[slot]);
          mbar_arrive(&d_full[slot]);
        }
      }
      if (good && leader) {
        tc_commit(&a_empty[st]);
        mbar_arrive(&a_empty[st]);
      }
      now.k += IU_PAIRS;
      now.settle(ktiles, walk);
    }
    // The MMAs issued are complete before TMEM is given back, whoever gave up on them.
    if (leader) {
      tc_commit(&drain[pair]);
      mbar_wait_drain(&drain[pair], 0, p.status);
    }
  } else {
    // ------------------------------------------------------------ scale, add up, store
    uint32_t q = 0;
    for (int i = 0; i < turns; ++i) {
      const int n = (first + i * walk) * IU_M + row;
      float total[RP] = {};
      for (int kt = 0; kt < ktiles; ++kt, ++q) {
#pragma unroll
        for (int b = 0; b < SPT; ++b) {
          const uint32_t a = q / IU_PAIRS * SPT + b, slot = q % IU_PAIRS * IU_RING + a % IU_RING;
          if (good) good = mbar_wait(&d_full[slot], a / IU_RING & 1, abort_flag, p.status, PK_STATUS_TIMEOUT_MMA);
          good = __all_sync(0xffffffffu, good);
          if (good) {
            tc_fence_after();
            const float scale = scales[(q % HELD * SPT + b) * IU_M + row];
            constexpr int LD = NP < 32 ? NP : 32;
#pragma unroll
            for (int c0 = 0; c0 < NP; c0 += LD) {
              uint32_t v[LD];
              const uint32_t from = accs + ((uint32_t)(quad * 32) << 16) + slot * NP + c0;
              if constexpr (LD == 32) tc_ld_32x32b_x32(from, v);
              else tc_ld_32x32b_x16(from, v);
              tc_wait_ld();
              if (c0 + LD == NP) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty[slot]);
              }
              if constexpr (PARTS == 1) {
#pragma unroll
                for (int c = 0; c < LD; ++c) total[c0 + c] = fmaf(scale, __uint_as_float(v[c]), total[c0 + c]);
              } else {
#pragma unroll
                for (int r = 0; r < LD / 2; r += 4) {
                  const float4 f = *reinterpret_cast<const float4*>(xscale + kt * RP + c0 / 2 + r);
                  const float2 fs[2] = {make_float2(f.x, f.y), make_float2(f.z, f.w)};
#pragma unroll
                  for (int j = 0; j < 2; ++j) {  // two rows
                    const uint32_t* w = v + 2 * r + 4 * j;
                    float* to = total + c0 / 2 + r + 2 * j;
                    const float2 u = make_float2(__uint_as_float(w[0]) + __uint_as_float(w[1]),
                                                 __uint_as_float(w[2]) + __uint_as_float(w[3]));
                    const float2 sum = ffma2(fmul2(make_float2(scale, scale), fs[j]), fmul2(u, fs[j]), make_float2(to[0], to[1]));
                    to[0] = sum.x;
                    to[1] = sum.y;
                  }
                }
              }
            }
          }
        }
      }
      // The sums pass through shared memory, so that the epilogue's code is there
      // once and not once per row.
      float* part = sums + (size_t)(i & 1) * p.rows_per_pass * IU_M;
#pragma unroll
      for (int r = 0; r < RP; ++r)
        if (r < rows) part[r * IU_M + row] = total[r];
      if (!plain && n < p.columns) {
        for (int r = 0; r < rows; ++r)
          if (special[r]) part[r * IU_M + row] += i4_special<T>(p, row0 + r, n, k0, ktiles);
      }
      const int to = (first + i * walk) * IU_M + 4 * lane;
      float bias[4] = {};
      if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (to + e < p.columns) bias[e] = __ldg(p.bias + to + e);
      }
      // Each CTA of the cluster finishes its share of the rows, a thread four
      // outputs at a time.  The sums of this parity are written again two tiles
      // on, behind the next tile's barrier.
      if (p.cluster > 1) {
        iu_cluster_arrive();
        iu_cluster_wait();
      } else {
        asm volatile("bar.sync 1, %0;" ::"n"(IU_EPI * 32) : "memory");
      }
      constexpr int AHEAD = 2;  // rows whose parts are on their way
      for (int r0 = rank + quad * p.cluster; r0 < rows; r0 += AHEAD * IU_EPI * p.cluster) {
        float4 u[AHEAD][I4_CLUSTER];
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
#pragma unroll
          for (int c = 0; c < I4_CLUSTER; ++c) {
            const int r = r0 + d * IU_EPI * p.cluster;
            u[d][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (c < p.cluster && r < rows) {
              const uint32_t from = smem_addr(part + r * IU_M + 4 * lane);
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                           : "=f"(u[d][c].x), "=f"(u[d][c].y), "=f"(u[d][c].z), "=f"(u[d][c].w)
                           : "r"(p.cluster > 1 ? mapa_shared(from, (uint32_t)c) : from));
            }
          }
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
          const int r = r0 + d * IU_EPI * p.cluster;
          float v[4] = {};
#pragma unroll
          for (int c = 0; c < I4_CLUSTER; ++c) {
            v[0] += u[d][c].x;
            v[1] += u[d][c].y;
            v[2] += u[d][c].z;
            v[3] += u[d][c].w;
          }
          if (good && r < rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (to + e < p.columns) i4_finish<T>(p, (size_t)(row0 + r) * p.columns + to + e, v[e] + bias[e]);
          }
        }
      }
    }
    ended = turns;
  }
  end_tiles(turns);
  if (p.cluster > 1) {
    if (turns > 0 && (warp < IU_DECODE || warp >= IU_MMA)) iu_cluster_wait();
    iu_cluster_arrive();  // no CTA leaves while another reads its sums
    iu_cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == IU_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, IU_TMEM);
  }
}

template <typename T, int NP, int GB>
int launch_one(const I4Params& p, dim3 grid, int smem, cudaStream_t stream) {
  const int st = set_max_dynamic_smem(reinterpret_cast<const void*>(int4_umma_kernel<T, NP, GB>), I4_SMEM);
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
  cfg.blockDim = dim3(IU_THREADS);
  cfg.dynamicSmemBytes = (size_t)std::max(smem, IU_MIN_SMEM);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  return cuda_error(cudaLaunchKernelEx(&cfg, int4_umma_kernel<T, NP, GB>, p), "int4_umma launch");
}

template <typename T, int NP>
int launch_group(const I4Params& p, int group, dim3 grid, int smem, cudaStream_t stream) {
  if (group == 32) return launch_one<T, NP, 1>(p, grid, smem, stream);
  if (group == 64) return launch_one<T, NP, 2>(p, grid, smem, stream);
  return launch_one<T, NP, 4>(p, grid, smem, stream);
}

template <typename T>
int launch_typed(const DeviceCtx& dev, I4Params p, int group, cudaStream_t stream) {
  constexpr int PARTS = sizeof(T) / 2;
  const int mtiles = (p.columns + IU_M - 1) / IU_M, spt = group == 32 ? 4 : group == 64 ? 2 : 1;
  int np = 0, smem = 0;
  // Columns per pass, then CTAs per cluster: the least that fit.
  for (int cols = std::min(p.rows * PARTS, IU_COLS);; cols /= 2) {
    np = cols <= 16 ? 16 : 32;
    p.rows_per_pass = std::min(p.rows, cols / PARTS);
    for (p.cluster = 1; p.cluster <= I4_CLUSTER; p.cluster *= 2) {
      // Few outputs: the inputs over more SMs, while each has a few tiles.
      if (mtiles * p.cluster * 2 <= dev.sm_count && p.cluster < I4_CLUSTER && p.ktiles >= p.cluster * 2 * 4) continue;
      p.ktiles_cta = (p.ktiles + p.cluster - 1) / p.cluster;
      smem = iu_layout(np, spt, PARTS, p.ktiles_cta, p.rows_per_pass).bytes;
      if (smem <= I4_SMEM) break;
    }
    if (p.cluster <= I4_CLUSTER || cols <= 16) break;
  }
  if (smem > I4_SMEM) return PK_E_SHAPE;
  int clusters = 0;
  const int st = int4_clusters(dev, p.cluster, &clusters);
  if (st != PK_OK) return st;
  const dim3 grid((unsigned)(std::min(clusters, mtiles) * p.cluster), (unsigned)((p.rows + p.rows_per_pass - 1) / p.rows_per_pass));
  if (np == 16) return launch_group<T, 16>(p, group, grid, smem, stream);
  return launch_group<T, 32>(p, group, grid, smem, stream);
}

}  // namespace

// PK_E_SHAPE where even 16 columns of A do not fit a cluster's shared memory.
int launch_int4_umma(const DeviceCtx& dev, const I4Params& p, int precision, int group, cudaStream_t stream) {
  return precision == PK_FP16 ? launch_typed<__half>(dev, p, group, stream) : launch_typed<float>(dev, p, group, stream);
}

}  // namespace pk
