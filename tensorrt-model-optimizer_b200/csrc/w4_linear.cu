// Products of a few rows with 4-bit weights:  out[m, n] = T(sum_k x[m, k] W[n, k] + bias[n])  with
//   INT4   W = (code - 8) / scale, one scale of type T per row and group (INT4QTensor; even element in the high nibble)
//   NVFP4  W = e2m1 * e4m3 * scale2, one E4M3 scale per row and 16 elements (NVFP4QTensor; even element in the low nibble)
// The weight is read once, in the layout it is stored in; nothing is dequantised to memory.
//
// What bounds it: 0.52 / 0.56 bytes a weight from HBM.  At the measured copy rate an SM gets 46 weights a clock,
// so a warp that handles 2048 weights (16 rows x 128) has about 180 issue slots for them; the conversions take 72
// (INT4: one mask and one add or multiply-add for two weights) or 64 (NVFP4: one conversion and one multiply).
//
// Mathematics.  mma.m16n8k16 with 16 weight rows as the rows and 8 rows of x as the columns.  code - 8 is an exact
// fp16 (1024 + code, minus 1032), and e2m1 * e4m3 is one too (six significant bits, [2^-10, 2688]); the INT4 scale
// multiplies the fp32 sum of its group, scale2 the result.  x in bf16 is multiplied by a power of two per row that
// brings the largest element of the CTA's part to [2^14, 2^15): exact in fp16 down to 2^-29 of it, and below that
// off by less than 2^-39 of it, far under the 2^-24 of the fp32 sums.  The k order inside a product is free, so a
// lane's operand is a contiguous run of the packed row and x is put into shared memory in that order.
//
// Work.  A cluster of 1 to 8 CTAs shares a tile of 16 weight rows, K split over its CTAs and over their 8 warps,
// and walks over the row tiles with its part of x resident in shared memory.  Each lane fetches its own operands
// with cp.async into a ring (kStages x 1 KB a warp, so 96 KB in flight on an SM), which runs on across tiles.
// Partial sums meet in shared memory, across the cluster through distributed shared memory, in a fixed order.
#include <atomic>

#include "umma.cuh"

namespace b200q {

constexpr int kW4Warps = 16, kW4Threads = 32 * kW4Warps;
constexpr int kW4Rows = 16;                  // weight rows of a tile
constexpr int kSlab = 128;                   // k elements a warp handles at a time
#ifndef W4ST
#define W4ST 3
#endif
constexpr int kW4Stages = W4ST;               // of two slabs
constexpr int kStageBytes = 2048;

struct W4Args {
  const void* x;
  int64_t x_stride;                          // elements
  const uint8_t* codes;                      // [n, k/2]
  const void* scales;                        // INT4: T [n, k/block]; NVFP4: E4M3 [n, k/16]
  const float* scale2;                       // NVFP4
  const void* bias;                          // T [n] or NULL
  void* out;                                 // [rows, n]
  int64_t out_stride;
  int rows, n, k, groups, group_slabs;       // groups a row; slabs a group (groups of 128 and more)
  int slabs_per_cta, tiles, wk, ks;
  FastDiv pairs;                             // slab pairs of a CTA
};

__device__ __forceinline__ uint32_t w4_pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void w4_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with a zero accumulator
__device__ __forceinline__ void w4_mma_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

// 8 INT4 codes -> code - 8 as fp16, in the order (1, 5), (0, 4), (3, 7), (2, 6) of the elements
__device__ __forceinline__ void int4x8_to_f16(uint32_t w, uint32_t* h) {
  const uint32_t w8 = w >> 8;
  uint32_t p0, p1, p2, p3;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p0) : "r"(w), "n"(0x000f000f), "n"(0x64006400));   // (a & b) | c
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p1) : "r"(w), "n"(0x00f000f0), "n"(0x64006400));
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p2) : "r"(w8), "n"(0x000f000f), "n"(0x64006400));
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(p3) : "r"(w8), "n"(0x00f000f0), "n"(0x64006400));
  const uint32_t m1032 = 0xe408e408u, m72 = 0xd480d480u, r16 = 0x2c002c00u;   // -1032, -72, 1/16
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(h[0]) : "r"(p0), "r"(m1032));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(h[1]) : "r"(p1), "r"(r16), "r"(m72));
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(h[2]) : "r"(p2), "r"(m1032));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(h[3]) : "r"(p3), "r"(r16), "r"(m72));
}
// 8 E2M1 codes -> fp16 in element order
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t w4_hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
enum { kFmtInt4 = 0, kFmtNvfp4 = 1 };

// LW: words (of 8 codes) in a lane's contiguous run.  Lane qd of a quad holds the elements
//   slab * 128 + (i / LW) * 32 LW + qd * 8 LW + 8 (i % LW) + 0..7   for i = 0..3,
// so that an instruction's 16 elements always lie in one group of 32 LW (INT4 groups of 32, 64, 128 n).
template <int FMT, typename T, int NT, int LW>
__global__ void __launch_bounds__(kW4Threads, 1)
w4_linear_kernel(const W4Args a) {
  constexpr int kSegs = 4 / LW;                     // groups a slab has (at least)
  constexpr int kRunBytes = 4 * LW;
  constexpr int kPart = kW4Rows * 8 * NT;           // partial sums of a warp
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t xmax[8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qd = lane & 3, gr = lane >> 2;
  const int ks = a.ks, wk = a.wk, wr = kW4Warps / wk;
  const int rank = static_cast<int>(cluster_ctarank());
  const int cluster = blockIdx.x / ks, nclusters = gridDim.x / ks;
  const int slab0 = rank * a.slabs_per_cta;
  const int slabs = max(min(a.slabs_per_cta, (a.k + kSlab - 1) / kSlab - slab0), 0);
  const int my_row = warp / wk, my_k = warp % wk;   // which of the CTA's tiles, which part of its slabs

  uint8_t* ring = smem + warp * kW4Stages * kStageBytes;      // [stages][2 slabs][2 rows][32 lanes][16 B]
  uint8_t* xs = smem + kW4Warps * kW4Stages * kStageBytes; // [slab][i][row][qd] 16 B
  float* part = reinterpret_cast<float*>(xs + static_cast<int64_t>(a.pairs.d) * 2 * kSlab * 2 * a.rows);   // [warps][8 NT][16], wk > 1
  float* recv = part + (wk > 1 ? kW4Warps * kPart : 0);                           // [ks][wr * 16 * rows / ks], ks > 1
  const uint32_t ring_addr = smem_u32(ring) + lane * 16;

  pdl_prologue();

  // tiles of round t: (t * wr + my_row) * nclusters + cluster, so that the last round is spread over the SMs
  const int npairs = (slabs + 1) / 2;
  const int mine = npairs > my_k ? (npairs - my_k + wk - 1) / wk : 0;             // slab pairs of this warp in each tile
  const int first_tile = my_row * nclusters + cluster, tile_step = wr * nclusters;
  const int rounds = (a.tiles - cluster + tile_step - 1) / tile_step;             // of the CTA
  const int my_tiles = a.tiles > first_tile ? (a.tiles - first_tile + tile_step - 1) / tile_step : 0;
  const int steps = mine * my_tiles;
  const int64_t row_bytes = a.k / 2;

  // ---- producer: this lane's operands of two slabs of one tile ----
  // Addresses are kept as pointers that step through a tile's slabs: the arithmetic of an address from
  // scratch costs as many issue slots as the conversions.
  const int slab_first = slab0 + 2 * my_k;
  const int code_step = wk * kSlab;
  auto row_of = [&](int tile, int r) { return static_cast<int64_t>(min(tile * kW4Rows + gr + 8 * r, a.n - 1)); };
  const int64_t code_first = slab_first * (kSlab / 2) + qd * kRunBytes;
  const uint8_t *pc0 = a.codes, *pc1 = a.codes;
  int p_tile = first_tile, p_i = 0, p_left = steps, p_k = 0;
  uint32_t p_dst = ring_addr;
  auto produce = [&]() {
    if (p_left > 0) {
      if (p_i == 0) {
        pc0 = a.codes + row_of(p_tile, 0) * row_bytes + code_first;
        pc1 = a.codes + row_of(p_tile, 1) * row_bytes + code_first;
        p_k = slab_first * kSlab + qd * 8 * LW;
        p_tile += tile_step;
      }
#pragma unroll
      for (int seg = 0; seg < 2 * kSegs; ++seg) {
        const uint32_t to = p_dst + (seg / kSegs) * 1024 + (seg % kSegs) * kRunBytes;
        if (p_k + seg * 32 * LW < a.k) {
          copy_async<kRunBytes>(to, pc0 + seg * 16 * LW);
          copy_async<kRunBytes>(to + 512, pc1 + seg * 16 * LW);
        }
      }
      pc0 += code_step;
      pc1 += code_step;
      p_k += 2 * code_step;
      p_i = p_i + 1 == mine ? 0 : p_i + 1;
      --p_left;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int s = 0; s < kW4Stages - 1; ++s) {
    p_dst = ring_addr + s * kStageBytes;
    produce();
  }

  // ---- scales, two slabs ahead of their use ----
  constexpr int kScales = FMT == kFmtInt4 ? 2 * kSegs : 2;                        // of a row in two slabs
  constexpr int kScaleSize = FMT == kFmtInt4 ? 2 : 1;
  using Raw = typename std::conditional<FMT == kFmtInt4, T, uint16_t>::type;      // INT4: a group's scale; NVFP4: two E4M3
  Raw nxt[2][kScales];
  const uint8_t *ps0 = nullptr, *ps1 = nullptr;     // the row's scales
  int s_tile = first_tile, s_i = 0, s_left = steps, s_at = 0;
  auto load_scales = [&]() {
    if (s_left > 0) {
      if (s_i == 0) {
        ps0 = static_cast<const uint8_t*>(a.scales) + row_of(s_tile, 0) * a.groups * kScaleSize;
        ps1 = static_cast<const uint8_t*>(a.scales) + row_of(s_tile, 1) * a.groups * kScaleSize;
        s_at = FMT == kFmtInt4 ? slab_first * kSegs : slab_first * (kSlab / 16) + 2 * qd;
        s_tile += tile_step;
      }
#pragma unroll
      for (int seg = 0; seg < kScales; ++seg) {
        int at = FMT == kFmtInt4 ? s_at + seg : s_at + seg * (kSlab / 16);
        if (FMT == kFmtInt4 && LW == 4 && a.group_slabs > 1) at /= a.group_slabs;
        at = min(at, a.groups - (FMT == kFmtInt4 ? 1 : 2));                        // behind the end of a row x is zero
        nxt[0][seg] = __ldg(reinterpret_cast<const Raw*>(ps0 + at * kScaleSize));
        nxt[1][seg] = __ldg(reinterpret_cast<const Raw*>(ps1 + at * kScaleSize));
      }
      s_at += FMT == kFmtInt4 ? 2 * wk * kSegs : 2 * wk * (kSlab / 16);
      s_i = s_i + 1 == mine ? 0 : s_i + 1;
      --s_left;
    }
  };
  load_scales();

  // ---- x into shared memory, as fp16 times a power of two ----
  // A warp takes two slabs of a row at a time; lane = 16 (slab) + 4 (word i) + q, so that the stores of eight lanes hit
  // all banks (two at a time where the rows are even).  All loads are issued before the first is used; the maximum and
  // the conversion both work on the registers.
  constexpr int kHold = 18;                         // of 16 warps: all that shared memory has room for, almost
  const T* x = static_cast<const T*>(a.x);
  const int units = a.rows * static_cast<int>(a.pairs.d);
  const int x_i = (lane >> 2) & 3, x_q = lane & 3;
  const int x_k = slab0 * kSlab + (lane >> 4) * kSlab + ((x_i / LW) * 4 * LW + x_q * LW + x_i % LW) * 8;
  auto load_x = [&](int u) {
    uint32_t row, pair;
    a.pairs.divmod(u, row, pair);
    const int k = x_k + pair * (2 * kSlab);
    return k < a.k ? __ldg(reinterpret_cast<const uint4*>(x + row * a.x_stride + k)) : make_uint4(0, 0, 0, 0);
  };
  auto max_x = [&](int u, const uint4& v) {
    uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16);
    if (m >= 0x7f80u) {                             // infinity or NaN: the largest of the others
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      m = 0;
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = w[j] & 0x7fffu, hi = (w[j] >> 16) & 0x7fffu;
        m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
      }
    }
    m = warp_max_u32(m);
    if (lane == 0 && m) atomicMax(&xmax[a.pairs.div(u)], m);
  };
  auto store_x = [&](int u, const uint4& v) {
    uint32_t row, pair;
    a.pairs.divmod(u, row, pair);
    const int slab = 2 * pair + (lane >> 4);
    uint32_t h[4] = {v.x, v.y, v.z, v.w};
    if constexpr (kBf16) {
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - max(static_cast<int>(xmax[row] >> 7), 28)) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = w4_pack_f16(__uint_as_float(h[j] << 16) * up, __uint_as_float(h[j] & 0xffff0000u) * up);
    }
    uint4 o;
    if constexpr (FMT == kFmtInt4) {                // (1, 5), (0, 4), (3, 7), (2, 6)
      o.x = __byte_perm(h[0], h[2], 0x7632);
      o.y = __byte_perm(h[0], h[2], 0x5410);
      o.z = __byte_perm(h[1], h[3], 0x7632);
      o.w = __byte_perm(h[1], h[3], 0x5410);
    } else {
      o = make_uint4(h[0], h[1], h[2], h[3]);
    }
    *reinterpret_cast<uint4*>(xs + (((slab * 4 + x_i) * a.rows + static_cast<int>(row)) * 4 + x_q) * 16) = o;
  };
  uint4 hold[kHold];
#pragma unroll
  for (int j = 0; j < kHold; ++j) {
    if (warp + j * kW4Warps >= units) break;
    hold[j] = load_x(warp + j * kW4Warps);
  }
  if constexpr (kBf16) {
    if (threadIdx.x < 8 * NT) xmax[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHold; ++j) {
      if (warp + j * kW4Warps >= units) break;
      max_x(warp + j * kW4Warps, hold[j]);
    }
#pragma unroll 1
    for (int u = warp + kHold * kW4Warps; u < units; u += kW4Warps) max_x(u, load_x(u));
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kHold; ++j) {
    if (warp + j * kW4Warps >= units) break;
    store_x(warp + j * kW4Warps, hold[j]);
  }
#pragma unroll 1
  for (int u = warp + kHold * kW4Warps; u < units; u += kW4Warps) store_x(u, load_x(u));
  if (ks > 1) cluster_barrier(); else __syncthreads();   // the others' shared memory may be written from here on

  float back[NT][2];                                // of the columns this thread's sums belong to
  const float s2 = FMT == kFmtNvfp4 ? __ldg(a.scale2) : 1.f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * qd + j;
      back[n][j] = s2;
      if constexpr (kBf16)
        if (row < a.rows) back[n][j] *= __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(xmax[row] >> 7), 28) - 14) << 23);
    }

  auto store = [&](int row, int col, float sum) {
    if (col >= a.n) return;
    if (a.bias) sum += Elem<T>::to_float(static_cast<const T*>(a.bias)[col]);
    static_cast<T*>(a.out)[row * a.out_stride + col] = Elem<T>::from_float(sum);
  };

  uint32_t slot = 0;                                // ring offset of the slab at hand
  p_dst = ring_addr + (kW4Stages - 1) * kStageBytes;
  const uint8_t* lane_ring = ring + lane * 16;
  // x of row 8 n + gr; columns beyond the last row repeat it, their sums are dropped
  const uint8_t* lane_x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) lane_x[n] = xs + (min(8 * n + gr, a.rows - 1) * 4 + qd) * 16;
  const int word_step = 4 * a.rows * 16, slab_step = 4 * word_step;
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    const int tile = first_tile + round * tile_step;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const int todo = tile < a.tiles ? mine : 0;
#pragma unroll 1
    for (int it = 0; it < todo; ++it) {
      const uint8_t* xp[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) xp[n] = lane_x[n] + 2 * (my_k + it * wk) * slab_step;
      Raw cur[2][kScales];
#pragma unroll
      for (int seg = 0; seg < kScales; ++seg) { cur[0][seg] = nxt[0][seg]; cur[1][seg] = nxt[1][seg]; }
      load_scales();
      asm volatile("cp.async.wait_group %0;" ::"n"(kW4Stages - 2) : "memory");
#pragma unroll
      for (int half = 0; half < 2; ++half) {        // behind the end of K x is zero, and the codes whatever they are
        const uint4 va = *reinterpret_cast<const uint4*>(lane_ring + slot + half * 1024);
        const uint4 vb = *reinterpret_cast<const uint4*>(lane_ring + slot + half * 1024 + 512);
        const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
        uint32_t sc[2][2];
        if constexpr (FMT == kFmtNvfp4) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t h;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(cur[r][half]));
            sc[r][0] = __byte_perm(h, h, 0x1010);
            sc[r][1] = __byte_perm(h, h, 0x3232);
          }
        }
        float tmp[NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t fa[4], fb[4];
          if constexpr (FMT == kFmtInt4) {
            int4x8_to_f16(wa[i], fa);
            int4x8_to_f16(wb[i], fb);
          } else {
            e2m1x8_to_f16(wa[i], fa);
            e2m1x8_to_f16(wb[i], fb);
#pragma unroll
            for (int j = 0; j < 4; ++j) { fa[j] = w4_hmul2(fa[j], sc[0][i / 2]); fb[j] = w4_hmul2(fb[j], sc[1][i / 2]); }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 b = *reinterpret_cast<const uint4*>(xp[n] + i * word_step);
            if constexpr (FMT == kFmtInt4) {
              if (i % LW == 0) w4_mma_first(tmp[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
              else w4_mma(tmp[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
              w4_mma(tmp[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
              if (i % LW == LW - 1) {
                const int seg = half * kSegs + i / LW;
                const float i0 = rcp_approx(Elem<T>::to_float(cur[0][seg])), i1 = rcp_approx(Elem<T>::to_float(cur[1][seg]));
                acc[n][0] += tmp[n][0] * i0; acc[n][1] += tmp[n][1] * i0;
                acc[n][2] += tmp[n][2] * i1; acc[n][3] += tmp[n][3] * i1;
              }
            } else {
              w4_mma(acc[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
              w4_mma(acc[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) xp[n] += slab_step;
      }
      produce();                                    // into the slot read one step ago
      p_dst = ring_addr + slot;
      slot = slot == (kW4Stages - 1) * kStageBytes ? 0 : slot + kStageBytes;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] *= back[n][j & 1];

    // ---- sums of the K parts, always in the order of the warps and CTAs ----
    const int elems = kW4Rows * a.rows;             // of a tile
    const int per = wr * elems / ks;                // of the CTA's tiles that one CTA of the cluster finishes
    auto push = [&](int e, float v) {               // element e of the CTA's tiles to the CTA that finishes it
      const uint32_t to = map_to_cta(recv + rank * per + e % per, e / per);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
    };
    if (wk > 1) {
      float* p = part + warp * kPart;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[gr + 8 * (j >> 1) + kW4Rows * (8 * n + 2 * qd + (j & 1))] = acc[n][j];
      __syncthreads();
      for (int e = threadIdx.x; e < wr * elems; e += kW4Threads) {
        const int t = e / elems, in = e - t * elems;
        float sum = 0.f;
        for (int w = 0; w < wk; ++w) sum += part[(t * wk + w) * kPart + in];
        if (ks > 1) push(e, sum);
        else store(in / kW4Rows, (first_tile - my_row * nclusters + round * tile_step + t * nclusters) * kW4Rows + in % kW4Rows, sum);
      }
      if (ks == 1) __syncthreads();                 // read before the next round writes
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int wrow = gr + 8 * (j >> 1), row = 8 * n + 2 * qd + (j & 1);
          if (row >= a.rows) continue;
          if (ks > 1) push(my_row * elems + row * kW4Rows + wrow, acc[n][j]);
          else if (tile < a.tiles) store(row, tile * kW4Rows + wrow, acc[n][j]);
        }
    }
    if (ks > 1) {
      cluster_barrier();
      for (int i = threadIdx.x; i < per; i += kW4Threads) {
        float sum = 0.f;
        for (int c = 0; c < ks; ++c) sum += recv[c * per + i];
        const int e = rank * per + i, t = e / elems, in = e - t * elems;
        store(in / kW4Rows, (cluster + round * tile_step + t * nclusters) * kW4Rows + in % kW4Rows, sum);
      }
      if (round + 1 < rounds) cluster_barrier();    // read before the next round's sums arrive
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

inline size_t w4_smem(int rows, int nt, int slabs, int wk, int ks) {
  return kW4Warps * kW4Stages * kStageBytes + static_cast<size_t>((slabs + 1) / 2 * 2) * kSlab * 2 * rows +
         (wk > 1 ? kW4Warps * kW4Rows * 8 * 4 * static_cast<size_t>(nt) : 0) +
         (ks > 1 ? static_cast<size_t>(kW4Warps / wk) * kW4Rows * 4 * rows : 0);
}
constexpr size_t kW4SmemLimit = 227 * 1024 - 1024;
inline int w4_nt(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// How K is cut: over the wk warps of a tile and the ks CTAs of a cluster.  x decides the least ks (its part has to fit
// beside the ring); then wk and after it ks grow until every warp of the GPU has a tile part, while a part keeps two slabs.
inline bool w4_cut(int rows, int slabs, int tiles, int sms, int& wk, int& ks) {
  const int nt = w4_nt(rows);
  for (ks = 1; ks < 8 && w4_smem(rows, nt, (slabs + ks - 1) / ks, 1, ks) > kW4SmemLimit; ks *= 2) {}
  wk = 1;
  auto fits = [&](int w, int c) { return w4_smem(rows, nt, (slabs + c - 1) / c, w, c) <= kW4SmemLimit; };
  if (!fits(1, ks)) return false;
  auto more = [&] { return static_cast<int64_t>(tiles) * wk * ks * 4 < 3ll * sms * kW4Warps && slabs >= 4 * wk * ks; };
  while (wk < kW4Warps && more() && fits(2 * wk, ks)) wk *= 2;
  while (ks < 8 && more() && fits(wk, 2 * ks)) ks *= 2;
  return true;
}

template <int FMT, typename T, int NT, int LW>
int launch_w4(W4Args a, cudaStream_t s) {
  auto kern = w4_linear_kernel<FMT, T, NT, LW>;
  const int slabs = (a.k + kSlab - 1) / kSlab, sms = sm_count_cached();
  if (!w4_cut(a.rows, slabs, a.tiles, sms, a.wk, a.ks)) return B200Q_ERR_CAPACITY;
  a.slabs_per_cta = ((slabs + a.ks - 1) / a.ks + 1) / 2 * 2;
  a.pairs = FastDiv(a.slabs_per_cta / 2);
  const size_t smem = w4_smem(a.rows, NT, a.slabs_per_cta, a.wk, a.ks);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kW4SmemLimit)) != cudaSuccess)
    return B200Q_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(a.ks);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  int room = sms / a.ks;                            // clusters the GPU holds at a time (they need SMs of one GPC)
  if (a.ks > 2) {
    static std::atomic<int> cached[2];              // clusters of 4, of 8; every block has an SM to itself
    int c = cached[a.ks == 4 ? 0 : 1];
    if (c == 0) {
      int got = 0;
      cfg.gridDim = dim3(static_cast<unsigned>(room * a.ks));
      if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) == cudaSuccess && got > 0)
        cached[a.ks == 4 ? 0 : 1] = c = got;
    }
    if (c > 0) room = min(room, c);
  }
  const int clusters = max(1, min(a.tiles, room));
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * a.ks));
  cudaLaunchKernelEx(&cfg, kern, a);
  return launch_status();
}

template <int FMT, int LW>
int dispatch_w4(const W4Args& a, int dtype, cudaStream_t s) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (a.rows <= 8) return launch_w4<FMT, T, 1, LW>(a, s);
    if (a.rows <= 16) return launch_w4<FMT, T, 2, LW>(a, s);
    return launch_w4<FMT, T, 4, LW>(a, s);
  };
  return dtype == B200Q_F16 ? go(__half()) : go(__nv_bfloat16());
}

inline int w4_check(const void* x, int64_t x_stride, int dtype, const uint8_t* codes, const void* scales, const void* out, int64_t out_stride,
                    int rows, int64_t n, int64_t k) {
  B200Q_REQUIRE_PTR(x); B200Q_REQUIRE_PTR(codes); B200Q_REQUIRE_PTR(scales); B200Q_REQUIRE_PTR(out);
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_DTYPE;
  if (rows <= 0 || n <= 0 || k <= 0 || k % 32 || x_stride < 0 || out_stride < n) return B200Q_ERR_SHAPE;
  if (rows > 32 || n > (1 << 30) || k > (1 << 24)) return B200Q_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) | static_cast<uintptr_t>(2 * x_stride)) & 15u) ||
      (reinterpret_cast<uintptr_t>(scales) & 1u))
    return B200Q_ERR_ALIGN;
  return B200Q_OK;
}

inline W4Args w4_args(const void* x, int64_t x_stride, const uint8_t* codes, const void* scales, const float* scale2,
                      const void* bias, void* out, int64_t out_stride, int rows, int64_t n, int64_t k, int block) {
  W4Args a{};
  a.x = x; a.x_stride = x_stride; a.codes = codes; a.scales = scales; a.scale2 = scale2; a.bias = bias;
  a.out = out; a.out_stride = out_stride;
  a.rows = rows; a.n = static_cast<int>(n); a.k = static_cast<int>(k);
  a.groups = static_cast<int>(k / block);
  a.group_slabs = block >= kSlab ? block / kSlab : 1;
  a.tiles = (a.n + kW4Rows - 1) / kW4Rows;
  return a;
}

}  // namespace b200q

using namespace b200q;

extern "C" int b200q_w4_linear_max_rows(int64_t k) {
  if (k <= 0 || k % 32 || k > (1 << 24)) return 0;
  const int slabs = static_cast<int>((k + kSlab - 1) / kSlab);
  for (int rows = 32; rows > 0; --rows)
    if (w4_smem(rows, w4_nt(rows), (slabs + 7) / 8, 1, 8) <= kW4SmemLimit) return rows;
  return 0;
}

extern "C" int b200q_int4_linear(const void* x, int64_t x_stride, int dtype, const uint8_t* codes, const void* scales, int block,
                                 const void* bias, void* out, int64_t out_stride, int rows, int64_t n, int64_t k, void* stream) {
  if (const int r = w4_check(x, x_stride, dtype, codes, scales, out, out_stride, rows, n, k)) return r;
  if (block <= 0 || k % block) return B200Q_ERR_SHAPE;
  if (block != 32 && block != 64 && block % kSlab) return B200Q_ERR_UNSUPPORTED;
  const W4Args a = w4_args(x, x_stride, codes, scales, nullptr, bias, out, out_stride, rows, n, k, block);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (block == 32) return dispatch_w4<kFmtInt4, 1>(a, dtype, s);
  if (block == 64) return dispatch_w4<kFmtInt4, 2>(a, dtype, s);
  return dispatch_w4<kFmtInt4, 4>(a, dtype, s);
}

extern "C" int b200q_nvfp4_linear(const void* x, int64_t x_stride, int dtype, const uint8_t* codes, const uint8_t* scales,
                                  const float* scale2, const void* bias, void* out, int64_t out_stride, int rows, int64_t n,
                                  int64_t k, void* stream) {
  if (const int r = w4_check(x, x_stride, dtype, codes, scales, out, out_stride, rows, n, k)) return r;
  B200Q_REQUIRE_PTR(scale2);
  const W4Args a = w4_args(x, x_stride, codes, scales, scale2, bias, out, out_stride, rows, n, k, 16);
  return dispatch_w4<kFmtNvfp4, 4>(a, dtype, static_cast<cudaStream_t>(stream));
}
