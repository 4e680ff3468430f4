// Products of a few rows with 4-bit weights:  out[m, n] = T(sum_k x[m, k] W[n, k] + bias[n])  with
//   INT4   W = (code - 8) / scale, one scale of type T per row and group (INT4QTensor; even element in the high nibble)
//   NVFP4  W = e2m1 * e4m3 * scale2, one E4M3 scale per row and 16 or 32 elements (NVFP4QTensor; even element in the low
//          nibble)
// The weight is read once, in the layout it is stored in; nothing is dequantised to memory.
//
// What bounds it: 0.52 / 0.56 bytes a weight from HBM.  At the measured copy rate an SM gets 46 weights a clock,
// so a warp that handles 2048 weights (16 rows x 128) has about 180 issue slots for them; the conversions take 72
// (INT4: one mask and one add or multiply-add for two weights) or 64 (NVFP4: one conversion and one multiply).
//
// Mathematics.  mma.m16n8k16 with 16 weight rows as the rows and 8 rows of x as the columns.  code - 8 is an exact
// fp16 (1024 + code, minus 1032), and e2m1 * e4m3 is one too (six significant bits, [2^-10, 2688]); the INT4 scale
// multiplies the fp32 sum of its group, scale2 the result.  x in bf16, and in fp16 where half of it is divided by 16
// (INT4), is multiplied by a power of two per row that brings the largest element of the CTA's part to [2^14, 2^15):
// exact in fp16 down to 2^-29 of it (2^-25 where divided), and below that off by less than 2^-35 of it, far under the
// 2^-24 of the fp32 sums.  The k order inside a product is free, so a
// lane's operand is a contiguous run of the packed row and x is put into shared memory in that order.
//
// Work.  A CTA of 16 warps has an SM to itself, with its part of x in shared memory: all of K, or one of ks parts
// where x does not fit (or the tiles are few).  wk of its warps share a tile of 16 weight rows, and it walks over the
// tiles.  Each warp fetches its codes by TMA into a ring of its own that runs on across tiles (64 to 128 KB on an SM).
// Sums of the warps meet in shared memory, sums of CTAs in a workspace that a second kernel adds up, in a fixed order.
//
// Measured (device time; the fetches alone in brackets): 1 x 28672 x 8192 INT4 27.9 us (22.1), NVFP4 31.0 us (23.2) =
// 4.3 TB/s; 16 x 8192 x 28672 INT4 41.7 us; 1 x 4096 x 4096 INT4 4.8 us (3.4); 8 x 8192 x 8192 INT4 13.3 us (10.0).  What
// is left: 120 to 130 instructions per 2048 weights at half an instruction a cycle and scheduler (three to four warps
// each, every one waiting on its own chain of products), and 3 to 4 us before the first product (launch, x).
#include <math.h>

#include "umma.cuh"

namespace b200q {

constexpr int kW4Warps = 16, kW4Threads = 32 * kW4Warps;
constexpr int kW4Rows = 16;                  // weight rows of a tile
constexpr int kW4MaxParts = 16;              // CTAs that K may be cut over
constexpr int kSlab = 128;                   // k elements a warp handles at a time
// Slabs of a step and steps of the ring: four slabs make the bookkeeping of a step cheap; with more than 8 rows
// shared memory is needed for x and the products themselves take longer, so there two have to do.
template <int NT> struct W4Ring {
  static constexpr int kSlabs = NT == 1 ? 4 : 2, kStages = 2, kBytes = 1024 * kSlabs;
};
inline int w4_ring_bytes(int nt) { return nt == 1 ? W4Ring<1>::kStages * W4Ring<1>::kBytes : W4Ring<2>::kStages * W4Ring<2>::kBytes; }
constexpr uint32_t kW4WaitCode = 1u << 21;

struct W4Args {
  const void* x;
  int64_t x_stride;                          // elements
  const uint8_t* codes;                      // [n, k/2]
  const void* scales;                        // INT4: T [n, k/block]; NVFP4: E4M3 [n, k/block]
  const float* scale2;                       // NVFP4
  const void* bias;                          // T [n] or NULL
  void* out;                                 // [rows, n]
  int64_t out_stride;
  int rows, n, k, groups, group_slabs;       // groups a row; slabs a group (groups of 128 and more)
  int slabs_per_cta, tiles, wk, ks;
  FastDiv pairs;                             // slab pairs of a CTA
  int wide_scales;                           // a lane's scales of a step are one aligned word
  uint32_t* status;
  float* parts;                              // [ks][rows][n], ks > 1
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
// N words through the read-only path
template <int N>
__device__ __forceinline__ void w4_ldg_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 1) {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (N == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void w4_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
// one of the two 16-bit numbers of a word
template <typename T>
__device__ __forceinline__ float w4_half_word(uint32_t w, int high) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(high ? w & 0xffff0000u : w << 16);
  else return __half2float(__ushort_as_half(static_cast<uint16_t>(high ? w >> 16 : w)));
}

// 8 INT4 codes as fp16 patterns, one mask for two: a code in the low mantissa bits is the subnormal number
// code * 2^-24, four bits higher code * 2^-20.  Order (1, 5), (0, 4), (3, 7), (2, 6) of the elements.
__device__ __forceinline__ void int4x8_to_f16(uint32_t w, uint32_t* h) {
  const uint32_t w8 = w >> 8;
  h[0] = w & 0x000f000fu;
  h[1] = w & 0x00f000f0u;
  h[2] = w8 & 0x000f000fu;
  h[3] = w8 & 0x00f000f0u;
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
__device__ __forceinline__ uint32_t w4_hadd2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
enum { kFmtInt4 = 0, kFmtNvfp4 = 1, kFmtNvfp4x32 = 2 };   // x32: one E4M3 scale for 32 elements

// LW: words (of 8 codes) in a lane's contiguous run.  Lane qd of a quad holds the elements
//   slab * 128 + (i / LW) * 32 LW + qd * 8 LW + 8 (i % LW) + 0..7   for i = 0..3,
// so that an instruction's 16 elements always lie in one group of 32 LW (INT4 groups of 32, 64, 128 n).
template <int FMT, typename T, int NT, int LW>
__global__ void __launch_bounds__(kW4Threads, 1)
w4_linear_kernel(const __grid_constant__ CUtensorMap map, const W4Args a) {
  constexpr int kSegs = 4 / LW;                     // groups a slab has (at least)
  constexpr int kRunBytes = 4 * LW;
  constexpr int kPart = kW4Rows * 8 * NT;           // partial sums of a warp
  constexpr int kStep = W4Ring<NT>::kSlabs, kStages = W4Ring<NT>::kStages, kStageBytes = W4Ring<NT>::kBytes;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kScaled = kBf16 || FMT == kFmtInt4;       // x is multiplied by a power of two per row
  constexpr uint32_t kInf = kBf16 ? 0x7f80u : 0x7c00u;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint32_t xmax[8 * NT];
  __shared__ int not_finite, xbad[8 * NT];          // INT4: x (a row of it) holds an infinity or a NaN
  if (threadIdx.x < 8 * NT) xbad[threadIdx.x] = not_finite = 0;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, qd = lane & 3, gr = lane >> 2;
  const int ks = a.ks, wk = a.wk, wr = kW4Warps / wk;
  const int group = blockIdx.x / ks, groups = gridDim.x / ks, rank = blockIdx.x - group * ks;
  const int slab0 = rank * a.slabs_per_cta;
  const int slabs = max(min(a.slabs_per_cta, (a.k + kSlab - 1) / kSlab - slab0), 0);
  const int my_row = warp / wk, my_k = warp % wk;   // which of the CTA's tiles, which part of its slabs

  uint8_t* ring = smem + warp * kStages * kStageBytes;      // NVFP4: [stages][16 rows][128 B]; INT4: [stages][2 slabs][16 rows][64 B]
  uint8_t* xs = smem + kW4Warps * kStages * kStageBytes; // [slab][row][i][qd] 16 B
  float* xsum = reinterpret_cast<float*>(xs + static_cast<int64_t>(a.pairs.d) * 2 * kSlab * 2 * a.rows);   // [slab][group][8 NT], INT4
  float* part = xsum + (FMT == kFmtInt4 ? static_cast<int>(a.pairs.d) * 2 * kSegs * 8 * NT : 0);           // [warps][8 NT][16], wk > 1
  __shared__ __align__(8) uint64_t all_bars[kW4Warps * kStages];
  __shared__ uint32_t abort_flag;
  uint64_t* bars = all_bars + warp * kStages;
  if (lane < kStages) mbar_init(&bars[lane], 1);
  if (threadIdx.x == 0) abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  pdl_prologue();

  // tiles of round t: (t * wr + my_row) * groups + group, so that the last round is spread over the SMs
  const int nsteps = (slabs + kStep - 1) / kStep;
  const int mine = nsteps > my_k ? (nsteps - my_k + wk - 1) / wk : 0;             // steps of this warp in each tile
  const int first_tile = my_row * groups + group, tile_step = wr * groups;
  const int rounds = (a.tiles - group + tile_step - 1) / tile_step;               // of the CTA
  const int my_tiles = a.tiles > first_tile ? (a.tiles - first_tile + tile_step - 1) / tile_step : 0;
  const int steps = mine * my_tiles;

  // ---- producer: one lane asks for a step's slabs of one tile (rows behind n and elements behind k arrive as zeros) ----
  const int slab_first = slab0 + kStep * my_k;
  int p_tile = first_tile, p_i = 0, p_left = steps, p_x = 0;
  auto produce = [&](uint32_t slot) {
    if (p_left > 0) {
      if (p_i == 0) p_x = slab_first * (kSlab / 2);
      if (lane == 0) {
        uint64_t* bar = reinterpret_cast<uint64_t*>(bars + slot / kStageBytes);
        mbar_expect_tx(bar, kStageBytes);
        constexpr int kBox = FMT == kFmtInt4 ? 1 : 2;                              // slabs a copy brings
#pragma unroll
        for (int j = 0; j < kStep; j += kBox)
          tma_load_2d(ring + slot + 1024 * j, &map, bar, p_x + j * (kSlab / 2), p_tile * kW4Rows);
      }
      p_x += wk * kStep * (kSlab / 2);
      if (++p_i == mine) { p_i = 0; p_tile += tile_step; }
      --p_left;
    }
  };
#pragma unroll 1
  for (int s = 0; s < kStages; ++s) produce(s * kStageBytes);

  // ---- scales, one step ahead of their use ----
  // INT4: 2 kSegs scales of a row in two slabs.  NVFP4: the four E4M3 of the lane's 64 elements.
  constexpr int kPairs = kStep / 2;
  constexpr int kScaleWords = kPairs * (FMT == kFmtInt4 ? kSegs : 1);             // of 32 bits
  uint32_t nxt[2][kScaleWords];
  const uint8_t* ps[2] = {nullptr, nullptr};        // the rows' scales
  int s_tile = first_tile, s_i = 0, s_left = steps, s_at = 0;
  auto load_scales = [&]() {
    if (s_left > 0) {
      if (s_i == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          ps[r] = static_cast<const uint8_t*>(a.scales) +
                  static_cast<int64_t>(min(s_tile * kW4Rows + gr + 8 * r, a.n - 1)) * a.groups * (FMT == kFmtInt4 ? 2 : 1);
        s_at = FMT == kFmtInt4 ? slab_first * kSegs : FMT == kFmtNvfp4 ? slab_first * (kSlab / 16) + 4 * qd : slab_first * (kSlab / 32) + 2 * qd;
        s_tile += tile_step;
      }
      if constexpr (FMT == kFmtInt4) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (a.wide_scales) {                      // whole steps, aligned
            w4_ldg_words<kScaleWords>(ps[r] + s_at * 2, nxt[r]);
          } else {
#pragma unroll
            for (int w = 0; w < kScaleWords; ++w) {
              uint32_t u[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                int at = s_at + 2 * w + h;
                if (LW == 4) at /= a.group_slabs;
                at = min(at, a.groups - 1);         // behind the end of a row x is zero
                u[h] = __ldg(reinterpret_cast<const uint16_t*>(ps[r]) + at);
              }
              nxt[r][w] = u[0] | (u[1] << 16);
            }
          }
        }
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int w = 0; w < kPairs; ++w) {
            const int at = s_at + (FMT == kFmtNvfp4 ? 16 : 8) * w;
            nxt[r][w] = 0;
            if constexpr (FMT == kFmtNvfp4x32) {    // the scales of the lane's two runs of 32
              if (at < a.groups) nxt[r][w] = __ldg(ps[r] + at);
              if (at + 1 < a.groups) nxt[r][w] |= static_cast<uint32_t>(__ldg(ps[r] + at + 1)) << 8;
            } else if (a.wide_scales) {
              if (at < a.groups) nxt[r][w] = __ldg(reinterpret_cast<const uint32_t*>(ps[r] + at));
            } else {
              if (at < a.groups) nxt[r][w] = __ldg(reinterpret_cast<const uint16_t*>(ps[r] + at));
              if (at + 2 < a.groups) nxt[r][w] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(ps[r] + at + 2))) << 16;
            }
          }
        }
      }
      s_at += FMT == kFmtInt4 ? kStep * wk * kSegs : kStep * wk * (kSlab / (FMT == kFmtNvfp4 ? 16 : 32));
      if (++s_i == mine) s_i = 0;
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
  const int x_k = slab0 * kSlab + (FMT == kFmtInt4 ? (lane >> 4) * kSlab + ((x_i / LW) * 4 * LW + x_q * LW + x_i % LW) * 8
                                                   : (2 * x_q + (lane >> 4)) * 32 + x_i * 8);
  auto load_x = [&](int u) {
    uint32_t row, pair;
    a.pairs.divmod(u, row, pair);
    const int k = x_k + pair * (2 * kSlab);
    return k < a.k ? __ldg(reinterpret_cast<const uint4*>(x + row * a.x_stride + k)) : make_uint4(0, 0, 0, 0);
  };
  auto max_x = [&](int u, const uint4& v) {
    uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    m = max(m & 0xffffu, m >> 16);
    if (m >= kInf) {                                // infinity or NaN: the largest of the others
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      m = 0;
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = w[j] & 0x7fffu, hi = (w[j] >> 16) & 0x7fffu;
        m = max(m, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
      }
    }
    m = warp_max_u32(m);
    if (lane == 0 && m) atomicMax(&xmax[a.pairs.div(u)], m);
  };
  // log2 of the power: from the biased exponent, kept where the power and its inverse are normal numbers
  auto row_shift = [&](uint32_t top) {
    return kBf16 ? 14 + 127 - max(static_cast<int>(top >> 7), 28) : max(14 + 15 - max(static_cast<int>(top >> 10), 1), 0);
  };
  auto store_x = [&](int u, const uint4& v) {
    uint32_t row, pair;
    a.pairs.divmod(u, row, pair);
    const int slab = 2 * pair + (lane >> 4);
    uint32_t h[4] = {v.x, v.y, v.z, v.w};
    if constexpr (kScaled) {
      const float up = __uint_as_float(static_cast<uint32_t>(127 + row_shift(xmax[row])) << 23);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = w4_pack_f16(w4_half_word<T>(h[j], 0) * up, w4_half_word<T>(h[j], 1) * up);
    }
    uint4 o;
    if constexpr (FMT == kFmtInt4) {
      // the group's sum, for the 8 in code - 8; elements 0, 4, 2, 6 meet codes that are 16 times too large
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        sum += t.x + t.y;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if constexpr (LW >= 2) sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      if constexpr (LW == 4) sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      if (!(fabsf(sum) < INFINITY)) not_finite = xbad[row] = 1;
      if (x_q == 0 && x_i % LW == 0) xsum[(slab * kSegs + x_i / LW) * 8 * NT + row] = sum * -4.76837158203125e-7f;   // -8 * 2^-24
      o.x = __byte_perm(h[0], h[2], 0x7632);        // (1, 5), (0, 4), (3, 7), (2, 6)
      o.y = w4_hmul2(__byte_perm(h[0], h[2], 0x5410), 0x2c002c00u);               // / 16
      o.z = __byte_perm(h[1], h[3], 0x7632);
      o.w = w4_hmul2(__byte_perm(h[1], h[3], 0x5410), 0x2c002c00u);
    } else {
      o = make_uint4(h[0], h[1], h[2], h[3]);
    }
    // [slab][row][word][q]; odd rows swap words 0, 1 and 2, 3, so that eight lanes of a load hit all banks
    *reinterpret_cast<uint4*>(xs + (((slab * a.rows + static_cast<int>(row)) * 4 + (x_i ^ (row & 1))) * 4 + x_q) * 16) = o;
  };
  uint4 hold[kHold];
#pragma unroll
  for (int j = 0; j < kHold; ++j) {
    if (warp + j * kW4Warps >= units) break;
    hold[j] = load_x(warp + j * kW4Warps);
  }
  if constexpr (kScaled) {
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
  __syncthreads();

  float back[NT][2];                                // of the columns this thread's sums belong to
  const float s2 = FMT != kFmtInt4 ? __ldg(a.scale2) : 16777216.f;                // 2^24 of the codes as subnormals
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * qd + j;
      back[n][j] = 1.f;
      if constexpr (kScaled)
        if (row < a.rows) back[n][j] = __uint_as_float(static_cast<uint32_t>(127 - row_shift(xmax[row])) << 23);
    }

  auto store = [&](int row, int col, float sum) {
    if (col >= a.n) return;
    if (ks > 1) {                                   // the other parts of K are other CTAs': w4_join_kernel adds them up
      a.parts[(static_cast<int64_t>(rank) * a.rows + row) * a.n + col] = sum;
      return;
    }
    if (a.bias) sum += Elem<T>::to_float(static_cast<const T*>(a.bias)[col]);
    static_cast<T*>(a.out)[row * a.out_stride + col] = Elem<T>::from_float(sum);
  };

  uint32_t slot = 0, phase = 0;                     // ring offset of the step at hand, parity of its barrier
  const float* lane_sum = xsum + 2 * qd;
  // x of row 8 n + gr; columns beyond the last row repeat it, their sums are dropped
  const uint8_t* lane_x[NT];
  int odd[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = min(8 * n + gr, a.rows - 1);
    odd[n] = (row & 1) * 64;
    lane_x[n] = xs + (kStep * my_k * a.rows + row) * 256 + qd * 16;
  }
  const int slab_step = a.rows * 256, pair_step = kStep * wk * slab_step;
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    const int tile = first_tile + round * tile_step;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const int todo = tile < a.tiles ? mine : 0;
    // signed_too: rows of x that are not finite have the 8 taken off every code instead of off the sum, so that infinity
    // times (code - 8) keeps its sign; the other rows' arithmetic stays what it is without them
    auto products = [&](auto signed_too) {
#pragma unroll 1
    for (int it = 0, x_at = 0; it < todo; ++it, x_at += pair_step) {
      uint32_t cur[2][kScaleWords];
#pragma unroll
      for (int w = 0; w < kScaleWords; ++w) { cur[0][w] = nxt[0][w]; cur[1][w] = nxt[1][w]; }
      load_scales();
      if (!mbar_wait_bounded(reinterpret_cast<uint64_t*>(bars + slot / kStageBytes), phase, &abort_flag, a.status, kW4WaitCode)) p_left = 0;
#pragma unroll
      for (int j4 = 0; j4 < kStep; ++j4) {          // behind the end of K x is zero
        const int half = j4 & 1;
        uint32_t wa[4], wb[4];
        if constexpr (FMT != kFmtInt4) {            // 128-byte rows, 16-byte pieces swizzled by the row
          const uint8_t* p = ring + slot + (j4 / 2) * 2048 + gr * 128 + (((2 * qd + half) ^ gr) << 4);
          const uint4 va = *reinterpret_cast<const uint4*>(p), vb = *reinterpret_cast<const uint4*>(p + 1024);
          wa[0] = va.x; wa[1] = va.y; wa[2] = va.z; wa[3] = va.w;
          wb[0] = vb.x; wb[1] = vb.y; wb[2] = vb.z; wb[3] = vb.w;
        } else {                                    // 64-byte rows of either slab
          const uint8_t* p = ring + slot + j4 * 1024 + gr * 64 + qd * kRunBytes;
#pragma unroll
          for (int seg = 0; seg < kSegs; ++seg) {
            w4_words<LW>(p + seg * 4 * kRunBytes, wa + seg * LW);
            w4_words<LW>(p + seg * 4 * kRunBytes + 512, wb + seg * LW);
          }
        }
        uint32_t sc[2][2];
        if constexpr (FMT != kFmtInt4) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t h;
            const uint32_t two = FMT == kFmtNvfp4 ? cur[r][j4 / 2] >> (16 * half) : cur[r][j4 / 2];
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
            sc[r][0] = __byte_perm(h, h, FMT == kFmtNvfp4 || half == 0 ? 0x1010 : 0x3232);
            sc[r][1] = __byte_perm(h, h, FMT == kFmtNvfp4 || half == 1 ? 0x3232 : 0x1010);
          }
        }
        float tmp[NT][4], stmp[NT][4];
        const uint8_t *xe[NT], *xo[NT];             // words 0, 2 and 1, 3
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint8_t* p = lane_x[n] + x_at + j4 * slab_step;
          xe[n] = p + odd[n];
          xo[n] = p + 64 - odd[n];
        }
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
            const uint4 b = *reinterpret_cast<const uint4*>((i & 1 ? xo[n] : xe[n]) + (i & 2) * 64);
            if constexpr (FMT == kFmtInt4) {
              if (i % LW == 0) {                    // from -8 times the sum of the group's x, in the codes' 2^-24
                const float2 xg = *reinterpret_cast<const float2*>(lane_sum + (kStep * (my_k + it * wk) * kSegs + j4 * kSegs + i / LW) * 8 * NT + 8 * n);
                tmp[n][0] = tmp[n][2] = xg.x;
                tmp[n][1] = tmp[n][3] = xg.y;
              }
              w4_mma(tmp[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
              w4_mma(tmp[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
              if constexpr (decltype(signed_too)::value) {
                uint32_t ga[4], gb[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {       // -8 at either scale
                  ga[j] = w4_hadd2(fa[j], j & 1 ? 0x80808080u : 0x80088008u);
                  gb[j] = w4_hadd2(fb[j], j & 1 ? 0x80808080u : 0x80088008u);
                }
                if (i % LW == 0) stmp[n][0] = stmp[n][1] = stmp[n][2] = stmp[n][3] = 0.f;
                w4_mma(stmp[n], ga[0], gb[0], ga[1], gb[1], b.x, b.y);
                w4_mma(stmp[n], ga[2], gb[2], ga[3], gb[3], b.z, b.w);
              }
              if (i % LW == LW - 1) {
                const int seg = j4 * kSegs + i / LW;
                const float i0 = rcp_approx(w4_half_word<T>(cur[0][seg / 2], seg & 1)), i1 = rcp_approx(w4_half_word<T>(cur[1][seg / 2], seg & 1));
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  v[j] = tmp[n][j];
                  if constexpr (decltype(signed_too)::value)
                    if (xbad[8 * n + 2 * qd + (j & 1)]) v[j] = stmp[n][j];
                }
                acc[n][0] += v[0] * i0; acc[n][1] += v[1] * i0;
                acc[n][2] += v[2] * i1; acc[n][3] += v[3] * i1;
              }
            } else {
              w4_mma(acc[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
              w4_mma(acc[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
            }
          }
        }
      }
      __syncwarp();                                 // the slot has been read by every lane
      produce(slot);
      slot += kStageBytes;
      if (slot == kStages * kStageBytes) { slot = 0; phase ^= 1; }
    }
    };
    if (FMT == kFmtInt4 && not_finite) products(std::true_type());
    else products(std::false_type());
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[n][j] = acc[n][j] * s2 * back[n][j & 1];

    // ---- sums of the warps' parts of K, always in their order ----
    if (wk > 1) {
      const int elems = kW4Rows * a.rows;           // of a tile
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
        store(in / kW4Rows, (group + round * tile_step + t * groups) * kW4Rows + in % kW4Rows, sum);
      }
      if (round + 1 < rounds) __syncthreads();      // read before the next round writes
    } else if (tile < a.tiles) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 8 * n + 2 * qd + (j & 1);
          if (row < a.rows) store(row, tile * kW4Rows + gr + 8 * (j >> 1), acc[n][j]);
        }
    }
  }
  grace_after_abort(&abort_flag);
}

// Sums of the CTAs' parts of K, in their order, plus the bias.
template <typename T>
__global__ void __launch_bounds__(256) w4_join_kernel(const W4Args a) {
  pdl_prologue();
  const int64_t total = static_cast<int64_t>(a.rows) * a.n, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int row = static_cast<int>(i / a.n), col = static_cast<int>(i - static_cast<int64_t>(row) * a.n);
  float sum = 0.f;
#pragma unroll 4
  for (int p = 0; p < a.ks; ++p) sum += a.parts[p * total + i];
  if (a.bias) sum += Elem<T>::to_float(static_cast<const T*>(a.bias)[col]);
  static_cast<T*>(a.out)[row * a.out_stride + col] = Elem<T>::from_float(sum);
}

// segs: INT4 groups a slab (0: NVFP4)
inline size_t w4_smem(int rows, int nt, int slabs, int segs, int wk) {
  const int step = nt == 1 ? W4Ring<1>::kSlabs : W4Ring<2>::kSlabs;
  slabs = (slabs + step - 1) / step * step;
  return kW4Warps * static_cast<size_t>(w4_ring_bytes(nt)) + static_cast<size_t>(slabs) * (kSlab * 2 * rows + 32 * segs * nt) +
         (wk > 1 ? kW4Warps * kW4Rows * 8 * 4 * static_cast<size_t>(nt) : 0);
}
constexpr size_t kW4SmemLimit = 227 * 1024 - 1024;
inline int w4_nt(int rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

// How K is cut, over the wk warps of a tile and over ks CTAs: the least of an estimate in steps of a fully loaded SM.
// A round takes a warp's steps in it; one that leaves warps idle is shorter, but not below what a warp needs by itself
// (0.6); a round that joins warps pays for its barriers, several CTAs for a launch that adds their sums, and with more
// than 8 rows a CTA for putting its part of x into shared memory.  Measured with other choices forced: 16 x 4096 x 4096
// NVFP4 9.3 us in parts against 11.2 whole, 16 x 8192 x 28672 INT4 41.7 us in 14 parts against 43.6 in 8, 8 x 8192 x 8192
// INT4 13.2 in 2 parts against 14.9 in more, 1 x 28672 x 8192 NVFP4 31.0 with wk = 1 against 32.2 (4) and 35.7 (16).
inline bool w4_cut(int rows, int slabs, int segs, int tiles, int sms, int& wk, int& ks) {
  // A decoding loop asks for the same few shapes again and again, and the search costs as much as a launch.
  struct Entry { int rows, slabs, segs, tiles, sms, wk, ks; };
  static thread_local Entry seen[64];
  const uint32_t hash = (rows * 2654435761u) ^ (slabs * 2246822519u) ^ (tiles * 3266489917u) ^ (segs * 668265263u);
  Entry& e = seen[(hash >> 16) & 63];
  if (e.rows == rows && e.slabs == slabs && e.segs == segs && e.tiles == tiles && e.sms == sms) {
    wk = e.wk;
    ks = e.ks;
    return ks > 0;
  }
  const int nt = w4_nt(rows), step = nt == 1 ? W4Ring<1>::kSlabs : W4Ring<2>::kSlabs;
  const double join = nt == 2 ? 1.6 : nt == 4 ? 1.0 : 2.0, fill = nt == 2 ? 0.4 : nt == 4 ? 0.25 : 0.0;
  double best = 1e30;
  for (int c = 1; c <= kW4MaxParts && c <= slabs; ++c) {
    const int part = ((slabs + c - 1) / c + step - 1) / step * step, steps = part / step;
    if (c > 1 && part * (c - 1) >= slabs) continue; // nothing left for the last part
    for (int w = 1; w <= kW4Warps && (w == 1 || w <= steps); w *= 2) {
      if (w4_smem(rows, nt, part, segs, w) > kW4SmemLimit) continue;
      const double load = static_cast<double>(tiles) * w / (static_cast<double>(sms / c) * kW4Warps);
      const double whole = floor(load), rest = load - whole;
      const double mine = (steps + w - 1) / w;
      const double cost = mine * (whole + (rest > 0 ? (rest > 0.6 ? rest : 0.6) : 0)) + ceil(load) * (w > 1 ? 0.15 : 0) +
                          (c > 1 ? join : 0) + fill * ((rows * part / 2 + kW4Warps - 1) / kW4Warps);
      if (cost < best) { best = cost; wk = w; ks = c; }
    }
  }
  e = Entry{rows, slabs, segs, tiles, sms, wk, best < 1e30 ? ks : 0};
  return best < 1e30;
}

inline int64_t w4_parts_bytes(int ks, int rows, int64_t n) { return static_cast<int64_t>(ks) * rows * n * 4; }

template <int FMT, typename T, int NT, int LW>
int launch_w4(W4Args a, int64_t parts_bytes, cudaStream_t s) {
  auto kern = w4_linear_kernel<FMT, T, NT, LW>;
  constexpr int kStep = W4Ring<NT>::kSlabs, kGroups = FMT == kFmtInt4 ? 4 / LW : 0;
  const int slabs = (a.k + kSlab - 1) / kSlab, sms = sm_count_cached();
  static std::atomic<uint64_t> done;
  if (!allow_smem(reinterpret_cast<const void*>(kern), kW4SmemLimit, done)) return B200Q_ERR_CUDA;
  if (!w4_cut(a.rows, slabs, kGroups, a.tiles, sms, a.wk, a.ks)) return B200Q_ERR_CAPACITY;
  if (a.ks > 1 && (!a.parts || parts_bytes < w4_parts_bytes(a.ks, a.rows, a.n))) return B200Q_ERR_CAPACITY;
  a.slabs_per_cta = ((slabs + a.ks - 1) / a.ks + kStep - 1) / kStep * kStep;
  a.pairs = FastDiv(a.slabs_per_cta / 2);
  const size_t smem = w4_smem(a.rows, NT, a.slabs_per_cta, kGroups, a.wk);
  const int unit = FMT == kFmtInt4 ? W4Ring<NT>::kSlabs * 4 / LW : 4, bytes = FMT == kFmtInt4 ? 2 : 1;   // scales a lane takes at a time
  a.wide_scales = (FMT != kFmtInt4 || LW < 4 || a.group_slabs == 1) && a.groups % unit == 0 &&
                  reinterpret_cast<uintptr_t>(a.scales) % min(unit * bytes, 16) == 0;
  CUtensorMap map;
  const EncodeTiledFn encode = encode_tiled_fn();
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.k) / 2, static_cast<cuuint64_t>(a.n)}, strides[1] = {static_cast<cuuint64_t>(a.k) / 2};
  const cuuint32_t box[2] = {FMT == kFmtInt4 ? 64u : 128u, kW4Rows}, ones[2] = {1, 1};
  if (!encode || encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(a.codes), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, FMT == kFmtInt4 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return B200Q_ERR_CUDA;
  const int groups = max(1, min(a.tiles, sms / a.ks));
  launch_pdl(kern, groups * a.ks, kW4Threads, smem, s, map, a);
  if (a.ks > 1)
    launch_pdl(w4_join_kernel<T>, static_cast<unsigned>((static_cast<int64_t>(a.rows) * a.n + 255) / 256), 256, 0, s, a);
  return launch_status();
}

template <int FMT, int LW>
int dispatch_w4(const W4Args& a, int dtype, int64_t parts_bytes, cudaStream_t s) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (a.rows <= 8) return launch_w4<FMT, T, 1, LW>(a, parts_bytes, s);
    if (a.rows <= 16) return launch_w4<FMT, T, 2, LW>(a, parts_bytes, s);
    return launch_w4<FMT, T, 4, LW>(a, parts_bytes, s);
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
                      const void* bias, void* out, int64_t out_stride, int rows, int64_t n, int64_t k, int block, void* workspace, uint32_t* status) {
  W4Args a{};
  a.status = status;
  a.parts = static_cast<float*>(workspace);
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
    if (w4_smem(rows, w4_nt(rows), (slabs + kW4MaxParts - 1) / kW4MaxParts, 4, 1) <= kW4SmemLimit) return rows;
  return 0;
}

extern "C" int64_t b200q_w4_linear_workspace(int rows, int64_t n, int64_t k, int int4_block) {
  if (rows <= 0 || rows > 32 || n <= 0 || n > (1 << 30) || k <= 0 || k % 32 || k > (1 << 24) || int4_block < 0) return B200Q_ERR_SHAPE;
  int wk = 1, ks = 1;
  const int groups = int4_block == 0 ? 0 : int4_block == 32 ? 4 : int4_block == 64 ? 2 : 1;
  if (!w4_cut(rows, static_cast<int>((k + kSlab - 1) / kSlab), groups, static_cast<int>((n + kW4Rows - 1) / kW4Rows), sm_count_cached(), wk, ks))
    return B200Q_ERR_CAPACITY;
  return ks > 1 ? w4_parts_bytes(ks, rows, n) : 0;
}

extern "C" int b200q_int4_linear(const void* x, int64_t x_stride, int dtype, const uint8_t* codes, const void* scales, int block,
                                 const void* bias, void* out, int64_t out_stride, int rows, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes,
                                 uint32_t* status_io, void* stream) {
  B200Q_REQUIRE_PTR(status_io);
  if (const int r = w4_check(x, x_stride, dtype, codes, scales, out, out_stride, rows, n, k)) return r;
  if (block <= 0 || k % block) return B200Q_ERR_SHAPE;
  if (block != 32 && block != 64 && block % kSlab) return B200Q_ERR_UNSUPPORTED;
  const W4Args a = w4_args(x, x_stride, codes, scales, nullptr, bias, out, out_stride, rows, n, k, block, workspace, status_io);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (block == 32) return dispatch_w4<kFmtInt4, 1>(a, dtype, workspace_bytes, s);
  if (block == 64) return dispatch_w4<kFmtInt4, 2>(a, dtype, workspace_bytes, s);
  return dispatch_w4<kFmtInt4, 4>(a, dtype, workspace_bytes, s);
}

extern "C" int b200q_nvfp4_linear(const void* x, int64_t x_stride, int dtype, const uint8_t* codes, const uint8_t* scales, int block,
                                  const float* scale2, const void* bias, void* out, int64_t out_stride, int rows, int64_t n,
                                  int64_t k, void* workspace, int64_t workspace_bytes,
                                 uint32_t* status_io, void* stream) {
  B200Q_REQUIRE_PTR(status_io);
  if (const int r = w4_check(x, x_stride, dtype, codes, scales, out, out_stride, rows, n, k)) return r;
  B200Q_REQUIRE_PTR(scale2);
  if (block != 16 && block != 32) return B200Q_ERR_UNSUPPORTED;
  const W4Args a = w4_args(x, x_stride, codes, scales, scale2, bias, out, out_stride, rows, n, k, block, workspace, status_io);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return block == 16 ? dispatch_w4<kFmtNvfp4, 4>(a, dtype, workspace_bytes, s) : dispatch_w4<kFmtNvfp4x32, 4>(a, dtype, workspace_bytes, s);
}
