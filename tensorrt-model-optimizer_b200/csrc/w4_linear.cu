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
#include "umma.cuh"

namespace b200q {

constexpr int kW4Warps = 8, kW4Threads = 32 * kW4Warps;
constexpr int kW4Rows = 16;                  // weight rows of a tile
constexpr int kSlab = 128;                   // k elements a warp handles at a time
constexpr int kW4Stages = 6;

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
  int slabs_per_cta, tiles;
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
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float r;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r) : "r"(addr) : "memory");
  return r;
}

enum { kFmtInt4 = 0, kFmtNvfp4 = 1 };

// LW: words (of 8 codes) in a lane's contiguous run.  Lane qd of a quad holds the elements
//   slab * 128 + (i / LW) * 32 LW + qd * 8 LW + 8 (i % LW) + 0..7   for i = 0..3,
// so that an instruction's 16 elements always lie in one group of 32 LW (INT4 groups of 32, 64, 128 n).
template <int FMT, typename T, int NT, int LW>
__global__ void __launch_bounds__(kW4Threads, 2)
w4_linear_kernel(const W4Args a) {
  constexpr int kSegs = 4 / LW;                     // groups a slab has (at least)
  constexpr int kRunBytes = 4 * LW;
  constexpr int kPart = kW4Rows * 8 * NT;           // partial sums of a warp
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t xmax[8 * NT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, qd = lane & 3, gr = lane >> 2;
  uint32_t ks = 1, rank = 0;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ks));
  rank = cluster_ctarank();
  const int cluster = blockIdx.x / ks, nclusters = gridDim.x / ks;
  const int slab0 = rank * a.slabs_per_cta;
  const int slabs = max(min(a.slabs_per_cta, (a.k + kSlab - 1) / kSlab - slab0), 0);

  float* part = reinterpret_cast<float*>(smem);                                   // [2][warps][16][8 NT]
  uint8_t* ring = smem + 2 * kW4Warps * kPart * 4 + warp * kW4Stages * 1024;      // [stages][2][32 lanes][16 B]
  uint8_t* xs = smem + 2 * kW4Warps * kPart * 4 + kW4Warps * kW4Stages * 1024;    // [slab][i][qd][row] 16 B
  const uint32_t ring_addr = smem_u32(ring) + lane * 16;

  pdl_prologue();

  // ---- producer: this lane's operands of one slab of one tile ----
  const int mine = slabs > warp ? (slabs - warp + kW4Warps - 1) / kW4Warps : 0;   // slabs of this warp in each tile
  const int my_tiles = a.tiles > cluster ? (a.tiles - cluster + nclusters - 1) / nclusters : 0;
  const int64_t row_bytes = a.k / 2;
  int p_tile = cluster, p_i = 0, p_stage = 0;
  int p_left = mine * my_tiles;
  auto produce = [&]() {
    if (p_left > 0) {
      const int slab = slab0 + warp + p_i * kW4Warps;
      const int r0 = min(p_tile * kW4Rows + gr, a.n - 1), r1 = min(p_tile * kW4Rows + gr + 8, a.n - 1);
#pragma unroll
      for (int seg = 0; seg < kSegs; ++seg) {
        const int kk = slab * kSlab + seg * 32 * LW + qd * 8 * LW;
        if (kk < a.k) {
          const uint32_t dst = ring_addr + p_stage * 1024 + seg * kRunBytes;
          copy_async<kRunBytes>(dst, a.codes + r0 * row_bytes + kk / 2);
          copy_async<kRunBytes>(dst + 512, a.codes + r1 * row_bytes + kk / 2);
        }
      }
      --p_left;
      if (++p_i == mine) { p_i = 0; p_tile += nclusters; }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    p_stage = p_stage + 1 == kW4Stages ? 0 : p_stage + 1;
  };
#pragma unroll 1
  for (int s = 0; s < kW4Stages - 1; ++s) produce();

  // ---- x into shared memory, as fp16 times a power of two ----
  const int packs = slabs * (kSlab / 8);            // 16-byte units a row
  const T* x = static_cast<const T*>(a.x);
  const int k0 = slab0 * kSlab;
  auto load_x = [&](int row, int p) {
    return k0 + 8 * p < a.k ? *reinterpret_cast<const uint4*>(x + row * a.x_stride + k0 + 8 * p) : make_uint4(0, 0, 0, 0);
  };
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if (threadIdx.x < 8 * NT) xmax[threadIdx.x] = 0;
    __syncthreads();
    for (int row = 0; row < a.rows; ++row) {
      uint32_t top = 0;                             // largest finite |x|, as a bf16 pattern
#pragma unroll 4
      for (int p = threadIdx.x; p < packs; p += kW4Threads) {
        const uint4 v = load_x(row, p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lo = w[j] & 0x7fffu, hi = (w[j] >> 16) & 0x7fffu;
          top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
      }
      top = warp_max_u32(top);
      if (lane == 0 && top) atomicMax(&xmax[row], top);
    }
    __syncthreads();
  }
  for (int row = 0; row < a.rows; ++row) {
    float up = 1.f;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - max(static_cast<int>(xmax[row] >> 7), 28)) << 23);
#pragma unroll 4
    for (int p = threadIdx.x; p < packs; p += kW4Threads) {
      const uint4 v = load_x(row, p);
      uint32_t h[4] = {v.x, v.y, v.z, v.w};
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = w4_pack_f16(__uint_as_float(h[j] << 16) * up, __uint_as_float(h[j] & 0xffff0000u) * up);
      }
      uint4 o;
      if constexpr (FMT == kFmtInt4) {              // (1, 5), (0, 4), (3, 7), (2, 6)
        o.x = __byte_perm(h[0], h[2], 0x7632);
        o.y = __byte_perm(h[0], h[2], 0x5410);
        o.z = __byte_perm(h[1], h[3], 0x7632);
        o.w = __byte_perm(h[1], h[3], 0x5410);
      } else {
        o = make_uint4(h[0], h[1], h[2], h[3]);
      }
      const int slab = p / 16, r = p % 16;          // unit r of the slab is word i of lane q
      const int seg = r / (4 * LW), q = (r % (4 * LW)) / LW, i = seg * LW + r % LW;
      *reinterpret_cast<uint4*>(xs + ((static_cast<int64_t>((slab * 4 + i) * 4 + q)) * a.rows + row) * 16) = o;
    }
  }
  __syncthreads();

  float back[NT][2];                                // of the columns this thread's sums belong to
  const float s2 = FMT == kFmtNvfp4 ? __ldg(a.scale2) : 1.f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * n + 2 * qd + j;
      back[n][j] = 1.f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        if (row < a.rows) back[n][j] = __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(xmax[row] >> 7), 28) - 14) << 23);
    }

  int stage = 0, buf = 0;
  for (int tile = cluster; tile < a.tiles; tile += nclusters) {
    const int r0 = min(tile * kW4Rows + gr, a.n - 1), r1 = min(tile * kW4Rows + gr + 8, a.n - 1);
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 1
    for (int it = 0; it < mine; ++it) {
      const int sl = warp + it * kW4Warps, slab = slab0 + sl;
      // scales of this slab (the codes are in flight or here already)
      float inv[2][kSegs];
      uint32_t sc[2][2];
      if constexpr (FMT == kFmtInt4) {
#pragma unroll
        for (int seg = 0; seg < kSegs; ++seg) {
          const int kk = slab * kSlab + seg * 32 * LW;
          const int grp = LW == 4 ? slab / a.group_slabs : kk / (32 * LW);
          const bool ok = kk < a.k;
          const T* s = static_cast<const T*>(a.scales) + (ok ? grp : 0);
          inv[0][seg] = ok ? Elem<T>::to_float(__ldg(s + static_cast<int64_t>(r0) * a.groups)) : INFINITY;
          inv[1][seg] = ok ? Elem<T>::to_float(__ldg(s + static_cast<int64_t>(r1) * a.groups)) : INFINITY;
        }
      } else {
        const int kk = slab * kSlab + 32 * qd;
        const uint8_t* s = static_cast<const uint8_t*>(a.scales) + kk / 16;
        const uint32_t u0 = kk < a.k ? __ldg(reinterpret_cast<const uint16_t*>(s + static_cast<int64_t>(r0) * a.groups)) : 0;
        const uint32_t u1 = kk < a.k ? __ldg(reinterpret_cast<const uint16_t*>(s + static_cast<int64_t>(r1) * a.groups)) : 0;
        uint32_t h0, h1;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"(static_cast<uint16_t>(u0)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"(static_cast<uint16_t>(u1)));
        sc[0][0] = __byte_perm(h0, h0, 0x1010); sc[0][1] = __byte_perm(h0, h0, 0x3232);
        sc[1][0] = __byte_perm(h1, h1, 0x1010); sc[1][1] = __byte_perm(h1, h1, 0x3232);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kW4Stages - 2) : "memory");
      const uint4 va = *reinterpret_cast<const uint4*>(ring + stage * 1024 + lane * 16);
      const uint4 vb = *reinterpret_cast<const uint4*>(ring + stage * 1024 + 512 + lane * 16);
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
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
          uint4 b = make_uint4(0, 0, 0, 0);
          const int row = 8 * n + gr;
          if (row < a.rows) b = *reinterpret_cast<const uint4*>(xs + (static_cast<int64_t>((sl * 4 + i) * 4 + qd) * a.rows + row) * 16);
          if constexpr (FMT == kFmtInt4) {
            if (i % LW == 0) tmp[n][0] = tmp[n][1] = tmp[n][2] = tmp[n][3] = 0.f;
            w4_mma(tmp[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
            w4_mma(tmp[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
            if (i % LW == LW - 1) {
              const float i0 = rcp_approx(inv[0][i / LW]), i1 = rcp_approx(inv[1][i / LW]);
              acc[n][0] += tmp[n][0] * i0; acc[n][1] += tmp[n][1] * i0;
              acc[n][2] += tmp[n][2] * i1; acc[n][3] += tmp[n][3] * i1;
            }
          } else {
            w4_mma(acc[n], fa[0], fb[0], fa[1], fb[1], b.x, b.y);
            w4_mma(acc[n], fa[2], fb[2], fa[3], fb[3], b.z, b.w);
          }
        }
      }
      produce();                                    // into the slot read one slab ago
      stage = stage + 1 == kW4Stages ? 0 : stage + 1;
    }
    // ---- partial sums of the warps and CTAs ----
    float* mypart = part + (buf * kW4Warps + warp) * kPart;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        mypart[(gr + 8 * (j >> 1)) + kW4Rows * (8 * n + 2 * qd + (j & 1))] = acc[n][j] * (back[n][j & 1] * s2);
    if (ks > 1) cluster_barrier(); else __syncthreads();
    const int todo = kW4Rows * a.rows;
    for (int e = rank * kW4Threads + threadIdx.x; e < todo; e += ks * kW4Threads) {
      const int wr = e % kW4Rows, row = e / kW4Rows, col = tile * kW4Rows + wr;
      float sum = 0.f;
      if (ks == 1) {
#pragma unroll
        for (int w = 0; w < kW4Warps; ++w) sum += part[(buf * kW4Warps + w) * kPart + e];
      } else {
        for (uint32_t c = 0; c < ks; ++c) {
          const uint32_t base = map_to_cta(part + buf * kW4Warps * kPart + e, c);
#pragma unroll
          for (int w = 0; w < kW4Warps; ++w) sum += ld_cluster_f32(base + w * kPart * 4);
        }
      }
      if (col < a.n) {
        if (a.bias) sum += Elem<T>::to_float(static_cast<const T*>(a.bias)[col]);
        static_cast<T*>(a.out)[row * a.out_stride + col] = Elem<T>::from_float(sum);
      }
    }
    buf ^= 1;                                       // the other half: its readers passed the barrier above
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (ks > 1) cluster_barrier();                    // nobody leaves while its partial sums may be read
}

// shared memory of a CTA that holds `rows` rows of x over `slabs` slabs
inline size_t w4_smem(int rows, int nt, int slabs) {
  return 2 * kW4Warps * kW4Rows * 8 * static_cast<size_t>(nt) * 4 + kW4Warps * kW4Stages * 1024 +
         static_cast<size_t>(slabs) * kSlab * 2 * rows;
}
constexpr size_t kW4SmemLimit = 227 * 1024 - 1024;

template <int FMT, typename T, int NT, int LW>
int launch_w4(W4Args a, cudaStream_t s) {
  auto kern = w4_linear_kernel<FMT, T, NT, LW>;
  const int slabs = (a.k + kSlab - 1) / kSlab;
  // K over 1, 2, 4 or 8 CTAs: until two CTAs fit an SM and every SM has two, while each warp keeps a slab
  int ks = 1;
  const int sms = sm_count_cached();
  while (ks < 8) {
    const size_t need = w4_smem(a.rows, NT, (slabs + ks - 1) / ks);
    const bool fits = need <= kW4SmemLimit / 2;
    const bool full = static_cast<int64_t>(a.tiles) * ks >= 2 * sms;
    if ((fits && full) || (need <= kW4SmemLimit && slabs / (2 * ks) < kW4Warps)) break;
    ks *= 2;
  }
  a.slabs_per_cta = (slabs + ks - 1) / ks;
  const size_t smem = w4_smem(a.rows, NT, a.slabs_per_cta);
  if (smem > kW4SmemLimit) return B200Q_ERR_CAPACITY;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return B200Q_ERR_CUDA;
  const int per_sm = smem <= kW4SmemLimit / 2 ? 2 : 1;
  const int clusters = max(1, min(a.tiles, sms * per_sm / ks));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * ks));
  cfg.blockDim = dim3(kW4Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ks);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
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
  const int slabs = static_cast<int>((k + kSlab - 1) / kSlab), part = (slabs + 7) / 8;
  for (int rows = 32; rows > 0; --rows)
    if (w4_smem(rows, rows <= 8 ? 1 : rows <= 16 ? 2 : 4, part) <= kW4SmemLimit) return rows;
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
