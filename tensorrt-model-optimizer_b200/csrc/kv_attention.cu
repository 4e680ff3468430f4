// Attention of a step's new tokens over the paged NVFP4 KV cache.
//
//   out[t, h] = sum_j softmax_j(scale * q[t, h] . K[j]) V[j],   K[j] = e2m1 * e4m3 * k_scale2,  V likewise,
// over the tokens j that query t of its request sees (its own position and everything before it).
//
// Work.  A segment is one kv head of one request and one tile of 8 NT query rows (query tokens x the heads
// that share the kv head); its cache tokens are cut into tiles of 128.  All tiles of all segments, each segment
// preceded by kSegCost units for beginning and ending it, form one line that is dealt out to the CTAs in equal
// contiguous shares, so ragged lengths balance without the host knowing a length.  A segment that lies inside one
// share is finished there; pieces of the others go to a workspace as (max, sum, unnormalised output) and
// kv_merge_kernel joins them in a fixed order.
//
// Inside a CTA the four warps take 32 tokens of each tile.  A warp fetches its codes and scales (2 KB + 256 B each for
// K and V at D = 128) with cp.async into a ring of its own, two steps deep, with the page ids read ahead; there is no
// block-wide barrier before the end of a segment.
//
// Mathematics.  S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: cache tokens (or head dimensions) fill the 16
// rows, the query rows the 8 columns, so a group of up to eight heads wastes nothing.  E2M1 times E4M3 has at
// most six significant bits and lies in [2^-10, 2688]: K and V without the per-tensor scale are EXACT in fp16.
// q is multiplied by a power of two per row that brings its largest element to [2^14, 2^15): bf16 elements stay
// exact in fp16 down to 2^-29 of the row's largest.  The only rounding besides fp32 accumulation is P to fp16:
// 2^-11 relative, and 2^-36 of the largest weight below fp16's normal range (P is 2^11 at the reference maximum, so
// that the many small weights of a long request are not lost); the softmax sum takes the unrounded fp32 values.
// The order of the head dimension inside a product and of the tokens inside a tile is free, so a thread's operand is
// one contiguous run of the row: D/4 dimensions of one token for K, D/8 dimensions of four tokens for V, whose nibbles
// are interleaved so that one conversion gives the same dimension of two neighbouring tokens.
//
// What bounds it.  The fetches alone run at 6.3 TB/s (0.95 of the copy rate); with the products 4.2 to 4.8 TB/s: 297
// instructions per 16 tokens of a head of 128, 64 of them conversions and 64 multiplies that issue every other cycle, at
// 0.6 instructions a cycle and scheduler with three warps each.  Measured (device time): 64 requests of 17 to 8192
// tokens, 8 kv heads, group 4, D 128: 69 us for 287 MB (72 with cu_q); 8 x 65536 tokens, group 8: 125 to 135 us for 604 MB
// (165 to 172 with cu_q); 16 requests with up to 8 queries, D 256: 29 us for 39 MB.  Four blocks of 128 registers an SM
// measured 74 / 132 us, blocks of 5, 7, 14 or 16 warps 81 / 147, 85 / 149, 88 / 142 and 83 / 135 us, bulk copies instead of
// cp.async 80 / 145 (four blocks).
#include "umma.cuh"

namespace b200q {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kChunk = 16;                          // tokens of a matrix product
constexpr int kStep = 2 * kChunk;                   // tokens a warp handles at a time
constexpr int kTile = kStep * kAttnWarps;           // tokens of a tile
constexpr int kSegCost = 2;                         // what beginning and ending a segment costs, in tiles
constexpr float kBase = 11.f, kTop = 15.f;          // log2 P at the reference maximum, and the most that P may reach
constexpr float kNone = -3.0e38f;                   // maximum of a row that has seen nothing: below any score, and finite
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const void* q;
  int64_t q_token_stride, q_head_stride;            // elements
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const float *k_scale2, *v_scale2;
  const int* table;
  int64_t table_stride;
  const int* lens;
  const int* cu_q;                                  // NULL: one query per request
  void* out;                                        // [tokens, heads * group, D]
  float* lse;                                       // [tokens, heads * group] or NULL
  float* part;                                      // [ctas, 2, rows, D]
  float2* part_ml;                                  // [ctas, 2, rows]
  int4* desc;                                       // [ctas][2]: pieces, first query, kv head, first row; rows
  FastDiv chunks_per_page, group_div;
  int width, requests, tokens, heads, group, page, pages;
  int zero_tail;                                    // rows of no request: 0 left as they are, 1 zero and lse -inf, 2 lse only
  float scale;
};

struct Request {                                    // one request as the scheduler sees it
  int q0, nq, len, nrt, nkt;
};

template <int RT>
__device__ __forceinline__ Request load_request(const AttnArgs& a, int b) {
  Request r;
  if (a.cu_q) {
    r.q0 = min(max(a.cu_q[b], 0), a.tokens);
    r.nq = min(max(a.cu_q[b + 1], r.q0), a.tokens) - r.q0;
  } else {
    r.q0 = b;
    r.nq = 1;
  }
  const int64_t room = static_cast<int64_t>(a.width) * a.page;
  const int len = max(a.lens[b], 0);
  r.len = len < room ? len : static_cast<int>(room);
  r.nrt = (r.nq * a.group + RT - 1) / RT;
  r.nkt = max((r.len + kTile - 1) / kTile, 1);
  return r;
}
__device__ __forceinline__ int64_t request_work(const AttnArgs& a, const Request& r) {
  return static_cast<int64_t>(a.heads) * r.nrt * (r.nkt + kSegCost);
}

// a place on the line of tiles
struct Cursor {
  int b, h, rt, kt;
  Request r;
};
template <int RT>
__device__ __forceinline__ void next_segment(const AttnArgs& a, Cursor& c) {
  c.kt = 0;
  if (++c.rt < c.r.nrt) return;
  c.rt = 0;
  if (++c.h < a.heads) return;
  c.h = 0;
  do {
    if (c.b + 1 >= a.requests) return;              // not reached while the lengths stay what they were at the start
    c.r = load_request<RT>(a, ++c.b);
  } while (c.r.nrt == 0);
}

// tokens that query row `row` (query token * group + head) of a request sees
__device__ __forceinline__ int row_limit(const AttnArgs& a, const Request& r, int row) {
  const int i = min(static_cast<int>(a.group_div.div(row)), r.nq - 1);
  return min(max(r.len - r.nq + i + 1, 0), r.len);
}

__device__ __forceinline__ void cvt_e2m1x8(uint32_t w, uint32_t* h) {   // 4 bytes -> 4 x f16x2, low nibble in the low half
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint32_t w) {            // low two bytes -> f16x2
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(w)));
  return h;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// N bytes (4, 8, 16 or 32) of shared memory as words
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}

template <int D, int NT>
struct AttnShape {
  static constexpr int kRT = 8 * NT;
  static constexpr int kCodeBytes = kStep * D / 2, kScaleBytes = kStep * D / 16;
  static constexpr int kSlot = 2 * (kCodeBytes + kScaleBytes);
  static constexpr int kStages = 2;
  static constexpr int kRing = kAttnWarps * kStages * kSlot;
  static constexpr int kMerge = kAttnWarps * kRT * D * 4;
  static constexpr int kSmem = kRing + kMerge;
  static constexpr int kCtas = D * NT >= 256 ? 2 : 3;                  // per SM: registers for two halves in flight
};

// kRagged: requests may have several queries (cu_q), so that rows of a tile may see different tokens.
template <typename T, int D, int NT, bool kRagged>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<D, NT>::kCtas)
kv_attention_kernel(const AttnArgs a) {
  using S = AttnShape<D, NT>;
  constexpr int RT = S::kRT, ST = S::kStages;
  constexpr int KW = D / 32;                        // words of codes a thread reads of one K token
  constexpr int KB = D / 64;                        // block scales of them
  constexpr int VW = D / 64;                        // words of codes a thread reads of one V token
  constexpr int VB = D >= 128 ? D / 128 : 1;        // block scales of them
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan_sums[kAttnWarps];
  __shared__ Cursor at_segment[2], pcs[kAttnWarps]; // this and the next segment, each warp's copies: read between segments only
  __shared__ int start_unit;                        // of the first segment
  __shared__ float2 merge_ml[kAttnWarps][RT];

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, qd = lane & 3, gr = lane >> 2;
  pdl_prologue();

  // ---- this CTA's share of the line of tiles ----
  const int per = (a.requests + kAttnThreads - 1) / kAttnThreads;
  const int r0 = min(static_cast<int>(threadIdx.x) * per, a.requests), r1 = min(r0 + per, a.requests);
  int64_t mine = 0;
  for (int b = r0; b < r1; ++b) mine += request_work(a, load_request<RT>(a, b));
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scan_sums[warp] = inc;
  __syncthreads();
  int64_t total = 0, before = inc - mine;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += scan_sums[w];
    total += scan_sums[w];
  }
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total / (kSegCost + 1)), cta = blockIdx.x;
  if (cta >= ctas) {
    if (threadIdx.x == 0) a.desc[2 * cta] = make_int4(0, 0, 0, 0);
    return;
  }
  const int64_t t0 = cta * total / ctas, t1 = (cta + 1) * total / ctas;
  if (t0 >= before && t0 < before + mine) {         // exactly one thread's requests hold the first tile
    int64_t at = before;
    Cursor c;
    for (c.b = r0;; ++c.b) {
      c.r = load_request<RT>(a, c.b);
      const int64_t w = request_work(a, c.r);
      if (t0 < at + w || c.b + 1 >= r1) break;
      at += w;
    }
    const int64_t in = t0 - at;
    const int units = c.r.nkt + kSegCost;           // the first kSegCost units of a segment hold no tile
    const int64_t seg = in / units;
    start_unit = static_cast<int>(in % units);
    c.kt = max(start_unit - kSegCost, 0);
    // (clamped: should somebody change the lengths while this runs, the result is lost, but nothing leaves its bounds)
    c.rt = static_cast<int>(seg % max(c.r.nrt, 1));
    c.h = static_cast<int>(min(seg / max(c.r.nrt, 1), static_cast<int64_t>(a.heads - 1)));
    at_segment[0] = c;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) pcs[w] = c;
  }
  __syncthreads();

  // ---- the warp's producer: cp.async of 32 tokens into a ring of its own ----
  constexpr int kSide = D / 16;                     // lanes that fetch a chunk's scales of one side, 16 bytes each
  uint8_t* ring = smem + warp * ST * S::kSlot;
  const uint32_t ring_addr = smem_u32(ring) + lane * 16;
  const uint32_t scale_addr = smem_u32(ring) + 2 * S::kCodeBytes + (lane < kSide ? lane * 16 : S::kScaleBytes + (lane - kSide) * 16);
  const uint8_t* scale_src = lane < kSide ? a.k_scales + lane * 16 : a.v_scales + (lane - kSide) * 16;
  Cursor& pc = pcs[warp];
  int p_tok = pc.kt * kTile + warp * kStep, p_end = pc.r.nkt * kTile, p_limit = row_limit(a, pc.r, pc.rt * RT + RT - 1);
  int p_left = static_cast<int>(t1 - t0) - max(kSegCost - start_unit, 0);
  const int p_left0 = p_left;                       // tiles and segment costs of the share
  const int* p_row = a.table + pc.b * a.table_stride;
  int p_head = pc.h * a.page;
  const int page_tokens = a.heads * a.page;
  const bool wide = a.page % kStep == 0;            // the 32 tokens of a step lie in one page: one address, no tail
  uint32_t live = 0;                                // bits 2s, 2s + 1: the halves of slot s that hold (or await) tokens
  int p_slot = 0;
  int p_id[2], p_in[2];                             // page ids of the step's halves (negative: nothing to read), tokens into the page
  auto look_up = [&]() {                            // the ids are not looked at before the next step: their latency is hidden
    p_id[0] = p_id[1] = -1;
    if (p_left <= 0 || p_tok >= p_limit) return;
    uint32_t col, in;
    a.chunks_per_page.divmod(p_tok / kChunk, col, in);
    p_in[0] = in * kChunk;
    p_id[0] = __ldg(p_row + col);
    if (!wide && p_tok + kChunk < p_limit) {
      const bool next = in + 1 == a.chunks_per_page.d;                             // the second half begins the next page
      p_in[1] = next ? 0 : p_in[0] + kChunk;
      p_id[1] = __ldg(p_row + col + next);
    }
  };
  look_up();
  auto produce = [&]() {
    uint32_t ok = 0;
    if (wide) {
      if (static_cast<uint32_t>(p_id[0]) < static_cast<uint32_t>(a.pages)) {
        ok = 3;                                     // tokens behind the limit are in the page too, and masked below
        const int64_t row = static_cast<int64_t>(p_id[0]) * page_tokens + (p_head + p_in[0]);
        const uint8_t* ksrc = a.k_codes + row * (D / 2) + lane * 16;
        const uint8_t* vsrc = a.v_codes + row * (D / 2) + lane * 16;
        const uint8_t* ssrc = scale_src + row * (D / 16);
        const uint32_t dst = ring_addr + p_slot * S::kSlot, sdst = scale_addr + p_slot * S::kSlot;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          copy_async16(dst + i * 512, ksrc + i * 512);
          copy_async16(dst + S::kCodeBytes + i * 512, vsrc + i * 512);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (lane < 2 * kSide) copy_async16(sdst + c * (S::kScaleBytes / 2), ssrc + c * (S::kScaleBytes / 2));
      }
    } else {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (static_cast<uint32_t>(p_id[c]) < static_cast<uint32_t>(a.pages)) {
        ok |= 1u << c;
        const int64_t row = static_cast<int64_t>(p_id[c]) * page_tokens + (p_head + p_in[c]);
        const uint8_t* ksrc = a.k_codes + row * (D / 2) + lane * 16;
        const uint8_t* vsrc = a.v_codes + row * (D / 2) + lane * 16;
        const uint32_t dst = ring_addr + p_slot * S::kSlot + c * (S::kCodeBytes / 2);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          copy_async16(dst + i * 512, ksrc + i * 512);
          copy_async16(dst + S::kCodeBytes + i * 512, vsrc + i * 512);
        }
        if (lane < 2 * kSide) copy_async16(scale_addr + p_slot * S::kSlot + c * (S::kScaleBytes / 2), scale_src + row * (D / 16));
      }
    }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    live = (live & ~(3u << (2 * p_slot))) | ok << (2 * p_slot);
    p_slot = p_slot + 1 == ST ? 0 : p_slot + 1;
    p_tok += kTile;
    if (--p_left > 0 && p_tok >= p_end && (p_left -= kSegCost) > 0) {
      __syncwarp();                                 // every lane has read the segment that lane 0 now replaces
      if (lane == 0) next_segment<RT>(a, pc);
      __syncwarp();
      p_tok = warp * kStep;
      p_end = pc.r.nkt * kTile;
      p_row = a.table + pc.b * a.table_stride;
      p_head = pc.h * a.page;
      p_limit = row_limit(a, pc.r, pc.rt * RT + RT - 1);
    }
    look_up();
  };
#pragma unroll 1
  for (int s = 0; s < ST; ++s) produce();

  const float qk = a.scale * kLog2e * __ldg(a.k_scale2), v2 = __ldg(a.v_scale2);
  int left = p_left0;
  int slot = 0;
  int4 my_desc = make_int4(0, 0, 0, 0);
  int my_rows = 0;

  // queries: thread (gr, qd) holds dimensions qd * D/4 ... of row gr of each 8-row tile
  uint32_t qf[NT][D / 8];
  auto load_q = [&](const Cursor& c) {
    const int first = c.rt * RT, rows = min(c.r.nq * a.group - first, RT);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) qf[n][i] = 0;
      if (8 * n + gr < rows) {
        uint32_t tok, hd;
        a.group_div.divmod(first + 8 * n + gr, tok, hd);
        hd += c.h * a.group;
        const T* src = static_cast<const T*>(a.q) + (c.r.q0 + tok) * a.q_token_stride + hd * a.q_head_stride + qd * (D / 4);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
          qf[n][4 * i] = v.x; qf[n][4 * i + 1] = v.y; qf[n][4 * i + 2] = v.z; qf[n][4 * i + 3] = v.w;
        }
      }
    }
  };
  load_q(at_segment[0]);

#pragma unroll 1
  for (int which = 0; left > 0; which ^= 1) {
    // ---- one segment, or this CTA's part of it ----
    const Cursor& cc = at_segment[which];
    const int kt_end = min(cc.r.nkt, cc.kt + left);
    const int row0 = cc.rt * RT, rows = min(cc.r.nq * a.group - row0, RT);
    const int lim_lo = row_limit(a, cc.r, row0), lim_hi = row_limit(a, cc.r, row0 + rows - 1);
    float qs[NT][2];                                // q becomes fp16 times 2^k of its row
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float back = 1.f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t top = 0;                           // largest finite |q| of the row, as a bf16 pattern
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t lo = qf[n][i] & 0x7fffu, hi = (qf[n][i] >> 16) & 0x7fffu;
          top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(static_cast<int>(top >> 7), 28);       // biased exponent, kept where 2^(14-e) is a normal number
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - e) << 23);
        back = __uint_as_float(static_cast<uint32_t>(e - 14) << 23);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          qf[n][i] = pack_f16(__uint_as_float(qf[n][i] << 16) * up, __uint_as_float(qf[n][i] & 0xffff0000u) * up);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {                 // of the rows this thread's accumulators belong to
        qs[n][j] = qk * __shfl_sync(0xffffffffu, back, 4 * (2 * qd + j));
      }
    }
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = kNone;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    }

    // row gr of the 16 x 8 product is token gr ^ bit 1 of gr: both operands' shared-memory reads then spread
    const int tg = gr ^ ((gr >> 1) & 1);
    // the tokens of V's operand: rows 2 qd and 2 qd + 1, and the same + 8
    const int ta = (2 * qd) ^ (qd & 1), tb = ta ^ 1;

#pragma unroll 1
    for (int kt = cc.kt; kt < kt_end; ++kt) {
      const uint32_t here = (live >> (2 * slot)) & 3u;
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
      __syncwarp();                                 // every lane's part of the slot has landed
      if (here != 0) {
        const uint8_t* kc = ring + slot * S::kSlot;
        const uint8_t* vc = kc + S::kCodeBytes;
        const uint8_t* ks = kc + 2 * S::kCodeBytes;
        const uint8_t* vs = ks + S::kScaleBytes;
        const int tok0 = kt * kTile + warp * kStep;
        // ---- scores of 32 tokens ----
        float s[2][NT][4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[c][n][0] = s[c][n][1] = s[c][n][2] = s[c][n][3] = 0.f;
          uint32_t w[2][KW];
          lds_words<4 * KW>(kc + (c * kChunk + tg) * (D / 2) + qd * (D / 8), w[0]);
          lds_words<4 * KW>(kc + (c * kChunk + tg + 8) * (D / 2) + qd * (D / 8), w[1]);
          uint32_t sc[2][KB];                       // block scales, each twice
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* p = ks + (c * kChunk + tg + 8 * r) * (D / 16) + qd * KB;
#pragma unroll
            for (int i = 0; i < KB; i += 2) {
              const uint32_t two = KB == 1 ? *p : *reinterpret_cast<const uint16_t*>(p + i);
              const uint32_t h = cvt_e4m3x2(two);
              sc[r][i] = __byte_perm(h, h, 0x1010);
              if constexpr (KB > 1) sc[r][i + 1] = __byte_perm(h, h, 0x3232);
            }
          }
#pragma unroll
          for (int i = 0; i < KW; ++i) {            // one word of each token = 8 dimensions = two k steps
            uint32_t x[4], y[4];
            cvt_e2m1x8(w[0][i], x);
            cvt_e2m1x8(w[1][i], y);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = hmul2(x[j], sc[0][i / 2]); y[j] = hmul2(y[j], sc[1][i / 2]); }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16(s[c][n], x[0], y[0], x[1], y[1], qf[n][4 * i], qf[n][4 * i + 1]);
              mma_f16(s[c][n], x[2], y[2], x[3], y[3], qf[n][4 * i + 2], qf[n][4 * i + 3]);
            }
          }
        }
        // ---- softmax, base 2 ----
        const bool masked = tok0 + kStep > lim_lo || here != 3u;
        uint32_t hidden = 0;                        // bit 8 n + 4 c + j: that score is masked
        if (masked) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int see = row_limit(a, cc.r, row0 + 8 * n + 2 * qd + j) - tok0 - tg;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (c * kChunk >= see || !(here >> c & 1u)) hidden |= 1u << (8 * n + 4 * c + j);
                if (c * kChunk + 8 >= see || !(here >> c & 1u)) hidden |= 1u << (8 * n + 4 * c + j + 2);
              }
            }
        }
        // less[c][n][j]: log2 P, the scaled score less the row's reference (kBase below a maximum of its scores)
        float less[2][NT][4];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) less[c][n][j] = fmaf(s[c][n][j], qs[n][j & 1], -m[n][j & 1]);
          if (hidden) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (hidden >> (8 * n + 4 * c + j) & 1u) less[c][n][j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
            grow |= fmaxf(fmaxf(less[0][n][j], less[0][n][j + 2]), fmaxf(less[1][n][j], less[1][n][j + 2])) > kTop;
        }
        // the reference follows only when a score passes the maximum by 2^4 (P stays within fp16): rarely
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float t = kNone;
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int r = 0; r < 4; r += 2)
                  if (less[c][n][j + r] != -INFINITY) t = fmaxf(t, s[c][n][j + r] * qs[n][j]);
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
              t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
              t = fmaxf(m[n][j], t - kBase);
              const float f = m[n][j] == t ? 1.f : exp2_fast(m[n][j] - t);
              m[n][j] = t;
              l[n][j] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[n][i][j] *= f; o[n][i][j + 2] *= f; }
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int r = 0; r < 4; r += 2)
                  if (less[c][n][j + r] != -INFINITY) less[c][n][j + r] = fmaf(s[c][n][j + r], qs[n][j], -t);
            }
          }
        }
        uint32_t pb[2][NT][2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float p0 = exp2_fast(less[c][n][0]), p1 = exp2_fast(less[c][n][1]);
            const float p2 = exp2_fast(less[c][n][2]), p3 = exp2_fast(less[c][n][3]);
            l[n][0] += p0 + p2;
            l[n][1] += p1 + p3;
            pb[c][n][0] = transpose8x8(pack_f16(p0, p1));
            pb[c][n][1] = transpose8x8(pack_f16(p2, p3));
          }
        // ---- output: tokens ta, tb and the same + 8 of either half ----
        uint32_t sb[2][2][VB];                      // scale bytes of a token pair
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < VB; ++i) {
              const int blk = D >= 128 ? gr * VB + i : gr >> 1, t = c * kChunk + 8 * r;
              sb[c][r][i] = vs[(ta + t) * (D / 16) + blk] | (vs[(tb + t) * (D / 16) + blk] << 8);
            }
        bool nan_v = false;
        if (masked) {                               // behind the last token anything may stand: 0 * NaN is NaN
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < VB; ++i) {
                const int t = tok0 + c * kChunk + 8 * r;
                const bool on = here >> c & 1u;
                sb[c][r][i] &= (on && t + ta < lim_hi ? 0xffu : 0u) | (on && t + tb < lim_hi ? 0xff00u : 0u);
                // some rows see tokens that others do not
                if constexpr (kRagged)
                  nan_v |= lim_lo < lim_hi && ((sb[c][r][i] & 0x7fu) == 0x7fu || (sb[c][r][i] & 0x7f00u) == 0x7f00u);
              }
        }
        if (!kRagged || !masked || !__any_sync(0xffffffffu, nan_v)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t wa[2][VW], wb[2][VW], sh[2][VB];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              lds_words<4 * VW>(vc + (c * kChunk + ta + 8 * r) * (D / 2) + gr * (D / 16), wa[r]);
              lds_words<4 * VW>(vc + (c * kChunk + tb + 8 * r) * (D / 2) + gr * (D / 16), wb[r]);
#pragma unroll
              for (int i = 0; i < VB; ++i) sh[r][i] = cvt_e4m3x2(sb[c][r][i]);
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              uint32_t x[2][4], y[2][4];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                cvt_e2m1x8((wa[r][w] & 0x0f0f0f0fu) | ((wb[r][w] << 4) & 0xf0f0f0f0u), x[r]);
                cvt_e2m1x8(((wa[r][w] >> 4) & 0x0f0f0f0fu) | (wb[r][w] & 0xf0f0f0f0u), y[r]);
#pragma unroll
                for (int j = 0; j < 4; ++j) { x[r][j] = hmul2(x[r][j], sh[r][w / 2]); y[r][j] = hmul2(y[r][j], sh[r][w / 2]); }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  mma_f16(o[n][4 * w + j], x[0][j], y[0][j], x[1][j], y[1][j], pb[c][n][0], pb[c][n][1]);
            }
          }
        } else if constexpr (kRagged) {
          // A NaN value that only some rows may see: each row's product on its own, with what it does not see
          // zeroed, and only that row's column kept.
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t wa[2][VW], wb[2][VW];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              lds_words<4 * VW>(vc + (c * kChunk + ta + 8 * r) * (D / 2) + gr * (D / 16), wa[r]);
              lds_words<4 * VW>(vc + (c * kChunk + tb + 8 * r) * (D / 2) + gr * (D / 16), wb[r]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll 1
              for (int col = 0; col < 8; ++col) {
                const int see = row_limit(a, cc.r, row0 + 8 * n + col) - tok0 - c * kChunk;
#pragma unroll
                for (int w = 0; w < VW; ++w) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    uint32_t f[4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                      uint32_t x[4], y[4];
                      cvt_e2m1x8((wa[r][w] & 0x0f0f0f0fu) | ((wb[r][w] << 4) & 0xf0f0f0f0u), x);
                      cvt_e2m1x8(((wa[r][w] >> 4) & 0x0f0f0f0fu) | (wb[r][w] & 0xf0f0f0f0u), y);
                      const uint32_t sh = cvt_e4m3x2(sb[c][r][w / 2] & ((ta + 8 * r < see ? 0xffu : 0u) | (tb + 8 * r < see ? 0xff00u : 0u)));
                      f[2 * r] = hmul2(x[j], sh);
                      f[2 * r + 1] = hmul2(y[j], sh);
                    }
                    float* acc = o[n][4 * w + j];
                    float t[4] = {acc[0], acc[1], acc[2], acc[3]};
                    mma_f16(t, f[0], f[1], f[2], f[3], pb[c][n][0], pb[c][n][1]);
                    if (col == 2 * qd) { acc[0] = t[0]; acc[2] = t[2]; }
                    if (col == 2 * qd + 1) { acc[1] = t[1]; acc[3] = t[3]; }
                  }
                }
              }
            }
          }
        }
      }
      __syncwarp();                                 // the slot has been read by every lane
      produce();
      slot = slot + 1 == ST ? 0 : slot + 1;
    }

    // ---- join the four warps ----
    float* merge = reinterpret_cast<float*>(smem + S::kRing);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = l[n][j];
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
        t += __shfl_xor_sync(0xffffffffu, t, 16);
        const int row = 8 * n + 2 * qd + j;
        if (gr == 0) merge_ml[warp][row] = make_float2(m[n][j], t);
        float* dst = merge + (warp * RT + row) * D + gr * (D / 8);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[n][i][j], o[n][i][j + 2]);
      }
    }
    const bool first_piece = cc.kt == 0, last_piece = kt_end == cc.r.nkt;
    left -= kt_end - cc.kt + kSegCost;
    if (threadIdx.x == 0 && left > 0) {
      Cursor next = cc;
      next_segment<RT>(a, next);
      at_segment[which ^ 1] = next;
    }
    __syncthreads();
    if (left > 0) load_q(at_segment[which ^ 1]);    // on its way while the warps' parts are joined
    const bool whole = first_piece && last_piece;
    const int piece = first_piece ? 1 : 0;          // slot 0: the segment began in an earlier CTA
    for (int i = threadIdx.x; i < RT * D / 4; i += kAttnThreads) {
      const int row = i / (D / 4), d = 4 * (i % (D / 4));
      if (row >= rows) continue;
      float mm = kNone, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) mm = fmaxf(mm, merge_ml[w][row].x);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float2 ml = merge_ml[w][row];
        // a warp that saw nothing weighs nothing; NaN sums stay NaN
        const float f = ml.x == kNone ? (ml.y == 0.f ? 0.f : ml.y) : exp2_fast(ml.x - mm);
        ll += ml.y * f;
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * RT + row) * D + d);
        if (f != 0.f) { acc[0] += v.x * f; acc[1] += v.y * f; acc[2] += v.z * f; acc[3] += v.w * f; }
      }
      if (whole) {
        uint32_t tok, hd;
        a.group_div.divmod(row0 + row, tok, hd);
        const int64_t at = static_cast<int64_t>(cc.r.q0 + tok) * (a.heads * a.group) + cc.h * a.group + hd;
        const float f = ll == 0.f ? 0.f : __fdividef(v2, ll);
        uint2 packed;
        packed.x = Elem<T>::pack2(acc[0] * f, acc[1] * f);
        packed.y = Elem<T>::pack2(acc[2] * f, acc[3] * f);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * D + d) = packed;
        if (a.lse && d == 0) a.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
      } else {
        const int64_t p = (cta * 2 + piece) * RT + row;
        *reinterpret_cast<float4*>(a.part + p * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) a.part_ml[p] = make_float2(mm, ll);
      }
    }
    if (first_piece && !last_piece) {               // the pieces that follow belong to the next CTAs, one each
      const int64_t seg_last = t1 + (cc.r.nkt - kt_end) - 1;
      const int64_t owner = ((seg_last + 1) * ctas - 1) / total;
      my_desc = make_int4(static_cast<int>(owner - cta + 1), cc.r.q0, cc.h, row0);
      my_rows = rows;
    }
    __syncthreads();                                // read before the next segment's parts are written
  }
  if (threadIdx.x == 0) {
    a.desc[2 * cta] = my_desc;
    a.desc[2 * cta + 1] = make_int4(my_rows, 0, 0, 0);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Pieces of the segments that span several CTAs, joined in the order of the CTAs.  Block (c, row): the segment
// that begins in CTA c's share and ends in a later one.  All pieces' maxima and sums first, which gives every piece
// its weight; then groups of D/4 threads add up every kGroups-th piece, with loads that depend on nothing.
constexpr int kMergeMost = 2048;                    // CTAs, hence pieces, at most

template <typename T, int D, int RT>
__global__ void __launch_bounds__(128)
kv_merge_kernel(const AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = 128 / kLanes;
  __shared__ float4 acc_s[kGroups][kLanes];
  __shared__ float weight[kMergeMost], red[2][4];
  pdl_prologue();
  if (a.zero_tail) {                                // rows in front of the first request and behind the last one
    const int heads = a.heads * a.group;
    const int64_t head = static_cast<int64_t>(min(max(a.cu_q[0], 0), a.tokens)) * heads;
    const int64_t tail = static_cast<int64_t>(min(max(a.cu_q[a.requests], 0), a.tokens)) * heads;
    const int64_t end = head + static_cast<int64_t>(a.tokens) * heads - tail, nb = static_cast<int64_t>(gridDim.x) * gridDim.y;
    for (int64_t i = blockIdx.y * gridDim.x + blockIdx.x; i < end; i += nb) {
      const int64_t r = i < head ? i : tail + i - head;
      if (a.zero_tail != 2)
        for (int d = threadIdx.x; d < D; d += 128) static_cast<T*>(a.out)[r * D + d] = Elem<T>::from_float(0.f);
      if (a.lse && threadIdx.x == 0) a.lse[r] = -INFINITY;
    }
  }
  const int4 seg = a.desc[2 * blockIdx.x];
  const int row = blockIdx.y, pieces = seg.x;
  if (pieces == 0 || row >= a.desc[2 * blockIdx.x + 1].x) return;
  auto slot_of = [&](int i) { return (static_cast<int64_t>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * RT + row; };
  const int warp = threadIdx.x >> 5, lane32 = threadIdx.x & 31;
  float mm = kNone;
  for (int i = threadIdx.x; i < pieces; i += 128) mm = fmaxf(mm, a.part_ml[slot_of(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (lane32 == 0) red[0][warp] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float ll = 0.f;
  for (int i = threadIdx.x; i < pieces; i += 128) {
    const float2 ml = a.part_ml[slot_of(i)];
    // a piece that saw nothing weighs nothing; NaN sums stay NaN
    const float f = ml.x == kNone ? (ml.y == 0.f ? 0.f : ml.y) : exp2_fast(ml.x - mm);
    weight[i] = f;
    ll += ml.y * f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, o);
  if (lane32 == 0) red[1][warp] = ll;
  __syncthreads();
  ll = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = grp; i < pieces; i += kGroups) {
    const float f = weight[i];
    const float4 v = *reinterpret_cast<const float4*>(a.part + slot_of(i) * D + 4 * lane);
    if (f != 0.f) { acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f; }
  }
  acc_s[grp][lane] = acc;
  __syncthreads();
  if (grp) return;
  for (int g = 1; g < kGroups; ++g) {
    const float4 v = acc_s[g][lane];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  uint32_t tok, hd;
  a.group_div.divmod(seg.w + row, tok, hd);
  const int64_t at = static_cast<int64_t>(seg.y + tok) * (a.heads * a.group) + seg.z * a.group + hd;
  const float f = ll == 0.f ? 0.f : __fdividef(__ldg(a.v_scale2), ll);
  uint2 packed;
  packed.x = Elem<T>::pack2(acc.x * f, acc.y * f);
  packed.y = Elem<T>::pack2(acc.z * f, acc.w * f);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * D + 4 * lane) = packed;
  if (a.lse && lane == 0) a.lse[at] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * kLn2;
}

template <typename T, int D, int NT>
int launch_attention(const AttnArgs& a, int ctas, cudaStream_t s) {
  using S = AttnShape<D, NT>;
  auto kern = a.cu_q ? kv_attention_kernel<T, D, NT, true> : kv_attention_kernel<T, D, NT, false>;
  static std::atomic<uint64_t> done[2];
  if (!allow_smem(reinterpret_cast<const void*>(kern), S::kSmem, done[a.cu_q ? 1 : 0])) return B200Q_ERR_CUDA;
  launch_pdl(kern, ctas, kAttnThreads, S::kSmem, s, a);
  launch_pdl(kv_merge_kernel<T, D, S::kRT>, dim3(ctas, S::kRT), 128, 0, s, a);
  return launch_status();
}

// 8-row tiles unless the rows of a request fill more than one; heads of 256 have registers for one only
inline int row_tiles(int dim, int tokens, int requests, int group) {
  const int64_t rows = static_cast<int64_t>(group) * ((tokens + requests - 1) / requests);
  return dim < 256 && rows > 8 ? 2 : 1;
}
inline int ctas_per_sm(int dim, int nt) { return dim * nt >= 256 ? 2 : 3; }

}  // namespace b200q

using namespace b200q;

extern "C" int64_t b200q_nvfp4_kv_attention_workspace(int tokens, int requests, int heads, int group, int dim) {
  if (tokens <= 0 || requests <= 0 || heads <= 0 || group <= 0 || (dim != 64 && dim != 128 && dim != 256)) return B200Q_ERR_SHAPE;
  const int nt = row_tiles(dim, tokens, requests, group);
  const int64_t ctas = static_cast<int64_t>(sm_count_cached()) * ctas_per_sm(dim, nt);
  return ctas * (32 + 2 * 8 * nt * (4 * static_cast<int64_t>(dim) + 8));
}

extern "C" int b200q_nvfp4_kv_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                        const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes,
                                        const uint8_t* v_scales, const float* k_scale2, const float* v_scale2,
                                        const int* table, int64_t table_stride, int width, const int* lens, const int* cu_q,
                                        int requests, int tokens, int heads, int group, int dim, int pages, int page,
                                        float scale, void* out, float* lse, int zero_tail, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  B200Q_REQUIRE_PTR(q); B200Q_REQUIRE_PTR(k_codes); B200Q_REQUIRE_PTR(k_scales); B200Q_REQUIRE_PTR(v_codes);
  B200Q_REQUIRE_PTR(v_scales); B200Q_REQUIRE_PTR(k_scale2); B200Q_REQUIRE_PTR(v_scale2); B200Q_REQUIRE_PTR(lens);
  B200Q_REQUIRE_PTR(out); B200Q_REQUIRE_PTR(workspace);
  if (width > 0) B200Q_REQUIRE_PTR(table);
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_DTYPE;
  if (requests <= 0 || tokens <= 0 || heads <= 0 || group <= 0 || pages <= 0 || width < 0 || table_stride < 0) return B200Q_ERR_SHAPE;
  if (page <= 0 || page % kChunk) return B200Q_ERR_SHAPE;
  if (!cu_q && tokens != requests) return B200Q_ERR_SHAPE;
  if (dim != 64 && dim != 128 && dim != 256) return B200Q_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(tokens) * group > kFastDivLimit / 2 || static_cast<int64_t>(heads) * group > kFastDivLimit ||
      static_cast<int64_t>(width) * page > (1 << 30) || static_cast<int64_t>(heads) * page > (1 << 30))
    return B200Q_ERR_UNSUPPORTED;
  const uintptr_t align = reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(2 * q_token_stride) |
                          static_cast<uintptr_t>(2 * q_head_stride) | reinterpret_cast<uintptr_t>(k_codes) |
                          reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_codes) |
                          reinterpret_cast<uintptr_t>(v_scales) | reinterpret_cast<uintptr_t>(out) |
                          reinterpret_cast<uintptr_t>(workspace);
  if (align & 15u) return B200Q_ERR_ALIGN;
  if (workspace_bytes < b200q_nvfp4_kv_attention_workspace(tokens, requests, heads, group, dim)) return B200Q_ERR_CAPACITY;
  const int nt = row_tiles(dim, tokens, requests, group);
  const int ctas = min(sm_count_cached() * ctas_per_sm(dim, nt), kMergeMost);
  AttnArgs a{};
  a.q = q; a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride;
  a.k_codes = k_codes; a.k_scales = k_scales; a.v_codes = v_codes; a.v_scales = v_scales;
  a.k_scale2 = k_scale2; a.v_scale2 = v_scale2;
  a.table = table; a.table_stride = table_stride; a.lens = lens; a.cu_q = cu_q;
  a.out = out; a.lse = lse;
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(a.desc + 2 * ctas);
  a.part_ml = reinterpret_cast<float2*>(a.part + static_cast<int64_t>(ctas) * 2 * 8 * nt * dim);
  a.width = width; a.requests = requests; a.tokens = tokens; a.heads = heads; a.group = group;
  a.page = page; a.pages = pages; a.zero_tail = cu_q ? zero_tail : 0;
  a.scale = scale;
  a.chunks_per_page = FastDiv(page / kChunk);
  a.group_div = FastDiv(group);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (dim == 64) return nt == 2 ? launch_attention<T, 64, 2>(a, ctas, s) : launch_attention<T, 64, 1>(a, ctas, s);
    if (dim == 128) return nt == 2 ? launch_attention<T, 128, 2>(a, ctas, s) : launch_attention<T, 128, 1>(a, ctas, s);
    return launch_attention<T, 256, 1>(a, ctas, s);
  };
  return dtype == B200Q_F16 ? go(__half()) : go(__nv_bfloat16());
}
