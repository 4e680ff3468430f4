// The paged NVFP4 KV cache: page tables and slots of a step, and the write of new keys and values.
//
// Cache layout: codes [pages, kv heads, page, D/2] (E2M1, low nibble first) and block scales
// [pages, kv heads, page, D/16] (E4M3), so the tokens of one head inside one page are one run of bytes:
// 16 tokens of a head of 128 are 1 KB of codes and 128 B of scales for whoever reads them.
#include "nvfp4.cuh"

namespace b200q {

// ---- step ------------------------------------------------------------------------------------------
// For request b with L tokens held and n new ones, page size p:
//   have = ceil(L/p), want = ceil((L+n)/p), need = want - have,
//   base = taken + exclusive scan of need,   table[b, have + i] = free[base + i]
//   cu   = exclusive scan of n,              token t of b: pos = L + t - cu[b], slot = table[b, pos/p]*p + pos%p
// A request that is malformed, wider than its table row or beyond the free list is refused: it keeps its
// length, its tokens get slot -1, and a status bit says why.  Its rows have no keys in the cache, so `seen`, the length
// that the step's attention takes, is 0 for it.
//
// One launch and no order between blocks: every block repeats the two scans in shared memory (4 words a
// request), then writes its share of the table entries and of the token rows, each found by a binary search
// in the scans.  New table entries are computed from the free list and never read back, so nothing waits for
// another block.  Latency-bound: 64 requests of one token each are 1.8 KB of traffic and take 3.1 us, 512 requests with
// 131 thousand new tokens 7.5 us (device time).
constexpr int kStepThreads = 256;
constexpr int kStepMaxRequests = 8192;

enum { kStepNoPages = 1, kStepRowFull = 2, kStepBadLength = 4, kStepRowsShort = 8 };

// last index i in [0, n) with scan[i] <= v, scan non-decreasing and scan[0] <= v
__device__ __forceinline__ int find_row(const int* scan, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (scan[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// exclusive scan of one value per thread; `total` receives the sum
__device__ __forceinline__ int64_t cta_scan_excl(int64_t v, int64_t* warp_sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kStepThreads / 32; ++w) {
    const int64_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();
  total = all;
  return before + inc - v;
}

__global__ void __launch_bounds__(kStepThreads, 5)   // 48 registers; 62, which the compiler takes unasked: 8.4 us instead of 7.5
kv_step_kernel(const int* __restrict__ lens, const int* __restrict__ new_lens, const int* __restrict__ free_pages,
               int nfree, const int* __restrict__ taken_in, int* __restrict__ table, int64_t table_stride, int width,
               int requests, int page, int tokens, int64_t* __restrict__ slots, int* __restrict__ positions,
               int* __restrict__ cu_out, int* __restrict__ lens_out, int* __restrict__ taken_out,
               int* __restrict__ status, int* __restrict__ seen) {
  extern __shared__ int step_smem[];
  int* cu = step_smem;                       // [requests + 1] first token row of a request, clamped to `tokens`
  int* base = cu + requests + 1;             // [requests + 1] first index into the free list, counted from `taken`
  int* have = base + requests + 1;           // [requests] pages held, -1 for a refused request
  __shared__ int64_t warp_sums[kStepThreads / 32];
  __shared__ int accepted_end, bits;
  pdl_prologue();
  if (threadIdx.x == 0) { accepted_end = 0; bits = 0; }
  const int per = (requests + kStepThreads - 1) / kStepThreads;
  const int r0 = min(static_cast<int>(threadIdx.x) * per, requests), r1 = min(r0 + per, requests);
  const int taken = *taken_in;
  const int avail = (taken >= 0 && taken <= nfree) ? nfree - taken : 0;

  int64_t sum_new = 0;
  for (int r = r0; r < r1; ++r) sum_new += max(new_lens[r], 0);
  int64_t total_new, total_need;
  int64_t at = cta_scan_excl(sum_new, warp_sums, total_new);
  int64_t sum_need = 0;
  int mine = 0;                              // status bits of this thread's requests
  for (int r = r0; r < r1; ++r) {
    const int64_t L = lens[r], n = new_lens[r], first = at;
    at += max(n, static_cast<int64_t>(0));
    cu[r] = static_cast<int>(min(first, static_cast<int64_t>(tokens)));
    const int64_t held = (L + page - 1) / page, want = (L + max(n, static_cast<int64_t>(0)) + page - 1) / page;
    int bad = 0;
    if (L < 0 || n < 0 || L + n > 0x7fffffff) bad = kStepBadLength;
    else if (want > width) bad = kStepRowFull;
    else if (at > tokens) bad = kStepRowsShort;
    mine |= bad;
    have[r] = bad ? -1 : static_cast<int>(held);
    base[r] = bad ? 0 : static_cast<int>(want - held);      // need, until the scan below replaces it
    sum_need += bad ? 0 : want - held;
  }
  int64_t p = cta_scan_excl(sum_need, warp_sums, total_need);
  int end = 0;
  for (int r = r0; r < r1; ++r) {
    const int need = base[r];
    base[r] = static_cast<int>(min(p, static_cast<int64_t>(avail)));
    p += need;
    if (need > 0) {                          // after one refusal every later request that needs a page is refused too
      if (p > avail) { mine |= kStepNoPages; have[r] = -1; }
      else end = static_cast<int>(p);
    }
  }
  if (end) atomicMax(&accepted_end, end);
  if (mine) atomicOr(&bits, mine);
  if (threadIdx.x == 0) cu[requests] = static_cast<int>(min(total_new, static_cast<int64_t>(tokens)));
  __syncthreads();

  const int step = gridDim.x * kStepThreads, first = blockIdx.x * kStepThreads + threadIdx.x;
  // requests are accepted in order until the free list runs out, so the pages taken are its first ones
  const int pages_taken = accepted_end;
  for (int i = first; i < pages_taken; i += step) {
    const int r = find_row(base, requests, i);
    if (have[r] >= 0) table[r * table_stride + have[r] + (i - base[r])] = free_pages[taken + i];
  }
  const int real = cu[requests];
  for (int t = first; t < tokens; t += step) {
    int64_t slot = -1;
    int pos = 0;
    if (t < real) {
      const int r = find_row(cu, requests, t);
      if (have[r] >= 0) {
        pos = lens[r] + (t - cu[r]);
        const int col = pos / page;
        const int id = col < have[r] ? table[r * table_stride + col] : free_pages[taken + base[r] + (col - have[r])];
        slot = id < 0 ? -1 : static_cast<int64_t>(id) * page + (pos - col * page);
      }
    }
    slots[t] = slot;
    positions[t] = pos;
  }
  for (int r = first; r < requests; r += step) {
    cu_out[r] = cu[r];
    const int held = lens[r], after = have[r] < 0 ? held : held + new_lens[r];
    lens_out[r] = after;
    if (seen) seen[r] = have[r] < 0 ? 0 : after;
  }
  if (first == 0) {
    cu_out[requests] = real;
    *taken_out = taken + pages_taken;
    *status = bits;
  }
}

// ---- append ----------------------------------------------------------------------------------------
// One thread quantises one 16-element block of a head's key and value (the arithmetic of nvfp4_quantize
// with saturating block scales) and stores 8 bytes of codes and one of scale at the token's slot, and, where
// `values` are asked for, what the cache now stands for.  Reads 2 bytes an element, writes 0.5625 (+ 2); bound by HBM.
// One block of threads per 256 units measured better than a grid of resident blocks that stride (54 against 61 us for
// 32768 tokens of 8 heads of 128 with values, 5.65 TB/s; 13.7 against 12.9 for 8192 tokens, which stay in L2).
struct KvSide {
  const void* x;
  int64_t token_stride, head_stride;       // in elements
  const float* scale2;
  uint8_t* codes;
  uint8_t* scales;
  void* values;                            // [tokens, heads, dim] or NULL
};

template <typename T>
__global__ void __launch_bounds__(256)
kv_append_kernel(KvSide k, KvSide v, const int64_t* __restrict__ slots, int nblocks, FastDiv blocks_per_head,
                 FastDiv heads, FastDiv page, int64_t nslots) {
  pdl_prologue();
  const Nvfp4Tensor tk(__ldg(k.scale2)), tv(__ldg(v.scale2));
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < nblocks) {
    uint32_t th, j, t, h;
    blocks_per_head.divmod(i, th, j);
    heads.divmod(th, t, h);
    Block16<T> kb, vb;                       // the key's and the value's block: both loads are in flight together
    kb.load(static_cast<const T*>(k.x) + t * k.token_stride + h * k.head_stride + 16 * j);
    vb.load(static_cast<const T*>(v.x) + t * v.token_stride + h * v.head_stride + 16 * j);
    const int64_t slot = __ldg(slots + t);
    int64_t b = -1;
    if (slot >= 0 && slot < nslots) {
      uint32_t id, row;
      page.divmod(static_cast<uint32_t>(slot), id, row);
      b = ((static_cast<int64_t>(id) * heads.d + h) * page.d + row) * blocks_per_head.d + j;
    }
    auto put = [&](const Block16<T>& blk, const KvSide& side, const Nvfp4Tensor& tn) {
      const float bamax = __uint_as_float(blk.amax_f32bits());
      const uint32_t code = nvfp4_scale_code<false>(bamax, tn);
      const float d = e4m3_to_f32(code) * tn.s2;
      float f[16];
      blk.decode(f);
      const uint2 packed = nvfp4_encode16<sizeof(T) == 2>(f, d, bamax);
      if (b >= 0) {
        *reinterpret_cast<uint2*>(side.codes + 8 * b) = packed;
        side.scales[b] = static_cast<uint8_t>(code);
      }
      if (side.values) {
        nvfp4_decode16(packed, d, f);
        store16(static_cast<T*>(side.values) + static_cast<int64_t>(i) * 16, f);
      }
    };
    put(kb, k, tk);
    put(vb, v, tv);
  }
}

}  // namespace b200q

using namespace b200q;

extern "C" int b200q_kv_step_seen(const int* lens, const int* new_lens, const int* free_pages, int nfree, const int* taken,
                                  int* table, int64_t table_stride, int width, int requests, int page, int tokens,
                                  int64_t* slots, int* positions, int* cu_new, int* lens_out, int* taken_out, int* status,
                                  int* seen, void* stream) {
  B200Q_REQUIRE_PTR(lens); B200Q_REQUIRE_PTR(new_lens); B200Q_REQUIRE_PTR(taken);
  B200Q_REQUIRE_PTR(cu_new); B200Q_REQUIRE_PTR(lens_out); B200Q_REQUIRE_PTR(taken_out); B200Q_REQUIRE_PTR(status);
  if (nfree > 0) B200Q_REQUIRE_PTR(free_pages);
  if (width > 0) B200Q_REQUIRE_PTR(table);
  if (tokens > 0) { B200Q_REQUIRE_PTR(slots); B200Q_REQUIRE_PTR(positions); }
  if (requests <= 0 || page <= 0 || tokens < 0 || nfree < 0 || width < 0 || table_stride < width) return B200Q_ERR_SHAPE;
  if (requests > kStepMaxRequests || tokens > (1 << 30)) return B200Q_ERR_UNSUPPORTED;
  const size_t smem = sizeof(int) * (3 * static_cast<size_t>(requests) + 2);
  static std::atomic<uint64_t> done;
  // the 48 KB of the default limit hold the kernel's static words too (1 KB is more than they take)
  if (smem > 47 * 1024 && !allow_smem(reinterpret_cast<const void*>(kv_step_kernel), 3 * sizeof(int) * (kStepMaxRequests + 1), done))
    return B200Q_ERR_CUDA;
  const int grid = grid_for(static_cast<int64_t>(tokens) + requests, 4 * kStepThreads, 1);
  launch_pdl(kv_step_kernel, grid, kStepThreads, smem, static_cast<cudaStream_t>(stream), lens, new_lens, free_pages, nfree,
             taken, table, table_stride, width, requests, page, tokens, slots, positions, cu_new, lens_out, taken_out, status, seen);
  return launch_status();
}

extern "C" int b200q_kv_step(const int* lens, const int* new_lens, const int* free_pages, int nfree, const int* taken,
                             int* table, int64_t table_stride, int width, int requests, int page, int tokens,
                             int64_t* slots, int* positions, int* cu_new, int* lens_out, int* taken_out, int* status,
                             void* stream) {
  return b200q_kv_step_seen(lens, new_lens, free_pages, nfree, taken, table, table_stride, width, requests, page, tokens, slots,
                            positions, cu_new, lens_out, taken_out, status, nullptr, stream);
}

extern "C" int b200q_nvfp4_kv_append(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                     int64_t v_token_stride, int64_t v_head_stride, int dtype, const int64_t* slots,
                                     int tokens, int heads, int dim, const float* k_scale2, const float* v_scale2,
                                     uint8_t* k_codes, uint8_t* k_scales, uint8_t* v_codes, uint8_t* v_scales, int pages,
                                     int page, void* k_values, void* v_values, void* stream) {
  B200Q_REQUIRE_PTR(k); B200Q_REQUIRE_PTR(v); B200Q_REQUIRE_PTR(slots); B200Q_REQUIRE_PTR(k_scale2); B200Q_REQUIRE_PTR(v_scale2);
  B200Q_REQUIRE_PTR(k_codes); B200Q_REQUIRE_PTR(k_scales); B200Q_REQUIRE_PTR(v_codes); B200Q_REQUIRE_PTR(v_scales);
  B200Q_REQUIRE_DTYPE(dtype);
  if (tokens <= 0 || heads <= 0 || dim <= 0 || dim % 16 || pages <= 0 || page <= 0) return B200Q_ERR_SHAPE;
  const int64_t nblocks = static_cast<int64_t>(tokens) * heads * (dim / 16), nslots = static_cast<int64_t>(pages) * page;
  if (nblocks > kFastDivLimit / 2 || nslots > kFastDivLimit) return B200Q_ERR_UNSUPPORTED;
  const int64_t es = dtype == B200Q_F32 ? 4 : 2;
  const uintptr_t align = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_values) |
                          reinterpret_cast<uintptr_t>(v_values) | static_cast<uintptr_t>(k_token_stride * es) |
                          static_cast<uintptr_t>(k_head_stride * es) | static_cast<uintptr_t>(v_token_stride * es) |
                          static_cast<uintptr_t>(v_head_stride * es);
  if ((align & 31u) || ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 7u)) return B200Q_ERR_ALIGN;
  const KvSide ks{k, k_token_stride, k_head_stride, k_scale2, k_codes, k_scales, k_values};
  const KvSide vs{v, v_token_stride, v_head_stride, v_scale2, v_codes, v_scales, v_values};
  const int grid = static_cast<int>((nblocks + 255) / 256);
  return B200Q_DISPATCH(dtype, [&] {
    launch_pdl(kv_append_kernel<T>, grid, 256, 0, static_cast<cudaStream_t>(stream), ks, vs, slots,
               static_cast<int>(nblocks), FastDiv(dim / 16), FastDiv(heads), FastDiv(page), nslots);
    return launch_status();
  });
}
