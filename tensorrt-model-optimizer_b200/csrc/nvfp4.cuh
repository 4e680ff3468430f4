// One 16-element NVFP4 block in registers: 256-bit access, abs-max, the two-level scale, encoding to
// E2M1 codes and decoding, shared by the tensor kernels and the KV-cache kernels.
#pragma once
#include "numerics.cuh"

namespace b200q {

struct u32x8 { uint32_t w[8]; };

__device__ __forceinline__ u32x8 ld256_stream(const void* p) {
  u32x8 v;
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]),
                 "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
  return v;
}
// same, asking L2 to keep the line: the quantise pass reads the tensor again right after
__device__ __forceinline__ u32x8 ld256_keep(const void* p) {
  u32x8 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::evict_last.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]),
                 "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p));
  return v;
}
__device__ __forceinline__ void st256_stream(void* p, const u32x8& v) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v.w[0]),
               "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]),
               "r"(v.w[7])
               : "memory");
}

// Raw storage of one 16-element block and its decoding.
template <typename T> struct Block16;
template <> struct Block16<float> {
  u32x8 a, b;
  __device__ __forceinline__ void load(const float* p) { a = ld256_stream(p); b = ld256_stream(p + 8); }
  __device__ __forceinline__ void load_keep(const float* p) { a = ld256_keep(p); b = ld256_keep(p + 8); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.w[i] = b.w[i] = 0;
  }
  __device__ __forceinline__ uint32_t amax_f32bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, max(a.w[i] & 0x7fffffffu, b.w[i] & 0x7fffffffu));
    return m;
  }
  __device__ __forceinline__ void decode(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) { f[i] = __uint_as_float(a.w[i]); f[8 + i] = __uint_as_float(b.w[i]); }
  }
};
template <> struct Block16<__nv_bfloat16> {
  u32x8 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = ld256_stream(p); }
  __device__ __forceinline__ void load_keep(const __nv_bfloat16* p) { a = ld256_keep(p); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.w[i] = 0;
  }
  __device__ __forceinline__ uint32_t amax_f32bits() const {
#ifdef B200Q_NV_HMAX
    // |x| max as packed bf16 arithmetic (NaN-propagating), tree of 7 ops
    __nv_bfloat162 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&a.w[i]));
#pragma unroll
    for (int s = 4; s > 0; s >>= 1)
#pragma unroll
      for (int i = 0; i < s; ++i) v[i] = __hmax2_nan(v[i], v[i + s]);
    const uint32_t m = *reinterpret_cast<uint32_t*>(&v[0]);
#else
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, a.w[i] & 0x7fff7fffu);
#endif
    return max(m & 0xffffu, m >> 16) << 16;
  }
  __device__ __forceinline__ void decode(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[2 * i] = __uint_as_float(a.w[i] << 16);
      f[2 * i + 1] = __uint_as_float(a.w[i] & 0xffff0000u);
    }
  }
};
template <> struct Block16<__half> {
  u32x8 a;
  __device__ __forceinline__ void load(const __half* p) { a = ld256_stream(p); }
  __device__ __forceinline__ void load_keep(const __half* p) { a = ld256_keep(p); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.w[i] = 0;
  }
  __device__ __forceinline__ uint32_t amax_f32bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __vmaxu2(m, a.w[i] & 0x7fff7fffu);
    uint16_t h = static_cast<uint16_t>(max(m & 0xffffu, m >> 16));
    return __float_as_uint(__half2float(__ushort_as_half(h)));
  }
  __device__ __forceinline__ void decode(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 t = __half22float2(*reinterpret_cast<const __half2*>(&a.w[i]));
      f[2 * i] = t.x; f[2 * i + 1] = t.y;
    }
  }
};

// ---- per-block arithmetic ----------------------------------------------------------------------
// Correctly rounded a/d for two lanes at once, given y = RN(1/d) and nd = -d.  The first product
// is within 1.5 ulp of the quotient; one residual correction makes it faithful and, by Markstein's
// theorem (y correctly rounded, quotient faithful, residual exact in an FMA), the second correction
// rounds to RN(a/d).  Callers guarantee d, a/d in the normal range with no overflow.  A zero
// numerator of either sign comes out as +0 ((+0) + (-0) = +0 in the corrections).
__device__ __forceinline__ float2 div2_rn(float2 a, float2 nd, float2 y) {
  float2 q = __fmul2_rn(a, y);
  float2 e = __ffma2_rn(q, nd, a);
  q = __ffma2_rn(e, y, q);
  e = __ffma2_rn(q, nd, a);
  return __ffma2_rn(e, y, q);
}
__device__ __forceinline__ float div1_rn(float a, float d, float y) {
  float q = a * y;
  float e = fmaf(-q, d, a);
  q = fmaf(e, y, q);
  e = fmaf(-q, d, a);
  return fmaf(e, y, q);
}

constexpr float kTwoP60 = 1152921504606846976.f;        // 2^60
constexpr float kTwoM60 = 8.673617379884035e-19f;       // 2^-60

// Per-tensor constants of the two-level scaling.
struct Nvfp4Tensor {
  float s2;    // weights_scaling_factor_2
  float c;     // 6 * s2
  float rc;    // RN(1/c) when c is in the safe range
  bool c_ok;
  __device__ __forceinline__ explicit Nvfp4Tensor(float s2_) : s2(s2_) {
    c = 6.f * s2;
    c_ok = c >= kTwoM60 && c <= kTwoP60;
    rc = __frcp_rn(c);
  }
};

// block scale code from the block abs-max: t = bamax/c (IEEE quotient), 0 -> 1, cast to E4M3
template <bool kTorchCast>
__device__ __forceinline__ uint32_t nvfp4_scale_code(float bamax, const Nvfp4Tensor& tn) {
  float t;
  if (tn.c_ok && (bamax == 0.f || (bamax >= kTwoM60 && bamax <= kTwoP60)))
    t = div1_rn(bamax, tn.c, tn.rc);
  else
    t = __fdiv_rn(bamax, tn.c);
  if (t == 0.f) t = 1.f;
  return kTorchCast ? f32_to_e4m3_torch(t) : f32_to_e4m3_sat(t);
}

// 16 values -> 8 bytes of E2M1 codes under divisor d = float(block scale) * s2.
// Fast path (16-bit inputs, divisor and block abs-max in a safe range — every ordinary block):
// quotients through div2_rn with one reciprocal per block.  Otherwise the IEEE division per
// element, with +0 added so that a negative-zero quotient does not set the sign bit.
template <bool kAllowFast>
__device__ __forceinline__ uint2 nvfp4_encode16(const float* f, float d, float bamax) {
  uint32_t w[2];
  if (kAllowFast && d >= kTwoM60 && d <= 65536.f && bamax <= kTwoP60) {
    const float r = __frcp_rn(d);
    const float2 y = make_float2(r, r), nd = make_float2(-d, -d);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float2 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q[j] = div2_rn(make_float2(f[8 * h + 2 * j], f[8 * h + 2 * j + 1]), nd, y);
      w[h] = f32x8_to_e2m1x8(q[0], q[1], q[2], q[3]);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t acc = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = __fdiv_rn(f[8 * h + 2 * j], d) + 0.f;
        const float o = __fdiv_rn(f[8 * h + 2 * j + 1], d) + 0.f;
        acc |= f32x2_to_e2m1x2(e, o) << (8 * j);
      }
      w[h] = acc;
    }
  }
  return make_uint2(w[0], w[1]);
}

// 8 bytes of codes -> 16 values times d.  The hardware conversion gives -0 for the negative-zero
// code; the fused multiply-add with +0 turns the product into +0 as the reference's table has it.
__device__ __forceinline__ void nvfp4_decode16(uint2 codes, float d, float* f) {
  const uint32_t w[2] = {codes.x, codes.y};
  const float2 dd = make_float2(d, d), zz = make_float2(0.f, 0.f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2_raw hr = __nv_cvt_fp4x2_to_halfraw2(
          static_cast<__nv_fp4x2_storage_t>((w[h] >> (8 * j)) & 0xffu), __NV_E2M1);
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hr));
      const float2 r = __ffma2_rn(v, dd, zz);
      f[8 * h + 2 * j] = r.x;
      f[8 * h + 2 * j + 1] = r.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ void store16(T* y, const float* f);
template <> __device__ __forceinline__ void store16<float>(float* y, const float* f) {
  u32x8 a, b;
#pragma unroll
  for (int i = 0; i < 8; ++i) { a.w[i] = __float_as_uint(f[i]); b.w[i] = __float_as_uint(f[8 + i]); }
  st256_stream(y, a); st256_stream(y + 8, b);
}
template <> __device__ __forceinline__ void store16<__nv_bfloat16>(__nv_bfloat16* y, const float* f) {
  u32x8 a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a.w[i] = Elem<__nv_bfloat16>::pack2(f[2 * i], f[2 * i + 1]);
  st256_stream(y, a);
}
template <> __device__ __forceinline__ void store16<__half>(__half* y, const float* f) {
  u32x8 a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a.w[i] = Elem<__half>::pack2(f[2 * i], f[2 * i + 1]);
  st256_stream(y, a);
}

}  // namespace b200q
