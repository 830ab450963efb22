// Codes of the 8-bit key/value cache as tensor-core operands, and typed rows:
// shared by the two attention kernels over it.
#pragma once

#include "kv_cache.cuh"

namespace tt {

// Codes to fp16 pairs, exact. int8: 1024 + (code + 128) is the fp16 with that
// low byte, minus 1152, so every bit pattern is a number. e4m3: one conversion
// a pair, which B200 runs at the rate of its integer operations (measured: 1.9
// a cycle and SM, against four operations to place the bits by hand); a slot
// that was never written can hold the NaN pattern, so callers zero the codes
// behind a sequence's end before they meet a probability of 0.
__device__ __forceinline__ uint32_t i8_pair(uint32_t biased, uint32_t sel) {
  uint32_t r = __byte_perm(biased, 0x64646464u, sel);
  asm("sub.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t &a, uint32_t &b) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(a), "=r"(b)
      : "r"(w));
}
// four consecutive codes -> (0, 1), (2, 3)
template <int FMT>
__device__ __forceinline__ void codes_along(uint32_t w, uint32_t &a, uint32_t &b) {
  if constexpr (FMT == TT_KV_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    a = i8_pair(u, 0x4140);
    b = i8_pair(u, 0x4342);
  } else {
    e4m3_pairs(w, a, b);
  }
}
// four codes of each of two tokens -> the pair (x, y) of each code
template <int FMT>
__device__ __forceinline__ void codes_across(uint32_t x, uint32_t y, uint32_t *r) {
  codes_along<FMT>(__byte_perm(x, y, 0x5140), r[0], r[1]);
  codes_along<FMT>(__byte_perm(x, y, 0x7362), r[2], r[3]);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A token's p is 2^(s' + e - M + c), its weight in the sum of p 2^(s' - M + c), which is
// p 2^-e as long as p is not flushed to 0 (below 2^-126). Where the value scale's exponent e
// is at least kFarScale, a flushed p has a weight below 2^(-126 + 22), and the largest
// weight is 2^(c - 64) >= 2^-57 at least (M is at most 64 above the largest s'): 2^23
// such tokens together do not reach 2^-24 of the sum. Below kFarScale (a page of zeros, or of
// magnitudes below 2^-14) the weights are computed by themselves.
constexpr float kFarScale = -22.f;

// Whether both scales of a page are as nearly all are: powers of two of the format's
// range, the values' from kFarScale on.
__device__ __forceinline__ bool usual_scales(float ks, float vs) {
  constexpr uint32_t kLow = (uint32_t)(kKvLeastExponent + 127) << 23, kTop = (uint32_t)(kKvMostExponent + 127) << 23,
                     kFar = (uint32_t)((int)kFarScale + 127) << 23;
  const uint32_t k = __float_as_uint(ks), v = __float_as_uint(vs);
  return ((k | v) & 0x807fffffu) == 0 && k - kLow <= kTop - kLow && v - kFar <= kTop - kFar;
}

// x * 2^d for a sum of weights x, which may be 2^64 and more, and a whole number d <= 0,
// minus infinity too; f is exp2_approx(d), which is flushed to 0 below 2^-126.
__device__ __forceinline__ float rescale(float x, float d, float f) {
  if (f != 0.f) return x * f;
  const int n = (int)fmaxf(d, -252.f), h = n >> 1;
  return x * kv_pow2(h) * kv_pow2(n - h);
}

// The exponent by which a row q with the largest magnitude mx is divided before its split
// into fp16 pieces: that element comes to lie in [2^14, 2^15), so that a piece's least step,
// 2^-24, is 2^-38 of it at most and one large channel takes no bits from the others.
__device__ __forceinline__ int q_exponent(float mx) {
  const int e = (__float_as_int(mx) >> 23) - 127;
  return mx > 0.f ? min(max(e, -112), 127) - 14 : 0;
}

__device__ __forceinline__ float kv_load_in(int dtype, const void *p, int64_t i) {
  if (dtype == TT_DTYPE_F32) return static_cast<const float *>(p)[i];
  if (dtype == TT_DTYPE_F16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// Four consecutive elements; i is a multiple of 4, `vec` as below.
__device__ __forceinline__ void kv_load_in4(int dtype, const void *p, int64_t i, bool vec, float *x) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = kv_load_in(dtype, p, i + k);
  } else if (dtype == TT_DTYPE_F32) {
    const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
    if (dtype == TT_DTYPE_F16) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
      x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
      x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
      x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void kv_store_out4(const KvOut &o, int64_t i, const float *x) {
  if (o.dtype == TT_DTYPE_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(o.p) + i) = make_float4(x[0], x[1], x[2], x[3]);
  } else if (o.dtype == kKvSplit) {
    uint2 h, l;
    f16_split2(x[0], x[1], h.x, l.x);
    f16_split2(x[2], x[3], h.y, l.y);
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.p) + i) = h;
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.lo) + i) = l;
  } else {
    uint2 v;
    if (o.dtype == TT_DTYPE_F16) {
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v.x) : "f"(x[1]), "f"(x[0]));
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v.y) : "f"(x[3]), "f"(x[2]));
    } else {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.x) : "f"(x[1]), "f"(x[0]));
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.y) : "f"(x[3]), "f"(x[2]));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o.p) + i) = v;
  }
}

// 16 consecutive elements from element i on; `vec`: the address is a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void load_row16(const T *p, bool vec, float *x) {
  constexpr int N = 16 * sizeof(T) / 16, E = 16 / sizeof(T);
  if (vec) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint4 raw = reinterpret_cast<const uint4 *>(p)[n];
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int i = 0; i < E; ++i) x[n * E + i] = kv_to_float(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = kv_to_float(p[i]);
  }
}
__device__ __forceinline__ void kv_load_row16(int dtype, const void *p, int64_t i, bool vec, float *x) {
  if (dtype == TT_DTYPE_F32) load_row16(static_cast<const float *>(p) + i, vec, x);
  else if (dtype == TT_DTYPE_F16) load_row16(static_cast<const __half *>(p) + i, vec, x);
  else load_row16(static_cast<const __nv_bfloat16 *>(p) + i, vec, x);
}
// 16 consecutive elements at a 16-byte-aligned address.
template <typename T>
__device__ __forceinline__ void store_row16(T *p, const float *x) {
  constexpr int N = 16 * sizeof(T) / 16, E = 16 / sizeof(T);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint4 raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < E; ++i) kv_store(e + i, x[n * E + i]);
    reinterpret_cast<uint4 *>(p)[n] = raw;
  }
}
__device__ __forceinline__ void kv_store_row16(const KvOut &o, int64_t i, const float *x) {
  if (o.dtype == TT_DTYPE_F32) {
    store_row16(static_cast<float *>(o.p) + i, x);
  } else if (o.dtype == TT_DTYPE_F16) {
    store_row16(static_cast<__half *>(o.p) + i, x);
  } else if (o.dtype == TT_DTYPE_BF16) {
    store_row16(static_cast<__nv_bfloat16 *>(o.p) + i, x);
  } else {
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f16_split2(x[2 * k], x[2 * k + 1], hi[k], lo[k]);
    uint4 *h = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(o.p) + i);
    uint4 *l = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(o.lo) + i);
    h[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]), h[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
    l[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]), l[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
  }
}

// 16 fp32 sums kept in an fp32 or split output row until its values are written
// there: their bits, in the split form as upper and lower halves.
__device__ __forceinline__ void kv_store_sum16(const KvOut &o, int64_t i, const float *x) {
  if (o.dtype == TT_DTYPE_F32) {
    store_row16(static_cast<float *>(o.p) + i, x);
    return;
  }
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    hi[k] = __byte_perm(__float_as_uint(x[2 * k]), __float_as_uint(x[2 * k + 1]), 0x7632);
    lo[k] = __byte_perm(__float_as_uint(x[2 * k]), __float_as_uint(x[2 * k + 1]), 0x5410);
  }
  uint4 *h = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(o.p) + i);
  uint4 *l = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(o.lo) + i);
  h[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]), h[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
  l[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]), l[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
}
__device__ __forceinline__ void kv_load_sum16(const KvOut &o, int64_t i, float *x) {
  if (o.dtype == TT_DTYPE_F32) {
    load_row16(static_cast<const float *>(o.p) + i, true, x);
    return;
  }
  uint4 h[2], l[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    h[k] = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(o.p) + i)[k];
    l[k] = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(o.lo) + i)[k];
  }
  const uint32_t *hw = &h[0].x, *lw = &l[0].x;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[2 * k] = __uint_as_float(__byte_perm(lw[k], hw[k], 0x5410));
    x[2 * k + 1] = __uint_as_float(__byte_perm(lw[k], hw[k], 0x7632));
  }
}

}  // namespace tt
