// The 8-bit paged key/value cache: its device view, codes and scales, and the
// launchers of its kernels (kv_cache.cu, kv_attention.cu).
//
// Format. Keys and values are held as 8-bit codes in pages of page_size tokens,
// [num_pages, kv_heads, page_size, head_dim], with one fp32 scale for each
// (page, head) of the keys and of the values: value = code * scale. A code is
// a float8 e4m3 (largest value 448) or an int8 in [-127, 127]. Every scale is a
// power of two 2^E, E >= -64: the smallest that brings the largest magnitude it
// was made from into the code's range, so quantising is one exact
// multiplication and one rounding (to nearest, ties to even), the codes do not
// hang on the order in which a division is done, and a page whose scale grows
// when later tokens are appended moves its old codes by an exponent shift and
// one more rounding. A (page, head) that was given a NaN, an infinity or a
// magnitude beyond the largest code times 2^63 has a NaN scale, reads as NaN,
// and keeps it until the page is started anew from its first slot.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "tt_common.cuh"

namespace tt {

constexpr int kKvLeastExponent = -64;  // of a scale; that of all zeros
constexpr int kKvMostExponent = 63;

// Detail codes latched with TT_ERR_DEVICE_FAULT in the cache's status word.
constexpr int kKvBadLength = 0x5100;  // lengths[b] outside [0, table_columns * page_size]
constexpr int kKvBadCount = 0x5200;   // counts[b] outside [0, min(tokens, lengths[b])]
constexpr int kKvBadPage = 0x5300;    // a block-table entry outside [0, num_pages)
constexpr int kKvBadScale = 0x5400;   // a scale that no write makes

struct KvView {
  uint8_t *k, *v;
  float *ks, *vs;
  const int32_t *table, *lengths;
  DeviceStatus *status;  // two ints: code, detail; or null
  int pages, page_log2, heads, hd, batch, columns, format;

  __device__ __forceinline__ int length(int b) const {
    const int len = lengths[b];
    const int64_t room = (int64_t)columns << page_log2;
    if (len < 0 || len > room) {
      raise_status(status, TT_ERR_DEVICE_FAULT, kKvBadLength);
      return len < 0 ? 0 : (int)room;
    }
    return len;
  }
  // new tokens of sequence b, at most `tokens` and `len`
  __device__ __forceinline__ int count(const int32_t *counts, int b, int tokens, int len) const {
    const int c = counts != nullptr ? counts[b] : tokens, most = min(tokens, len);
    if (c < 0 || c > most) {
      raise_status(status, TT_ERR_DEVICE_FAULT, kKvBadCount);
      return c < 0 ? 0 : most;
    }
    return c;
  }
  // the page that holds tokens [col * page_size, (col + 1) * page_size) of
  // sequence b; -1 (its tokens are then absent) for an entry that names none
  __device__ __forceinline__ int page_of(int b, int col) const {
    const int p = table[(int64_t)b * columns + col];
    if ((unsigned)p >= (unsigned)pages) {
      raise_status(status, TT_ERR_DEVICE_FAULT, kKvBadPage);
      return -1;
    }
    return p;
  }
  // first code of (page p, head h) in a pool
  __device__ __forceinline__ int64_t tile(int p, int h) const {
    // kv_view: num_pages * kv_heads fits 32 bits
    return (int64_t)((uint64_t)((uint32_t)p * (uint32_t)heads + (uint32_t)h) * (uint32_t)(hd << page_log2));
  }
};

// Strides of a [batch, tokens, heads, head_dim] tensor in elements; head_dim
// is contiguous.
struct KvStrides {
  int64_t batch, token, head;
};

// 2^e as a float, -126 <= e <= 127.
__device__ __forceinline__ float kv_pow2(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ float kv_to_float(float x) { return x; }
__device__ __forceinline__ float kv_to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float kv_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void kv_store(float *p, float x) { *p = x; }
__device__ __forceinline__ void kv_store(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void kv_store(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// Whether s is a scale that a write makes: a power of two within the range, or NaN; or
// the 0 of a page never written.
__device__ __forceinline__ bool kv_scale_ok(float s) {
  const uint32_t u = __float_as_uint(s), lo = (uint32_t)(kKvLeastExponent + 127) << 23,
                 hi = (uint32_t)(kKvMostExponent + 127) << 23;
  return ((u & 0x807fffffu) == 0 && u >= lo && u <= hi) || u == 0 || s != s;
}
// A scale as attention takes it, whose arithmetic needs a power of two: NaN, latched,
// in place of any that is none; the least one for a page never written.
__device__ __forceinline__ float kv_scale(float s, DeviceStatus *status) {
  if (!kv_scale_ok(s)) {
    raise_status(status, TT_ERR_DEVICE_FAULT, kKvBadScale);
    return __int_as_float(0x7fc00000);
  }
  return s == 0.f ? kv_pow2(kKvLeastExponent) : s;
}

// Four codes to fp32 values (exact).
template <int FMT>
__device__ __forceinline__ void kv_decode4(uint32_t w, float *x) {
  if constexpr (FMT == TT_KV_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    uint32_t a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
    const float2 p = __half22float2(*reinterpret_cast<__half2 *>(&a));
    const float2 q = __half22float2(*reinterpret_cast<__half2 *>(&b));
    x[0] = p.x, x[1] = p.y, x[2] = q.x, x[3] = q.y;
  }
}

// Four fp32 values within the code's range to codes, to nearest, ties to even.
template <int FMT>
__device__ __forceinline__ uint32_t kv_encode4(const float *x) {
  if constexpr (FMT == TT_KV_INT8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(uint8_t)(int8_t)__float2int_rn(x[i]) << (8 * i);
    return w;
  } else {
    uint32_t w;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(w)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]));
    return w;
  }
}

// kv_cache.cu
// The checks every entry point makes of a cache; fills *v.
int kv_view(const tt_kv_cache *c, const char *what, KvView *v);
// mask[b * tokens + i] = i < counts[b]
int launch_kv_mask(const KvView &c, const int32_t *counts, int64_t tokens, uint8_t *mask,
                   cudaStream_t stream);
int launch_kv_write(const KvView &c, int dtype, const void *k, const void *v, KvStrides ks,
                    KvStrides vs, int64_t tokens, const int32_t *counts, cudaStream_t stream);
int launch_kv_read(const KvView &c, int dtype, void *k, void *v, int64_t max_tokens,
                   cudaStream_t stream);

// Where attention writes [batch, tokens, heads, head_dim], contiguous: elements
// of a TT_DTYPE_*, or (kKvSplit) their fp16 split, the high pieces at p and the
// low ones at lo, which the split-precision out_proj reads.
constexpr int kKvSplit = -1;
struct KvOut {
  void *p, *lo;
  int dtype;
};

struct KvAttentionArgs {
  KvView c;
  const void *q;
  KvStrides qs;
  KvOut out;
  const int32_t *counts;
  float *ws;  // partial results
  int dtype, tokens, heads, group;  // dtype: of q
  float scale;
  bool q_vec;  // q's rows are 16-byte aligned
  int test_hold_back;  // set by the tile kernel's launcher (tt_test_arm_kv_wait_timeout)
};

// kv_attention.cu
// The current device's number of SMs, looked up once per device.
// Tokens of a sequence, and query rows of a key head, at most: sums of a position and
// a tile's width stay in 32 bits.
constexpr int64_t kKvMost = 1 << 30;
int kv_sm_count(int *out);
// Sets a kernel's dynamic shared memory limit once per device, and checks that it
// was built with `regs` registers a thread (0: any number).
struct KvSmemSet {
  std::atomic<bool> done[64] = {};
  int ensure(const void *kernel, size_t bytes, int regs = 0);
};
size_t kv_attention_ws_bytes(const KvView &c, int dtype, int64_t tokens, int heads);
int launch_kv_attention(const KvAttentionArgs &a, cudaStream_t stream);
// kv_attention_tc.cu
size_t kv_attention_tiles_ws_bytes(const KvView &c, int dtype, int64_t tokens, int heads);
int launch_kv_attention_tiles(const KvAttentionArgs &a, cudaStream_t stream);

}  // namespace tt
