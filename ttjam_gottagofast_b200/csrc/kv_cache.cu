// Writing new tokens into the 8-bit key/value cache and reading tokens back
// (the format: kv_cache.cuh), and the C entry points of the cache.
#include <algorithm>
#include <cmath>

#include "kv_cache.cuh"

namespace tt {
namespace {

// 16 bytes of input: 4 fp32 or 8 16-bit elements, as fp32 bits.
template <typename T>
constexpr int kPiece = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ void widen(const uint4 &raw, float *x) {
  const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
  for (int i = 0; i < kPiece<T>; ++i) x[i] = kv_to_float(e[i]);
}

// The larger of the magnitudes in `mx` and those of 16 bytes, on their bits: fp32
// words, or two 16-bit halves a word (integers order like the values; infinities
// and NaN come on top); and the bits of that maximum as fp32.
template <typename T>
__device__ __forceinline__ uint32_t magnitude(uint32_t mx, const uint4 &raw) {
  const uint32_t *w = &raw.x;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    mx = sizeof(T) == 4 ? max(mx, w[i] & 0x7fffffffu) : __vmaxu2(mx, w[i] & 0x7fff7fffu);
  return mx;
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t mx) {
  if constexpr (sizeof(T) == 4) return mx;
  const uint16_t h = (uint16_t)max(mx & 0xffffu, mx >> 16);
  return __float_as_uint(kv_to_float(*reinterpret_cast<const T *>(&h))) & 0x7fffffffu;
}

// NW warps for each item: (sequence, page that new tokens of it land in, head, keys
// or values). The item's pieces of 16 bytes stay in registers between the maximum
// and the rounding, so each new element is read once, every load of a warp is 512
// consecutive bytes, and an item of one warp meets no barrier. (One block of 256
// threads an item, with 32 bytes a thread: 65 us for 16 prompts of 2048 tokens, 16
// heads of 64, bf16; this form 43.5 us, of which the bytes need 30.7 at the rate of a
// plain copy.) The maximum is taken on the bits of |x| (ordered like the
// values; infinities and NaN on top), so it does not hang on the order of the
// reduction. Bound by memory for prompts, by its dependent loads (length, page,
// scale) for a step.
constexpr int block_warps(int nw) { return nw < 4 ? 4 : nw; }

template <typename T, int FMT, int NW, int NC>
__global__ void __launch_bounds__(32 * block_warps(NW))
    kv_write_kernel(KvView c, const T *k, const T *v, KvStrides kst, KvStrides vst, int tokens,
                    const int32_t *counts, int touched, unsigned items, bool vec) {
  constexpr int E = kPiece<T>, LANES = 32 * NW;
  __shared__ uint32_t s_max[block_warps(NW)];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = NW == 1 ? threadIdx.x & 31 : threadIdx.x % LANES;
  unsigned item = blockIdx.x * (block_warps(NW) / NW) + warp / NW;
  const bool any = item < items;
  if (NW == 1 && !any) return;
  if (!any) item = items - 1;  // to the barrier with the others, and nothing written
  const int h = item % c.heads;
  item /= c.heads;
  const bool is_v = item & 1;
  item >>= 1;
  const int b = item / touched, j = item % touched;
  pdl_wait();
  const int len = c.length(b), count = c.count(counts, b, tokens, len);
  const int start = len - count, page = 1 << c.page_log2;
  const int col = (start >> c.page_log2) + j;
  const int lo = max(start, col << c.page_log2), hi = min(len, (col + 1) << c.page_log2);
  // no new token of this sequence in that page, or a page that does not exist
  const int pg = any && lo < hi ? c.page_of(b, col) : -1;
  if (NW == 1 && pg < 0) return;
  const KvStrides st = is_v ? vst : kst;
  const T *src = (is_v ? v : k) + b * st.batch + h * st.head + (int64_t)(lo - start) * st.token;
  const int row = c.hd / E, pieces = pg >= 0 ? (hi - lo) * row : 0;  // pieces of a token, in all

  uint4 raw[NC];
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int i = u * LANES + lane;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (i < pieces) {
      const int t = i / row, d = (i - t * row) * E;
      const T *p = src + t * st.token + d;
      if (vec) {
        raw[u] = __ldcs(reinterpret_cast<const uint4 *>(p));
      } else {
        T *e = reinterpret_cast<T *>(&raw[u]);
#pragma unroll
        for (int q = 0; q < E; ++q) e[q] = p[q];
      }
    }
  }
  const int slot = lo & (page - 1);  // tokens the page held before
  float *scale_p = (is_v ? c.vs : c.ks) + (int64_t)max(pg, 0) * c.heads + h;
  const float old = pg >= 0 && slot > 0 ? *scale_p : 0.f;
  uint32_t mx = 0;
#pragma unroll
  for (int u = 0; u < NC; ++u) mx = magnitude<T>(mx, raw[u]);
  mx = __reduce_max_sync(0xffffffffu, magnitude_bits<T>(mx));
  if constexpr (NW > 1) {
    if ((threadIdx.x & 31) == 0) s_max[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = max(mx, s_max[warp / NW * NW + w]);
    if (pg < 0) return;
  }
  // the exponent: |x| = 1.m * 2^e; 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr int TOP_E = FMT == TT_KV_INT8 ? 6 : 8;
  constexpr uint32_t TOP_M = FMT == TT_KV_INT8 ? 0x7e0000u : 0x600000u;
  int e = (int)(mx >> 23) - 127 - TOP_E + ((mx & 0x7fffffu) > TOP_M);
  const bool odd = !kv_scale_ok(old);  // its codes cannot be moved exactly
  if (odd && lane == 0) raise_status(c.status, TT_ERR_DEVICE_FAULT, kKvBadScale);
  const bool bad = mx >= 0x7f800000u || e > kKvMostExponent || !(old == old) || odd;
  e = max(e, kKvLeastExponent);
  float scale = kv_pow2(bad ? 0 : e);
  if (!bad) scale = fmaxf(scale, old);
  const float inv = 1.f / scale;  // a power of two: exact
  uint8_t *dst = (is_v ? c.v : c.k) + c.tile(pg, h);
  if (lane == 0) *scale_p = bad ? __int_as_float(0x7fc00000) : scale;
  if (slot > 0 && !bad && scale != old) {
    // the page's scale grew: its old codes move to the new one
    const float ratio = old * inv;
    for (int i = lane; i < slot * (c.hd >> 4); i += LANES) {
      uint4 w = reinterpret_cast<uint4 *>(dst)[i];
      uint32_t *ww = &w.x;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float y[4];
        kv_decode4<FMT>(ww[q], y);
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] *= ratio;
        ww[q] = kv_encode4<FMT>(y);
      }
      reinterpret_cast<uint4 *>(dst)[i] = w;
    }
  }
  uint32_t *out = reinterpret_cast<uint32_t *>(dst + slot * c.hd);
#pragma unroll
  for (int u = 0; u < NC; ++u) {
    const int i = u * LANES + lane;
    if (i >= pieces) break;
    float x[E];
    widen<T>(raw[u], x);
    uint32_t w[E / 4];
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = bad ? 0.f : x[4 * q + r] * inv;
      w[q] = kv_encode4<FMT>(y);
    }
    if constexpr (E == 8) reinterpret_cast<uint2 *>(out)[i] = make_uint2(w[0], w[1]);
    else out[i] = w[0];
  }
}

// A thread takes 16 bytes of output in each of kReadRows rows ((token, head) pairs),
// whose loads it has under way at once; x runs along a row, so every store of a warp
// covers consecutive bytes. Rows behind a sequence's end, and of pages that do not
// exist, are zero. Bound by memory: one sequence of 100000 tokens, 16 heads of 64, to
// bf16, 96 to 102 us, 6.0 to 6.4 TB/s (one row a thread: 119 us).
constexpr int kReadRows = 4;

template <typename T, int FMT>
__global__ void __launch_bounds__(256) kv_read_kernel(KvView c, T *k, T *v, uint32_t rows) {
  constexpr int E = kPiece<T>;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, d = threadIdx.x * E;
  const uint32_t r0 = (blockIdx.x * kReadRows) * blockDim.y + threadIdx.y;
  const int len = c.length(b);
  const uint8_t *pool = blockIdx.z ? c.v : c.k;
  const float *scales = blockIdx.z ? c.vs : c.ks;
  uint2 w[kReadRows];
  float s[kReadRows];
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const uint32_t r = r0 + u * blockDim.y;
    const int t = r / c.heads, h = r - t * c.heads;
    w[u] = make_uint2(0, 0);
    s[u] = 0.f;
    if (r < rows && t < len) {
      const int pg = c.page_of(b, t >> c.page_log2);
      if (pg >= 0) {
        const uint8_t *p = pool + c.tile(pg, h) + (t & ((1 << c.page_log2) - 1)) * c.hd + d;
        if constexpr (E == 8) w[u] = __ldcs(reinterpret_cast<const uint2 *>(p));
        else w[u].x = __ldcs(reinterpret_cast<const uint32_t *>(p));
        s[u] = scales[(int64_t)pg * c.heads + h];
      }
    }
  }
  T *out = (blockIdx.z ? v : k) + (int64_t)b * rows * c.hd + d;
#pragma unroll
  for (int u = 0; u < kReadRows; ++u) {
    const uint32_t r = r0 + u * blockDim.y;
    if (r >= rows) break;
    float x[8];
    kv_decode4<FMT>(w[u].x, x);
    if constexpr (E == 8) kv_decode4<FMT>(w[u].y, x + 4);
    uint4 raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int q = 0; q < E; ++q) kv_store(e + q, x[q] * s[u]);
    __stcs(reinterpret_cast<uint4 *>(out + (int64_t)r * c.hd), raw);
  }
}

__global__ void __launch_bounds__(256) kv_mask_kernel(KvView c, const int32_t *counts, int tokens,
                                                      uint8_t *mask) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  const int count = c.count(counts, b, tokens, c.length(b));
  if (i < tokens) mask[(int64_t)b * tokens + i] = i < count;
}

bool vec_ok(const void *p, const KvStrides &s, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (s.batch * size) % 16 == 0 &&
         (s.token * size) % 16 == 0 && (s.head * size) % 16 == 0;
}

template <typename T, int FMT, int NW, int NC>
int write_nc(const KvView &c, const void *k, const void *v, KvStrides ks, KvStrides vs,
             int tokens, const int32_t *counts, int touched, unsigned items,
             cudaStream_t stream) {
  const bool vec = vec_ok(k, ks, sizeof(T)) && vec_ok(v, vs, sizeof(T));
  constexpr int per_block = block_warps(NW) / NW;
  TT_CUDA_TRY(launch_kernel(kv_write_kernel<T, FMT, NW, NC>, dim3((items + per_block - 1) / per_block),
                            dim3(32 * block_warps(NW)), 0, stream, 1, c, static_cast<const T *>(k),
                            static_cast<const T *>(v), ks, vs, tokens, counts, touched, items, vec));
  return TT_OK;
}

template <typename T, int FMT>
int write_typed(const KvView &c, const void *k, const void *v, KvStrides ks, KvStrides vs,
                int tokens, const int32_t *counts, cudaStream_t stream) {
  const int page = 1 << c.page_log2;
  const int touched = (tokens + page - 2) / page + 1;  // pages that `tokens` in a row can touch
  const int64_t items = (int64_t)2 * c.heads * touched * c.batch;
  if (items > INT32_MAX) return fail(TT_ERR_UNSUPPORTED, "tt_kv_write: too many tokens");
  const int pieces = std::min(tokens, page) * (c.hd / kPiece<T>);  // of 16 bytes, in one page
#define TT_KV_WRITE(NW, NC) \
  return write_nc<T, FMT, NW, NC>(c, k, v, ks, vs, tokens, counts, touched, (unsigned)items, stream)
  if (pieces <= 32) TT_KV_WRITE(1, 1);
  if (pieces <= 128) TT_KV_WRITE(1, 4);
  if (pieces <= 512) TT_KV_WRITE(1, 16);
  if (pieces <= 1024) TT_KV_WRITE(2, 16);
  if (pieces <= 2048) TT_KV_WRITE(4, 16);
  if (pieces <= 4096) TT_KV_WRITE(8, 16);
  TT_KV_WRITE(16, 16);  // 128 tokens of 256 fp32 elements, the largest page
#undef TT_KV_WRITE
}

}  // namespace

int launch_kv_write(const KvView &c, int dtype, const void *k, const void *v, KvStrides ks,
                    KvStrides vs, int64_t tokens, const int32_t *counts, cudaStream_t stream) {
  const bool i8 = c.format == TT_KV_INT8;
  const int n = (int)tokens;
  switch (dtype) {
    case TT_DTYPE_F32:
      return i8 ? write_typed<float, TT_KV_INT8>(c, k, v, ks, vs, n, counts, stream)
                : write_typed<float, TT_KV_E4M3>(c, k, v, ks, vs, n, counts, stream);
    case TT_DTYPE_F16:
      return i8 ? write_typed<__half, TT_KV_INT8>(c, k, v, ks, vs, n, counts, stream)
                : write_typed<__half, TT_KV_E4M3>(c, k, v, ks, vs, n, counts, stream);
    default:
      return i8 ? write_typed<__nv_bfloat16, TT_KV_INT8>(c, k, v, ks, vs, n, counts, stream)
                : write_typed<__nv_bfloat16, TT_KV_E4M3>(c, k, v, ks, vs, n, counts, stream);
  }
}

int launch_kv_mask(const KvView &c, const int32_t *counts, int64_t tokens, uint8_t *mask,
                   cudaStream_t stream) {
  TT_CUDA_TRY(launch_kernel(kv_mask_kernel, dim3((unsigned)ceil_div(tokens, 256), c.batch), dim3(256),
                            0, stream, 1, c, counts, (int)tokens, mask));
  return TT_OK;
}

template <typename T>
static int read_typed(const KvView &c, void *k, void *v, int64_t max_tokens, cudaStream_t stream) {
  const int64_t rows = max_tokens * c.heads;
  if (rows > INT32_MAX || c.batch > 65535)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_read: too many tokens or sequences");
  auto *kern = c.format == TT_KV_INT8 ? kv_read_kernel<T, TT_KV_INT8> : kv_read_kernel<T, TT_KV_E4M3>;
  const unsigned x = c.hd / kPiece<T>, y = 256 / x;
  TT_CUDA_TRY(launch_kernel(kern, dim3((unsigned)ceil_div(rows, y * kReadRows), c.batch, 2), dim3(x, y), 0,
                            stream, 1, c, static_cast<T *>(k), static_cast<T *>(v), (uint32_t)rows));
  return TT_OK;
}

int launch_kv_read(const KvView &c, int dtype, void *k, void *v, int64_t max_tokens,
                   cudaStream_t stream) {
  switch (dtype) {
    case TT_DTYPE_F32: return read_typed<float>(c, k, v, max_tokens, stream);
    case TT_DTYPE_F16: return read_typed<__half>(c, k, v, max_tokens, stream);
    default: return read_typed<__nv_bfloat16>(c, k, v, max_tokens, stream);
  }
}

int kv_view(const tt_kv_cache *c, const char *what, KvView *v) {
  auto no = [&](int code, const std::string &m) { return fail(code, std::string(what) + ": " + m); };
  if (c == nullptr) return no(TT_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (c->format != TT_KV_E4M3 && c->format != TT_KV_INT8)
    return no(TT_ERR_INVALID_ARGUMENT, "format must be TT_KV_E4M3 or TT_KV_INT8");
  if (c->reserved != 0) return no(TT_ERR_INVALID_ARGUMENT, "reserved field must be 0");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return no(TT_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16 != 0)
    return no(TT_ERR_UNSUPPORTED, "head_dim must be a multiple of 16, at most 256");
  if (c->kv_heads <= 0 || c->num_pages <= 0 || c->batch < 0 || c->table_columns <= 0)
    return no(TT_ERR_INVALID_ARGUMENT, "kv_heads, num_pages and table_columns must be positive");
  if ((int64_t)c->num_pages * c->kv_heads > INT32_MAX)
    return no(TT_ERR_UNSUPPORTED, "num_pages * kv_heads must fit 32 bits");
  if ((int64_t)c->table_columns * c->page_size > kKvMost)
    return no(TT_ERR_UNSUPPORTED, "table_columns * page_size must be at most 2^30");
  if (c->batch > 0 && (c->k_codes == nullptr || c->v_codes == nullptr || c->k_scale == nullptr ||
                       c->v_scale == nullptr || c->block_table == nullptr || c->lengths == nullptr))
    return no(TT_ERR_INVALID_ARGUMENT, "a cache pointer is NULL");
  if (((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15) ||
      ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) |
        reinterpret_cast<uintptr_t>(c->block_table) | reinterpret_cast<uintptr_t>(c->lengths) |
        reinterpret_cast<uintptr_t>(c->status)) & 3))
    return no(TT_ERR_INVALID_ARGUMENT, "a cache pointer is misaligned (codes: 16 bytes)");
  v->k = static_cast<uint8_t *>(c->k_codes);
  v->v = static_cast<uint8_t *>(c->v_codes);
  v->ks = c->k_scale;
  v->vs = c->v_scale;
  v->table = c->block_table;
  v->lengths = c->lengths;
  v->status = reinterpret_cast<DeviceStatus *>(c->status);
  v->pages = c->num_pages;
  v->page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  v->heads = c->kv_heads;
  v->hd = c->head_dim;
  v->batch = c->batch;
  v->columns = c->table_columns;
  v->format = c->format;
  return TT_OK;
}

static bool dtype_ok(int dtype) {
  return dtype == TT_DTYPE_F32 || dtype == TT_DTYPE_F16 || dtype == TT_DTYPE_BF16;
}

}  // namespace tt

using namespace tt;

extern "C" {

int tt_kv_write(const tt_kv_cache *cache, int dtype, const void *k, const void *v,
                const int64_t *k_strides, const int64_t *v_strides, int64_t tokens,
                const int32_t *counts, void *stream) {
  KvView c;
  const int rc = kv_view(cache, "tt_kv_write", &c);
  if (rc != TT_OK) return rc;
  if (!dtype_ok(dtype))
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_write: dtype must be a TT_DTYPE_* value");
  if (tokens < 0 || tokens > INT32_MAX)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_write: tokens must be >= 0 and fit 32 bits");
  if (tokens == 0 || c.batch == 0) return TT_OK;
  if (k == nullptr || v == nullptr || k_strides == nullptr || v_strides == nullptr)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_write: NULL k, v or strides");
  const int64_t room = (int64_t)c.columns << c.page_log2;
  if (counts == nullptr && tokens > room)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_write: more tokens than a sequence has room for");
  tokens = std::min(tokens, room);  // rows behind those are behind every count
  return launch_kv_write(c, dtype, k, v, {k_strides[0], k_strides[1], k_strides[2]},
                         {v_strides[0], v_strides[1], v_strides[2]}, tokens, counts,
                         static_cast<cudaStream_t>(stream));
}

int tt_kv_read(const tt_kv_cache *cache, int dtype, void *k, void *v, int64_t max_tokens,
               void *stream) {
  KvView c;
  const int rc = kv_view(cache, "tt_kv_read", &c);
  if (rc != TT_OK) return rc;
  if (!dtype_ok(dtype))
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_read: dtype must be a TT_DTYPE_* value");
  if (max_tokens < 0 || max_tokens > kKvMost)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_read: max_tokens must be >= 0 and at most 2^30");
  if (max_tokens == 0 || c.batch == 0) return TT_OK;
  if (k == nullptr || v == nullptr)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_read: NULL k or v");
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_read: k and v must be 16-byte aligned");
  return launch_kv_read(c, dtype, k, v, max_tokens, static_cast<cudaStream_t>(stream));
}

size_t tt_kv_attention_typed_workspace_bytes(const tt_kv_cache *cache, int dtype, int64_t tokens,
                                             int32_t heads) {
  KvView c;
  if (kv_view(cache, "tt_kv_attention_workspace_bytes", &c) != TT_OK || !dtype_ok(dtype)) return 0;
  if (tokens <= 0 || tokens > INT32_MAX || c.batch == 0 || heads <= 0 || heads % c.heads != 0 ||
      tokens * (heads / c.heads) > kKvMost)
    return 0;
  return kv_attention_ws_bytes(c, dtype, tokens, heads);
}

size_t tt_kv_attention_workspace_bytes(const tt_kv_cache *cache, int64_t tokens, int32_t heads) {
  // float16 rows need the most
  return tt_kv_attention_typed_workspace_bytes(cache, TT_DTYPE_F16, tokens, heads);
}

int tt_kv_attention(const tt_kv_cache *cache, int dtype, const void *q, const int64_t *q_strides,
                    int64_t tokens, int32_t heads, const int32_t *counts, float scale, void *out,
                    void *workspace, size_t workspace_bytes, void *stream) {
  KvView c;
  const int rc = kv_view(cache, "tt_kv_attention", &c);
  if (rc != TT_OK) return rc;
  if (!dtype_ok(dtype))
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: dtype must be a TT_DTYPE_* value");
  if (tokens < 0 || tokens > INT32_MAX)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: tokens must be >= 0 and fit 32 bits");
  if (heads <= 0 || heads % c.heads != 0)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: heads must be a multiple of kv_heads");
  if (tokens * (heads / c.heads) > kKvMost)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_attention: more than 2^30 rows a key head");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: scale must be positive and finite");
  if (tokens == 0 || c.batch == 0) return TT_OK;
  if (q == nullptr || q_strides == nullptr || out == nullptr)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: NULL q, strides or out");
  if (q == out) return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: out may not alias q");
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_attention: out and workspace must be 16-byte aligned");
  const size_t need = kv_attention_ws_bytes(c, dtype, tokens, heads);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return fail(TT_ERR_WORKSPACE, "tt_kv_attention: workspace smaller than "
                                  "tt_kv_attention_workspace_bytes (" + std::to_string(need) + " bytes)");
  KvAttentionArgs a{};
  a.c = c;
  a.q = q;
  a.qs = {q_strides[0], q_strides[1], q_strides[2]};
  a.out = {out, nullptr, dtype};
  a.counts = counts;
  a.ws = static_cast<float *>(workspace);
  a.dtype = dtype;
  a.tokens = (int)tokens;
  a.heads = heads;
  a.group = heads / c.heads;
  a.scale = scale;
  a.q_vec = vec_ok(q, a.qs, dtype == TT_DTYPE_F32 ? 4 : 2);
  return launch_kv_attention(a, static_cast<cudaStream_t>(stream));
}

int tt_kv_read_status(const tt_kv_cache *cache, int32_t *code, int32_t *detail, void *stream_) {
  if (cache == nullptr || cache->status == nullptr || code == nullptr)
    return fail(TT_ERR_INVALID_ARGUMENT, "tt_kv_read_status: NULL cache, status or code");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int32_t st[2] = {0, 0};
  TT_CUDA_TRY(cudaMemcpyAsync(st, cache->status, sizeof st, cudaMemcpyDeviceToHost, stream));
  TT_CUDA_TRY(cudaStreamSynchronize(stream));
  TT_CUDA_TRY(cudaMemsetAsync(cache->status, 0, sizeof st, stream));
  *code = st[0];
  if (detail) *detail = st[1];
  return TT_OK;
}

}  // extern "C"
