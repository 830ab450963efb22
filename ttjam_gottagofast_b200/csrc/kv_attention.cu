// Causal attention of new tokens over the 8-bit paged key/value cache, for few
// query rows (the format: kv_cache.cuh).
//
// For row r (query head h of new token i) at position pos, key head g = h / group:
//   s_j = scale * q . k_j for j <= pos,  k_j = code_j * ks[page of j]
//   out = sum_j 2^(s'_j - M) v_j / sum_j 2^(s'_j - M),  s' = s * log2 e,
// one pass over the tokens with a running reference M. The scales never touch a
// code: ks multiplies the score, and vs = 2^e joins the exponent,
//   p_j = 2^(s'_j + e - M),  out = sum p_j code_j / sum p_j 2^-e,
// with M the running maximum of s' + e rounded up to a whole number, so that
// e - M and every rescaling by 2^(M_old - M_new) are exact.
//
// A block of 8 query rows of one key head is one m16n8k16 tensor-core operand:
// q and p are split into two fp16 pieces (22 significant bits, as the forward's
// split-precision schedule), the high pieces in operand rows 0-7, the low ones
// in rows 8-15, whose products meet in one thread's accumulators. So a step of
// one token has fp32 accuracy at the cost of one product, and the codes, exact
// in fp16, are the other operand. Row q is scaled by a power of two to have its
// largest element in [1, 2), p by 2^14 to stay clear of the fp16 subnormals.
//
// A warp takes 16 tokens at a time, straight from global memory into operand
// registers: the tokens and head dims are numbered within a step so that a
// thread's operand elements are consecutive bytes (which token or dim stands at
// which operand index is free as long as both operands agree).
//
// Work is split into units of kUnit tokens of one (sequence, key head, row block);
// every CTA takes an equal run of consecutive units, whatever the lengths, and a
// second kernel joins the (sequence, head) runs that ended up on several CTAs.
#include <math_constants.h>

#include <algorithm>

#include "kv_cache.cuh"
#include "kv_codes.cuh"

namespace tt {
namespace {

constexpr int kRows = 8;     // query rows per block
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

template <int HD>
struct RowShape {
  static constexpr int GR = HD <= 64 ? 2 : 1;        // 16-token groups per warp step
  static constexpr int kStep = 16 * GR;              // tokens per warp step
  static constexpr int kUnit = kStep * kWarps;       // tokens per unit
  // tensor cores add by rounding toward zero: after 1024 tokens the sum moves to
  // shared memory, so that it does not drift
  static constexpr int kFlush = 1024 / kStep;
  static constexpr int KW = HD / 16;                 // words of a token's keys per thread
  static constexpr int VW = HD / 32;                 // words of a token's values per thread
  static constexpr int kSlot = kRows * HD + 2 * kRows;  // floats of a partial result
};

__device__ __forceinline__ void mma16816(float *c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Units of sequence b for one (key head, row block): at least one, which writes
// the zeros of a sequence that has no new token.
__device__ __forceinline__ int units_of(const KvAttentionArgs &a, int b, int unit, int &len,
                                        int &count) {
  len = a.c.length(b);
  count = a.c.count(a.counts, b, a.tokens, len);
  return count > 0 ? (len + unit - 1) / unit : 1;
}

// What one warp knows of 16 tokens of its step, loaded ahead.
template <int HD>
struct Group {
  uint32_t k[2][RowShape<HD>::KW];
  uint32_t v[2][2][RowShape<HD>::VW];  // [operand half][token parity]
  float ks, vs;
};

template <int HD>
__device__ __forceinline__ void load_group(Group<HD> &g, const KvView &c, int pg, int h, int t0,
                                           int lane) {
  constexpr int KW = RowShape<HD>::KW, VW = RowShape<HD>::VW;
  const int gid = lane >> 2, tig = lane & 3;
  if (pg < 0) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int i = 0; i < KW; ++i) g.k[x][i] = 0;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < VW; ++i) g.v[x][p][i] = 0;
    }
    g.ks = g.vs = 1.f;
    return;
  }
  const int64_t tile = c.tile(pg, h) + (int64_t)(t0 & ((1 << c.page_log2) - 1)) * c.hd;
  g.ks = c.ks[(int64_t)pg * c.heads + h];
  g.vs = c.vs[(int64_t)pg * c.heads + h];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    // operand column n of half x is token 8 x + 4 (n & 1) + (n >> 1) of the group
    const uint8_t *row = c.k + tile + (8 * x + 4 * (gid & 1) + (gid >> 1)) * c.hd;
    if constexpr (HD == 32) {
      uint2 w = make_uint2(0, 0);
      if (8 * tig < c.hd) w = __ldcs(reinterpret_cast<const uint2 *>(row + 8 * tig));
      g.k[x][0] = w.x, g.k[x][1] = w.y;
    } else {
#pragma unroll
      for (int j = 0; j < HD / 64; ++j) {
        const int d = 64 * j + 16 * tig;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (d < c.hd) w = __ldcs(reinterpret_cast<const uint4 *>(row + d));
        g.k[x][4 * j] = w.x, g.k[x][4 * j + 1] = w.y;
        g.k[x][4 * j + 2] = w.z, g.k[x][4 * j + 3] = w.w;
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint8_t *vrow = c.v + tile + (8 * x + 4 * p + tig) * c.hd;
      if constexpr (HD == 32) {
        g.v[x][p][0] = 4 * gid < c.hd ? __ldcs(reinterpret_cast<const uint32_t *>(vrow + 4 * gid)) : 0;
      } else if constexpr (HD == 64) {
        uint2 w = make_uint2(0, 0);
        if (8 * gid < c.hd) w = __ldcs(reinterpret_cast<const uint2 *>(vrow + 8 * gid));
        g.v[x][p][0] = w.x, g.v[x][p][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < HD / 128; ++j) {
          const int d = 128 * j + 16 * gid;
          uint4 w = make_uint4(0, 0, 0, 0);
          if (d < c.hd) w = __ldcs(reinterpret_cast<const uint4 *>(vrow + d));
          g.v[x][p][4 * j] = w.x, g.v[x][p][4 * j + 1] = w.y;
          g.v[x][p][4 * j + 2] = w.z, g.v[x][p][4 * j + 3] = w.w;
        }
      }
    }
  }
}

// The head dim of output tile 4 w + i (8 columns), column n.
template <int HD>
__device__ __forceinline__ int out_dim(int w, int i, int n) {
  if constexpr (HD <= 128) return HD / 8 * n + 4 * w + i;
  else return 128 * (w / 4) + 16 * n + 4 * (w % 4) + i;
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kThreads) kv_attention_rows_kernel(KvAttentionArgs a,
                                                                     int row_blocks, bool join) {
  using Sh = RowShape<HD>;
  constexpr int KW = Sh::KW, VW = Sh::VW, GR = Sh::GR;
  __shared__ float s_o[kWarps][kRows][HD];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ int64_t s_scan[kThreads];
  pdl_trigger();
  pdl_wait();
  const KvView &c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int64_t hr = (int64_t)c.heads * row_blocks;  // (key head, row block) pairs
  const int rows_all = a.tokens * a.group;           // query rows of a key head

  // the CTA's run of units [lo, hi), and the sequence that holds unit lo
  const int per_thread = (c.batch + kThreads - 1) / kThreads;
  const int b0 = min(c.batch, tid * per_thread), b1 = min(c.batch, b0 + per_thread);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    int len, count;
    mine += units_of(a, b, Sh::kUnit, len, count);
  }
  s_scan[tid] = mine;
  __syncthreads();
  for (int o = 1; o < kThreads; o <<= 1) {
    const int64_t x = tid >= o ? s_scan[tid - o] : 0;
    __syncthreads();
    s_scan[tid] += x;
    __syncthreads();
  }
  const int64_t total = s_scan[kThreads - 1] * hr;
  const int64_t run = (total + gridDim.x - 1) / gridDim.x;
  const int64_t lo = blockIdx.x * run, hi = min(total, lo + run);
  if (lo >= hi) return;
  int b = 0;
  int64_t first = 0;  // first unit of sequence b
  {
    int t = 0;
    while (s_scan[t] * hr <= lo) ++t;
    b = t * per_thread;
    first = t > 0 ? s_scan[t - 1] * hr : 0;
  }
  int len, count;
  int units = units_of(a, b, Sh::kUnit, len, count);
  while (first + units * hr <= lo) {
    first += units * hr;
    units = units_of(a, ++b, Sh::kUnit, len, count);
  }

  for (int64_t u = lo; u < hi;) {
    if (u >= first + units * hr) {
      first += units * hr;
      units = units_of(a, ++b, Sh::kUnit, len, count);
    }
    const int64_t pair = (u - first) / units;
    const int h = (int)(pair / row_blocks), rb = (int)(pair % row_blocks);
    const int64_t seg0 = first + pair * units, seg1 = seg0 + units;
    const int t_lo = (int)(u - seg0), t_hi = (int)(min(hi, seg1) - seg0);

    // the row of this thread's accumulators, and the tokens it sees
    const int r = rb * kRows + gid;
    const int tok = r / a.group;
    const bool live = r < rows_all && tok < count;
    const int end = live ? len - count + tok + 1 : 0;
    const int r_first = rb * kRows / a.group;
    const int r_last = min(rb * kRows + kRows - 1, rows_all - 1) / a.group;
    const int all_end = len - count + min(r_first, count) + 1;      // tokens that every live row sees
    const int any_end = r_first < count ? len - count + min(r_last, count - 1) + 1 : 0;

    // q, scaled to [1, 2) and split
    uint32_t qa[KW][4];
    float sc;
    {
      float x[KW][4];
      float mx = 0.f;
      const int64_t off = b * a.qs.batch + tok * a.qs.token + (h * a.group + r % a.group) * a.qs.head;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int d = HD == 32 ? 8 * tig + 4 * w : 64 * (w / 4) + 16 * tig + 4 * (w % 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[w][i] = live && d < c.hd ? kv_load_in(a.dtype, a.q, off + d + i) : 0.f;
          mx = fmaxf(mx, fabsf(x[w][i]));
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = (__float_as_int(mx) >> 23) - 127;
      e = mx > 0.f ? min(max(e, -126), 126) : 0;
      const float f = kv_pow2(-e);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        f16_split2(x[w][0] * f, x[w][1] * f, qa[w][0], qa[w][1]);
        f16_split2(x[w][2] * f, x[w][3] * f, qa[w][2], qa[w][3]);
      }
      sc = a.scale * 1.4426950408889634f * kCodeUnit<FMT> * kv_pow2(e);
    }

    float m = -CUDART_INF_F, l = 0.f;
    float o[4 * VW][4];
#pragma unroll
    for (int i = 0; i < 4 * VW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

    bool flushed = false;
    float beta = 1.f;  // what the flushed sum is scaled by when read next
    auto flush = [&] {
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            float &sum = s_o[warp][gid][out_dim<HD>(w, i, 2 * tig + n)];
            const float v = o[4 * w + i][n] + o[4 * w + i][2 + n];
            sum = flushed ? fmaf(sum, beta, v) : v;
          }
      flushed = true;
      beta = 1.f;
    };
    auto t0_of = [&](int t) { return t * Sh::kUnit + warp * Sh::kStep; };
    auto page_at = [&](int t0) {
      return t0 < any_end ? c.page_of(b, t0 >> c.page_log2) : -1;
    };
    Group<HD> cur[GR], nxt[GR];
    int pg[GR], npg[GR];
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      pg[g] = page_at(t0_of(t_lo) + 16 * g);
      load_group<HD>(cur[g], c, pg[g], h, t0_of(t_lo) + 16 * g, lane);
    }
    for (int t = t_lo; t < t_hi; ++t) {
      const int t0 = t0_of(t);
      if (t > t_lo && (t - t_lo) % Sh::kFlush == 0) {
        flush();
#pragma unroll
        for (int i = 0; i < 4 * VW; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      }
      if (t + 1 < t_hi) {
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          npg[g] = page_at(t0_of(t + 1) + 16 * g);
          load_group<HD>(nxt[g], c, npg[g], h, t0_of(t + 1) + 16 * g, lane);
        }
      }
      if (t0 < any_end) {  // the same for the whole warp
        float s[GR][2][4];
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[g][x][i] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int g = 0; g < GR; ++g)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t k0, k1;
              codes_along<FMT>(cur[g].k[x][w], k0, k1);
              mma16816(s[g][x], qa[w][0], qa[w][1], qa[w][2], qa[w][3], k0, k1);
            }
        // scores of this thread: row gid, tokens 8 x + 4 p + tig of group g
        float kc[GR], ve[GR], top = -CUDART_INF_F;
        bool masked[GR];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const int tg = t0 + 16 * g;
          kc[g] = cur[g].ks * sc;
          // vs = 2^e; a NaN scale stays NaN
          ve[g] = cur[g].vs == cur[g].vs ? (float)((__float_as_int(cur[g].vs) >> 23) - 127) : cur[g].vs;
          masked[g] = pg[g] < 0 || tg + 16 > all_end;
          float mx = -CUDART_INF_F;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              float v = s[g][x][p] + s[g][x][2 + p];
              if (masked[g] && (pg[g] < 0 || tg + 8 * x + 4 * p + tig >= end)) v = -CUDART_INF_F;
              s[g][x][p] = v;
              mx = fmaxf(mx, v);
            }
          top = fmaxf(top, fmaf(mx, kc[g], ve[g]));
        }
        // p stays below 2^15: the reference moves when a score passes it by more than 1
        if (__any_sync(0xffffffffu, top > m + 1.f || (m == -CUDART_INF_F && top > m))) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float mn = fmaxf(m, ceilf(top));
          const float alpha = mn == m ? 1.f : exp2_approx(m - mn);  // 0 from -inf
          m = mn;
          l *= alpha;
          beta *= alpha;
#pragma unroll
          for (int i = 0; i < 4 * VW; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] *= alpha;
        }
        const float ref = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const int tg = t0 + 16 * g;
          const float base = ve[g] - ref + 14.f;
          float p[2][2], sum = 0.f;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float v = exp2_approx(fmaf(s[g][x][q], kc[g], base));
              if (masked[g] && (pg[g] < 0 || tg + 8 * x + 4 * q + tig >= end)) v = 0.f;
              p[x][q] = v;
              sum += v;
            }
          // a NaN scale counts only where a token of its page is seen
          if (sum != 0.f) l = fmaf(sum, 1.f / cur[g].vs, l);
          uint32_t pa[4];
          f16_split2(p[0][0], p[0][1], pa[0], pa[1]);
          f16_split2(p[1][0], p[1][1], pa[2], pa[3]);
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t v0[4], v1[4];
            codes_across<FMT>(cur[g].v[0][0][w], cur[g].v[0][1][w], v0);
            codes_across<FMT>(cur[g].v[1][0][w], cur[g].v[1][1][w], v1);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma16816(o[4 * w + i], pa[0], pa[1], pa[2], pa[3], v0[i], v1[i]);
          }
        }
      }
#pragma unroll
      for (int g = 0; g < GR; ++g) cur[g] = nxt[g], pg[g] = npg[g];
    }

    // the warps' results joined
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (tig == 0) s_m[warp][gid] = m, s_l[warp][gid] = l;
    flush();
    __syncthreads();
    const bool whole = t_lo == 0 && t_hi == units;
    const int rows = min(kRows, rows_all - rb * kRows);
    float *slot = a.ws + ((int64_t)blockIdx.x * 2 + (t_lo == 0 ? 1 : 0)) * Sh::kSlot;
    for (int i = tid; i < rows * HD; i += kThreads) {
      const int rr = i / HD, d = i % HD;
      float mm = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][rr]);
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp whose scores are all NaN has m = -inf and a NaN sum
        const float f = s_m[w][rr] == mm ? 1.f : exp2_approx(s_m[w][rr] - mm);
        const float fw = s_l[w][rr] == s_l[w][rr] ? f : 1.f;
        ll = fmaf(s_l[w][rr], fw, ll);
        oo = fmaf(s_o[w][rr][d], fw, oo);
      }
      if (whole) {
        const int row = rb * kRows + rr, ti = row / a.group;
        if (d < c.hd) {
          const float v = ti >= count || ll == 0.f ? 0.f : oo * kCodeUnit<FMT> / ll;
          kv_store_out(a.out, (((int64_t)b * a.tokens + ti) * a.heads + h * a.group + row % a.group) * c.hd + d, v);
        }
      } else {
        slot[rr * HD + d] = oo;
        if (d == 0) slot[kRows * HD + rr] = mm, slot[kRows * HD + kRows + rr] = ll;
      }
    }
    __syncthreads();
    u += t_hi - t_lo;
  }
}

// Joins the partial results of the (sequence, key head, row block) runs that
// several CTAs shared, in the order of the CTAs; the others are done already.
template <int HD, int FMT>
__global__ void __launch_bounds__(kThreads) kv_attention_join_kernel(KvAttentionArgs a,
                                                                     int row_blocks, int ctas) {
  using Sh = RowShape<HD>;
  __shared__ int64_t s_sum[kWarps][2];
  pdl_trigger();
  pdl_wait();
  const KvView &c = a.c;
  const int tid = threadIdx.x;
  const int b = blockIdx.y;
  const int64_t hr = (int64_t)c.heads * row_blocks;
  int64_t before = 0, total = 0;
  for (int i = tid; i < c.batch; i += kThreads) {
    int len, count;
    const int n = units_of(a, i, Sh::kUnit, len, count);
    total += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if ((tid & 31) == 0) s_sum[tid >> 5][0] = before, s_sum[tid >> 5][1] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) before += s_sum[w][0], total += s_sum[w][1];
  int len, count;
  const int units = units_of(a, b, Sh::kUnit, len, count);
  const int64_t run = (total * hr + ctas - 1) / ctas;
  const int64_t pair = blockIdx.x;
  const int64_t u0 = before * hr + pair * units, u1 = u0 + units;
  const int64_t c0 = u0 / run, c1 = (u1 - 1) / run;
  if (c0 == c1) return;
  const int h = (int)(pair / row_blocks), rb = (int)(pair % row_blocks);
  const int rows_all = a.tokens * a.group, rows = min(kRows, rows_all - rb * kRows);
  auto slot = [&](int64_t cta) { return a.ws + (cta * 2 + (cta == c0 ? 1 : 0)) * Sh::kSlot; };
  for (int i = tid; i < rows * HD; i += kThreads) {
    const int rr = i / HD, d = i % HD;
    const int row = rb * kRows + rr, ti = row / a.group;
    if (d >= c.hd) continue;
    float mm = -CUDART_INF_F;
    for (int64_t k = c0; k <= c1; ++k) mm = fmaxf(mm, slot(k)[kRows * HD + rr]);
    float ll = 0.f, oo = 0.f;
    for (int64_t k = c0; k <= c1; ++k) {
      const float *s = slot(k);
      const float mk = s[kRows * HD + rr], lk = s[kRows * HD + kRows + rr];
      const float f = mk == mm || !(lk == lk) ? 1.f : exp2_approx(mk - mm);
      ll = fmaf(lk, f, ll);
      oo = fmaf(s[rr * HD + d], f, oo);
    }
    const float v = ti >= count || ll == 0.f ? 0.f : oo * kCodeUnit<FMT> / ll;
    kv_store_out(a.out, (((int64_t)b * a.tokens + ti) * a.heads + h * a.group + row % a.group) * c.hd + d, v);
  }
}

template <int HD, int FMT>
int rows_ctas(int *out) {
  static int cached[64] = {};
  int dev = 0;
  TT_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && cached[dev] > 0) {
    *out = cached[dev];
    return TT_OK;
  }
  int sms = 0, per = 0;
  TT_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  TT_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(
      &per, kv_attention_rows_kernel<HD, FMT>, kThreads, 0));
  *out = sms * std::max(per, 1);
  if (dev < 64) cached[dev] = *out;
  return TT_OK;
}

struct RowPlan {
  int row_blocks;
  int ctas;
  bool join;
  size_t ws_bytes;
};

template <int HD, int FMT>
int rows_plan(const KvView &c, int64_t tokens, int heads, RowPlan *p) {
  using Sh = RowShape<HD>;
  const int64_t rows = tokens * (heads / c.heads);
  const int64_t blocks = ceil_div(rows, kRows);
  if (rows > INT32_MAX || blocks * c.heads > INT32_MAX || c.batch > 65535)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_attention: too many rows or sequences");
  p->row_blocks = (int)blocks;
  int most = 0;
  const int rc = rows_ctas<HD, FMT>(&most);
  if (rc != TT_OK) return rc;
  const int64_t each = ceil_div((int64_t)c.columns << c.page_log2, Sh::kUnit);
  // no run is split when every sequence is one unit
  p->join = each > 1;
  p->ctas = (int)std::min<int64_t>(most, each * blocks * c.heads * c.batch);
  p->ws_bytes = p->join ? (size_t)p->ctas * 2 * Sh::kSlot * sizeof(float) : 0;
  return TT_OK;
}

template <int HD, int FMT>
int launch_rows(const KvAttentionArgs &a, cudaStream_t stream) {
  RowPlan p;
  const int rc = rows_plan<HD, FMT>(a.c, a.tokens, a.heads, &p);
  if (rc != TT_OK) return rc;
  TT_CUDA_TRY(launch_kernel(kv_attention_rows_kernel<HD, FMT>, dim3(p.ctas), dim3(kThreads), 0,
                            stream, 1, a, p.row_blocks, p.join));
  if (p.join)
    TT_CUDA_TRY(launch_kernel(kv_attention_join_kernel<HD, FMT>,
                              dim3(p.row_blocks * a.c.heads, a.c.batch), dim3(kThreads), 0, stream,
                              1, a, p.row_blocks, p.ctas));
  return TT_OK;
}

// The instantiation for a head_dim: the smallest width that holds it.
template <class F>
int for_shape(const KvView &c, F &&f) {
  const bool i8 = c.format == TT_KV_INT8;
#define TT_KV_SHAPE(HD)                                                        \
  return i8 ? f(std::integral_constant<int, HD>(), std::integral_constant<int, TT_KV_INT8>()) \
            : f(std::integral_constant<int, HD>(), std::integral_constant<int, TT_KV_E4M3>())
  if (c.hd <= 32) TT_KV_SHAPE(32);
  if (c.hd <= 64) TT_KV_SHAPE(64);
  if (c.hd <= 128) TT_KV_SHAPE(128);
  TT_KV_SHAPE(256);
#undef TT_KV_SHAPE
}

}  // namespace

// Rows of a key head from which the tile kernel takes over.
static bool use_tiles(const KvView &c, int64_t tokens, int heads) {
  return tokens * (heads / c.heads) >= 64;
}

size_t kv_attention_ws_bytes(const KvView &c, int64_t tokens, int heads) {
  if (use_tiles(c, tokens, heads)) return kv_attention_tiles_ws_bytes(c, tokens, heads);
  RowPlan p{};
  const int rc = for_shape(c, [&](auto hd, auto fmt) {
    return rows_plan<decltype(hd)::value, decltype(fmt)::value>(c, tokens, heads, &p);
  });
  return rc == TT_OK ? p.ws_bytes : 0;
}

int launch_kv_attention(const KvAttentionArgs &a, cudaStream_t stream) {
  if (use_tiles(a.c, a.tokens, a.heads)) return launch_kv_attention_tiles(a, stream);
  return for_shape(a.c, [&](auto hd, auto fmt) {
    return launch_rows<decltype(hd)::value, decltype(fmt)::value>(a, stream);
  });
}

}  // namespace tt
