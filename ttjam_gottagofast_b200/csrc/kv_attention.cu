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
// Tensor cores, m16n8k16: 16 tokens' codes, exact in fp16, are the 16-row operand of
// both products (S^T = K q^T, O^T = V^T p^T), a block of 8 query rows of one key head
// the 8 columns of the other. p, and q of fp32 rows (TWO), are split into two fp16
// pieces (22 significant bits, as the forward's split-precision schedule), both added
// into the same sums, so a row has fp32 accuracy before its one rounding to its own type.
// q of 16-bit rows needs one piece (scaled as below, a bfloat16 element below 2^-28 of the
// row's largest loses at most 2^-39 of that). With one piece of p, a float16 output was
// 2.9e-4 off against 2.1e-4 for its own rounding. p leaves the first product with the
// token along the rows and enters the second along them too; a transposition of 8 x 8
// fp16 values between registers (movmatrix) lies in between. Row q is scaled by a
// power of two to have its largest element in [2^14, 2^15), p by 2^14, to stay clear of
// the fp16 subnormals.
//
// Where a key head has a single query row (ONE: a step of one token without grouped
// heads), the 8 columns hold the two pieces for each of 4 groups of 16 tokens instead:
// every lane then works on 2 tokens of 64 rather than every eighth on one, and the
// sums of a group's columns meet at the end.
//
// A warp takes kStep tokens at a time from a ring of its own in shared memory,
// which its lanes fill with asynchronous 16-byte copies up to kStages steps ahead,
// over the borders of heads and sequences, so that a warp always has its next
// copies in flight and never waits for another warp. Bytes go from there straight
// into operand registers: the tokens and head dims are numbered within a step so
// that a thread's operand elements are consecutive bytes (which token or dim stands
// at which operand index is free as long as both operands agree), and 16-byte
// chunks are exchanged within a row so that a load's rows lie in different banks.
//
// Work is counted in units: kStep tokens of one (sequence, key head, row block), and
// kOver units for each such segment, as its start and end cost about that much
// (without them, warps with many short sequences end last). Every warp takes an
// equal run of consecutive units, whatever the lengths, and a second kernel joins
// the segments that ended up on several warps. Where no segment is longer than
// kWhole steps, warps take whole ones, and nothing is left to join.
//
// Measured, one new token a sequence: 2 sequences of 100000, 16 heads of 64, int8, 80
// to 82 us with the join, its first kernel at 5.5 TB/s of codes (0.83 of a plain
// copy's rate), bound by memory and by instructions (0.53 of the issue slots); 64 of
// up to 2048, e4m3, fp32, 38 us; 32 of up to 8192, 32 query heads on 4 of 128, fp16 on
// e4m3, 44 us, bound by the latency between dependent instructions, as registers leave 12 warps an
// SM. One short sequence: 8 us, a chain of loads (length, page, scale, codes). One sequence
// of 100000 with a single key head of 128: 148 us for one row, 258 for eight, nearly all of it the
// join, whose few blocks add up hundreds of partial results each.
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "kv_cache.cuh"
#include "kv_codes.cuh"

namespace tt {
namespace {

constexpr int kRows = 8;     // query rows per block
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

template <int HD, bool ONE>
struct RowShape {
  // groups of 16 tokens computed at once: as many as registers hold, since a group is
  // one chain of dependent instructions. (head_dim 128, one group against two, fp32 rows:
  // 8 rows 43 / 39 us and 32 rows 83 / 68 us, 4 sequences of 20000; one of 1500 23 / 17. head_dim 64,
  // two against four: 32 rows 126 / 119 us, 8 rows 47.9 / 47.3.)
  static constexpr int GC = HD == 32 ? 4 : HD == 64 ? 4 : HD == 128 ? 2 : 1;
  // ... and copied at once: a step
  static constexpr int GR = HD == 32 ? 8 : HD == 64 ? 4 : GC;
  static constexpr int kStep = 16 * GR;              // tokens
  static constexpr int kOver = GR >= 4 ? 1 : 2;      // units of a segment besides its steps
  static constexpr int kWhole = GR >= 4 ? 2 : 4;     // steps of a segment that is never split
  static constexpr int kStages = 2;  // steps in a warp's ring
  static constexpr uint32_t kStage = 2 * kStep * HD;  // bytes: keys, then values
  static constexpr uint32_t kSmem = kWarps * kStages * kStage;
  static constexpr int kCtas = HD == 256 && !ONE ? 2 : 3;  // per SM, as registers and shared memory allow
  // tensor cores add by rounding toward zero: after 1024 tokens the sum moves to the
  // place of the warp's partial result, so that it does not drift
  static constexpr int kFlush = 1024 / kStep;
  static_assert(kWhole <= kFlush, "segments that are never split have no such place");
  static constexpr int KW = HD / 16;                 // words of a token's keys per thread
  static constexpr int VW = HD / 32;                 // words of a token's values per thread
  static constexpr int kSlot = kRows * HD + 2 * kRows;  // floats of a partial result
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t *r) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(addr));
}
// An 8 x 8 matrix of 16-bit values, row lane / 4, columns 2 (lane % 4) and the next:
// transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c += a b (or c = a b); not volatile, so that independent products are interleaved
__device__ __forceinline__ void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Units of a segment of sequence b; at least one step, which writes the zeros of
// a sequence that has no new token.
template <int HD, bool ONE>
__device__ __forceinline__ int units_of(const KvAttentionArgs &a, int b, int &len, int &count) {
  using Sh = RowShape<HD, ONE>;
  len = a.c.length(b);
  count = a.c.count(a.counts, b, a.tokens, len);
  return Sh::kOver + (count > 0 ? (len + Sh::kStep - 1) / Sh::kStep : 1);
}

// Token (0-7) of operand column n of an 8-token half, and the swizzle of a row's
// 16-byte chunks (chunk c of row r stands at c ^ chunk_swizzle(r)): together they
// put the 8 lanes that load K in one cycle (2 rows, 4 chunks) and those that load
// V (4 rows, at one or two chunks) into different banks, at every width.
template <int HD>
__device__ __forceinline__ int half_token(int n) {
  const int t = n >> 1;
  return n & 1 ? 4 + (t ^ (HD == 64 ? 1 : 2)) : t;
}
template <int HD, bool EXACT>
__device__ __forceinline__ int chunk_swizzle(int row) {
  if constexpr (!EXACT || HD == 32) return 0;
  return HD == 64 ? row & 2 : (row & 3) << 1;
}

// Where a warp's run of units stands: unit t of the segment whose units [lo, hi)
// the run holds. The steps are the units from kOver on.
template <int HD, bool ONE>
struct Cursor {
  int64_t left;  // units of the run from unit lo of this segment on
  int b, len, count, units, pair, t, lo, hi;

  // the segment that holds unit `skip` of the sequence
  __device__ __forceinline__ void enter(int64_t skip, bool whole) {
    pair = (int)(skip / units);
    lo = (int)(skip - (int64_t)pair * units);
    bound(whole);
  }
  __device__ __forceinline__ void bound(bool whole) {
    hi = whole ? units : (int)min((int64_t)units, lo + left);
    t = max(lo, RowShape<HD, ONE>::kOver);
  }
  // to the run's next segment; false at its end
  __device__ __forceinline__ bool next(const KvAttentionArgs &a, int64_t hr, bool whole) {
    left -= hi - lo;
    if (left <= 0) return false;
    if (++pair >= hr) {
      pair = 0;
      units = units_of<HD, ONE>(a, ++b, len, count);
    }
    lo = 0;
    bound(whole);
    return true;
  }
  // past segments of which the run holds no step
  __device__ __forceinline__ bool to_step(const KvAttentionArgs &a, int64_t hr, bool whole) {
    while (t >= hi)
      if (!next(a, hr, whole)) return false;
    return true;
  }
};

// The head dim of output tile 4 w + i (8 columns), column n.
template <int HD>
__device__ __forceinline__ int out_dim(int w, int i, int n) {
  if constexpr (HD <= 128) return HD / 8 * n + 4 * w + i;
  else return 128 * (w / 4) + 16 * n + 4 * (w % 4) + i;
}

template <int HD, int FMT, bool EXACT, bool ONE, bool TWO>
__global__ void __launch_bounds__(kThreads, RowShape<HD, ONE>::kCtas)
    kv_attention_rows_kernel(KvAttentionArgs a, int row_blocks, bool whole) {
  using Sh = RowShape<HD, ONE>;
  constexpr int KW = Sh::KW, VW = Sh::VW, GR = Sh::GR, GC = Sh::GC, S = Sh::kStages;
  constexpr int NR = ONE ? 1 : 2;  // rows of a lane's results
  static_assert(TWO || !ONE, "the columns of a single row are there for both pieces");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_scan[kThreads];
  const KvView &c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int hd = EXACT ? HD : c.hd;
  const int64_t hr = (int64_t)c.heads * row_blocks;  // (key head, row block) pairs
  const int rows_all = a.tokens * a.group;           // query rows of a key head
  const uint32_t ring = smem_u32(smem) + warp * S * Sh::kStage;
  pdl_wait();

  // the warp's run of units, and the sequence that holds its first
  const int per_thread = (c.batch + kThreads - 1) / kThreads;
  const int b0 = min(c.batch, tid * per_thread), b1 = min(c.batch, b0 + per_thread);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    int len, count;
    mine += units_of<HD, ONE>(a, b, len, count);
  }
  // inclusive sums over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, mine, o);
    if (lane >= o) mine += v;
  }
  s_scan[tid] = mine;
  __syncthreads();
  for (int w = 0; w < warp; ++w) mine += s_scan[32 * w + 31];
  __syncthreads();
  s_scan[tid] = mine;
  __syncthreads();
  const int64_t total = s_scan[kThreads - 1] * hr;
  const int gw = blockIdx.x * kWarps + warp;
  const int64_t run = (total + gridDim.x * kWarps - 1) / (gridDim.x * kWarps);
  const int64_t lo = gw * run;
  if (lo >= total) return;
  Cursor<HD, ONE> use;  // what is computed; `fill` below is what is copied, ahead of it
  use.left = min(run, total - lo);
  {
    int t = 0;  // threads whose sequences end at or before lo
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k)
      t += __popc(__ballot_sync(0xffffffffu, s_scan[32 * k + lane] * hr <= lo));
    use.b = t * per_thread;
    int64_t first = t > 0 ? s_scan[t - 1] * hr : 0;
    use.units = units_of<HD, ONE>(a, use.b, use.len, use.count);
    while (first + use.units * hr <= lo) {
      first += use.units * hr;
      use.units = units_of<HD, ONE>(a, ++use.b, use.len, use.count);
    }
    use.enter(lo - first, whole);
    // whole segments belong to the run that holds their first unit
    if (whole && use.lo > 0 && !use.next(a, hr, whole)) return;
    if (!use.to_step(a, hr, whole)) return;
  }

  // tokens that the last live row of the cursor's row block sees
  auto seen_by_block = [&](const Cursor<HD, ONE> &u) {
    const int rb = u.pair % row_blocks;
    const int r_first = rb * kRows / a.group;
    const int r_last = min(rb * kRows + kRows - 1, rows_all - 1) / a.group;
    return r_first < u.count ? u.len - u.count + min(r_last, u.count - 1) + 1 : 0;
  };
  auto t0_of = [&](int t) { return (t - Sh::kOver) * Sh::kStep; };

  // ---- the copies -----------------------------------------------------------
  // Lane g < GR looks group g's page up one step before its bytes are copied; its
  // scales wait in the lane's queue for as long as the bytes do in the ring. A
  // group without a page, or past the last seen token, copies nothing and has the
  // key scale -1 and the value scale kNoPage.
  Cursor<HD, ONE> fill = use;
  bool more = true;
  int fill_end = seen_by_block(fill), fill_stage = 0, pg_next;
  const float kNoPage = __int_as_float(1);  // no scale that a write makes
  float q_ks[S], q_vs[S];
  auto look_up = [&] {
    const int t0 = t0_of(fill.t) + 16 * lane;
    pg_next = lane < GR && t0 < fill_end ? c.page_of(fill.b, t0 >> c.page_log2) : -1;
  };
  // where this lane's 16 bytes of every 512 of a group go
  constexpr int kCopies = HD / 32;  // of 512 bytes, in a group of full width
  uint32_t copy_at[EXACT && HD > 64 ? 2 : 1];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(copy_at) / 4); ++i) {
    const int at = 32 * i + lane, row = EXACT ? at / (HD / 16) : 0, ch = EXACT ? at % (HD / 16) : at;
    copy_at[i] = ring + row * HD + ((ch ^ chunk_swizzle<HD, EXACT>(row)) << 4);
  }
  auto issue = [&](float &ks, float &vs) {
    ks = -1.f;
    vs = kNoPage;
    const int h = fill.pair / row_blocks;
    if (pg_next >= 0) {  // lanes 0 .. GR - 1
      const uint32_t at = (uint32_t)pg_next * (uint32_t)c.heads + (uint32_t)h;
      ks = c.ks[at];
      vs = c.vs[at];
    }
    const int t0 = t0_of(fill.t);
#pragma unroll
    for (int g = 0; g < GR; ++g) {
      const int pg = __shfl_sync(0xffffffffu, pg_next, g);
      if (pg < 0) continue;
      const int64_t from = c.tile(pg, h) + ((t0 + 16 * g) & ((1 << c.page_log2) - 1)) * hd + 16 * lane;
      const uint32_t to = fill_stage * Sh::kStage + 16 * g * hd;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        // rows of 128 bytes and more: the swizzle of every other copy's rows differs
        const uint32_t dst = EXACT && HD > 64 ? copy_at[i & 1] + (i >> 1) * 1024 + to : copy_at[0] + i * 512 + to;
        if (EXACT || 512 * i + 16 * lane < 16 * hd) {
          copy16(dst, c.k + from + 512 * i);
          copy16(dst + Sh::kStep * hd, c.v + from + 512 * i);
        }
      }
    }
    fill_stage = fill_stage + 1 == S ? 0 : fill_stage + 1;
    if (++fill.t == fill.hi) {
      more = fill.to_step(a, hr, whole);
      if (more) fill_end = seen_by_block(fill);
    }
    if (more) look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < S; ++s) {
    q_ks[s] = -1.f, q_vs[s] = kNoPage;
    if (more) issue(q_ks[s], q_vs[s]);
    copies_commit();
  }
  int stage = 0;

  bool going = true;
  while (going) {
    const int h = use.pair / row_blocks, rb = use.pair % row_blocks;
    const int b = use.b, len = use.len, count = use.count;
    const int r_first = rb * kRows / a.group;
    const int all_end = len - count + min(r_first, count) + 1;  // tokens that every live row sees
    const int any_end = seen_by_block(use);
    // the block's row that column n stands for, its token and how many tokens that sees
    auto row_of = [&](int n) { return rb * kRows + (ONE ? 0 : n); };
    auto end_of = [&](int r) {
      const int tok = r / a.group;
      return r < rows_all && tok < count ? len - count + tok + 1 : 0;
    };

    // q of column gid, scaled to [1, 2) and split
    uint32_t qb[KW][TWO && !ONE ? 4 : 2];
    float sc[NR];
    {
      float x[KW][4];
      float mx = 0.f;
      const int r = row_of(gid), tok = r / a.group;
      const bool live = end_of(r) > 0;
      const int64_t off = b * a.qs.batch + tok * a.qs.token + (h * a.group + r % a.group) * a.qs.head;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const int d = HD == 32 ? 8 * tig + 4 * w : 64 * (w / 4) + 16 * tig + 4 * (w % 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[w][i] = 0.f;
        if (live && d < hd) kv_load_in4(a.dtype, a.q, off + d, a.q_vec, x[w]);
      }
#pragma unroll
      for (int w = 0; w < KW; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(x[w][i]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int e = q_exponent(mx);
      const float f = kv_pow2(-e);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        uint32_t hi[2], lo[2];
        f16_split2(x[w][0] * f, x[w][1] * f, hi[0], lo[0]);
        f16_split2(x[w][2] * f, x[w][3] * f, hi[1], lo[1]);
        if constexpr (ONE) {  // even columns the high pieces, odd ones the low ones
          qb[w][0] = gid & 1 ? lo[0] : hi[0];
          qb[w][1] = gid & 1 ? lo[1] : hi[1];
        } else {
          qb[w][0] = hi[0], qb[w][1] = hi[1];
          if constexpr (TWO) qb[w][2] = lo[0], qb[w][3] = lo[1];
        }
      }
      float scale = a.scale * 1.4426950408889634f * kv_pow2(e);
      if (mx == CUDART_INF_F) scale = CUDART_NAN_F;  // also where all its scores are -inf
#pragma unroll
      for (int j = 0; j < NR; ++j) sc[j] = __shfl_sync(0xffffffffu, scale, 4 * (2 * tig + j));
    }

    // rows of this lane's results: columns 2 tig + j
    int end[NR];
    float m[NR], l[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      end[j] = end_of(row_of(2 * tig + j));
      m[j] = -CUDART_INF_F, l[j] = 0.f;
    }
    float o[2 * VW][4];  // dims out_dim(w, 0, gid) + 0 .. 3 in tiles 2 w and 2 w + 1
#pragma unroll
    for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    const int t_lo = use.t, t_hi = use.hi;
    const bool from_start = t_lo == Sh::kOver, done = from_start && t_hi == use.units;
    float *const slot = a.ws + ((int64_t)gw * 2 + (from_start ? 1 : 0)) * Sh::kSlot;
    bool flushed = false;
    float beta[NR];  // what the flushed sums are scaled by when read next
    // the sums of row j, dims out_dim(w, 0, gid) and the three after it. (ONE: the
    // columns' sums meet in every lane of a quad; one of them keeps them.)
    auto sums = [&](int w, int j, float *v) {
      float4 *at = reinterpret_cast<float4 *>(slot + (ONE ? 0 : 2 * tig + j) * HD + out_dim<HD>(w, 0, gid));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float *c4 = o[2 * w + i / 2] + 2 * (i % 2);
        if constexpr (ONE) {
          v[i] = c4[0] + c4[1];
          v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1);
          v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
        } else {
          v[i] = c4[j];
        }
      }
      if (flushed && (!ONE || tig == 0)) {
        const float4 f = *at;
        v[0] = fmaf(f.x, beta[j], v[0]), v[1] = fmaf(f.y, beta[j], v[1]);
        v[2] = fmaf(f.z, beta[j], v[2]), v[3] = fmaf(f.w, beta[j], v[3]);
      }
      return at;
    };
    auto flush = [&] {
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          float v[4];
          float4 *at = sums(w, j, v);
          if (!ONE || tig == 0) *at = make_float4(v[0], v[1], v[2], v[3]);
        }
      flushed = true;
#pragma unroll
      for (int j = 0; j < NR; ++j) beta[j] = 1.f;
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    };
    // groups g0 .. g0 + GC - 1 of a step, the first at token t0: scores, running
    // maximum, p, p v. A lane's scores: rows j, tokens 8 x + half_token(gid) of group g;
    // ONE: of group tig alone.
    constexpr int GS = ONE ? 1 : GC;
    auto compute = [&](auto masked_form, int g0, int t0, uint32_t absent) {
      constexpr bool MASKED = decltype(masked_form)::value;  // or with value scales below kFarScale
      const uint32_t kb = ring + stage * Sh::kStage + 16 * g0 * hd;
      const uint32_t vb = kb + Sh::kStep * hd;
      float s[GS][2][NR];
      {
        constexpr int LB = HD == 32 ? 8 : 16;  // bytes a load
        float acc[GC][4];
#pragma unroll
        for (int g = 0; g < GC; ++g) {
          uint32_t w[2][KW];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r8 = half_token<HD>(gid);
            const uint32_t row = kb + (16 * g + 8 * x + r8) * hd;
#pragma unroll
            for (int i = 0; i < KW * 4 / LB; ++i) {
              const int d = 4 * LB * i + LB * tig;
              if (EXACT || d < hd) {
                lds<LB>(row + (d ^ (chunk_swizzle<HD, EXACT>(r8) << 4)), &w[x][i * (LB / 4)]);
              } else {
#pragma unroll
                for (int k = 0; k < LB / 4; ++k) w[x][i * (LB / 4) + k] = 0;
              }
            }
          }
          float low[4];  // the low pieces' sums, apart: two chains of products
#pragma unroll
          for (int i = 0; i < KW; ++i) {
            uint32_t k4[4];
            codes_along<FMT>(w[0][i], k4[0], k4[2]);
            codes_along<FMT>(w[1][i], k4[1], k4[3]);
            if (i == 0) mma16816_first(acc[g], k4, qb[i][0], qb[i][1]);
            else mma16816(acc[g], k4, qb[i][0], qb[i][1]);
            if constexpr (TWO && !ONE) {
              if (i == 0) mma16816_first(low, k4, qb[i][2], qb[i][3]);
              else mma16816(low, k4, qb[i][2], qb[i][3]);
            }
          }
          if constexpr (!ONE) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int j = 0; j < NR; ++j) s[g][x][j] = acc[g][2 * x + j] + (TWO ? low[2 * x + j] : 0.f);
          }
        }
        if constexpr (ONE) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float hi = acc[0][2 * x], lo = acc[0][2 * x + 1];
#pragma unroll
            for (int g = 1; g < GC; ++g) {
              hi = tig == g ? acc[g][2 * x] : hi;
              lo = tig == g ? acc[g][2 * x + 1] : lo;
            }
            s[0][x][0] = hi + lo;
          }
        }
      }
      const float ve_lane = q_vs[0] == q_vs[0] ? (float)((__float_as_int(q_vs[0]) >> 23) - 127) : q_vs[0];
      auto group = [&](int g) { return ONE ? tig : g; };
      auto sees = [&](int g, int x, int j) {
        return !((absent >> (g0 + group(g))) & 1u) &&
               t0 + 16 * group(g) + 8 * x + half_token<HD>(gid) < end[j];
      };
      float ks[GS], ve[GS], top[NR];
#pragma unroll
      for (int j = 0; j < NR; ++j) top[j] = -CUDART_INF_F;
#pragma unroll
      for (int g = 0; g < GS; ++g) {
        ve[g] = __shfl_sync(0xffffffffu, ve_lane, g0 + group(g));
        ks[g] = fabsf(__shfl_sync(0xffffffffu, q_ks[0], g0 + group(g)));  // never negative: it meets -inf
#pragma unroll
        for (int j = 0; j < NR; ++j) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if ((MASKED && !sees(g, x, j)) || (ONE && GC < 4 && tig >= GC)) s[g][x][j] = -CUDART_INF_F;
          top[j] = fmaxf(top[j], fmaf(fmaxf(s[g][0][j], s[g][1][j]), ks[g] * sc[j], ve[g]));
        }
      }
      // p stays below 2^15: a row's reference moves when a score passes it by more than 1
      bool moves = false;
#pragma unroll
      for (int j = 0; j < NR; ++j) moves |= top[j] > m[j] + 1.f;
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int j = 0; j < NR; ++j) {
#pragma unroll
          for (int k = ONE ? 1 : 4; k < 32; k *= 2) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], k));
          const float mn = fmaxf(m[j], ceilf(top[j]));
          const float alpha = mn == m[j] ? 1.f : exp2_approx(m[j] - mn);  // 0 from -inf
          l[j] = rescale(l[j], m[j] - mn, alpha);
          m[j] = mn;
          beta[j] *= alpha;
#pragma unroll
          for (int i = 0; i < 2 * VW; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (ONE || (k & 1) == j) o[i][k] *= alpha;
        }
      }
      float ref[NR];
#pragma unroll
      for (int j = 0; j < NR; ++j) ref[j] = 14.f - (m[j] == -CUDART_INF_F ? 0.f : m[j]);
      uint32_t pb[2][2];  // p of a group as the second product's columns: [piece][half]
      auto probabilities = [&](int g) {
        float p[2][NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
          auto powers = [&](float e, float *r) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              r[x] = exp2_approx(fmaf(s[g][x][j], ks[g] * sc[j], e + ref[j]));
              // a NaN scale leaves NaN at the tokens behind the mask
              if ((MASKED && !sees(g, x, j)) || (ONE && GC < 4 && tig >= GC)) r[x] = 0.f;
            }
          };
          float r[2];
          powers(ve[g], r);
          p[0][j] = r[0], p[1][j] = r[1];
          if (MASKED && ve[g] < kFarScale) {
            powers(0.f, r);
            l[j] += r[0] + r[1];
          } else {
            // 2^-e; a NaN counts only where a token of its page is seen
            const float sum = p[0][j] + p[1][j], more_l = fmaf(sum, exp2_approx(-ve[g]), l[j]);
            l[j] = !(MASKED || (ONE && GC < 4)) || sum != 0.f ? more_l : l[j];
          }
        }
        uint32_t hi[2], lo[2];
        if constexpr (ONE) {  // (high, low) of each token: the columns of group tig
          f16_split2(p[0][0], p[1][0], hi[0], lo[0]);
          pb[0][0] = transpose8(__byte_perm(hi[0], lo[0], 0x5410));
          pb[0][1] = transpose8(__byte_perm(hi[0], lo[0], 0x7632));
        } else {  // (row 2 tig, row 2 tig + 1) of each token
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            f16_split2(p[x][0], p[x][NR - 1], hi[x], lo[x]);
            pb[0][x] = transpose8(hi[x]);
            pb[1][x] = transpose8(lo[x]);
          }
        }
      };
      if constexpr (ONE) probabilities(0);
#pragma unroll
      for (int g = 0; g < GC; ++g) {
        uint32_t v[2][2][VW];
        constexpr int LB = VW >= 4 ? 16 : 4 * VW;  // bytes a load
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int in_g = 8 * x + half_token<HD>(2 * tig + q);
            const uint32_t row = vb + (16 * g + in_g) * hd;
#pragma unroll
            for (int i = 0; i < VW * 4 / LB; ++i) {
              const int d = 8 * LB * i + LB * gid;
              if (EXACT || d < hd) {
                lds<LB>(row + (d ^ (chunk_swizzle<HD, EXACT>(in_g & 7) << 4)), &v[x][q][i * (LB / 4)]);
              } else {
#pragma unroll
                for (int k = 0; k < LB / 4; ++k) v[x][q][i * (LB / 4) + k] = 0;
              }
            }
            // what stands behind the last token may be any bits, e4m3's NaN among them
            if (MASKED && FMT == TT_KV_E4M3 && (((absent >> (g0 + g)) & 1u) || t0 + 16 * g + in_g >= len)) {
#pragma unroll
              for (int i = 0; i < VW; ++i) v[x][q][i] = 0;
            }
          }
        uint32_t b4[2][2];
        if constexpr (ONE) {  // only the columns of this group
          b4[0][0] = gid >> 1 == g ? pb[0][0] : 0u;
          b4[0][1] = gid >> 1 == g ? pb[0][1] : 0u;
        } else {
          probabilities(g);
          b4[0][0] = pb[0][0], b4[0][1] = pb[0][1];
          b4[1][0] = pb[1][0], b4[1][1] = pb[1][1];
        }
        uint32_t va[VW][2][4];
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t v0[4], v1[4];
          codes_across<FMT>(v[0][0][w], v[0][1][w], v0);
          codes_across<FMT>(v[1][0][w], v[1][1][w], v1);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            va[w][i][0] = v0[2 * i], va[w][i][1] = v0[2 * i + 1];
            va[w][i][2] = v1[2 * i], va[w][i][3] = v1[2 * i + 1];
            mma16816(o[2 * w + i], va[w][i], b4[0][0], b4[0][1]);
            if constexpr (!ONE) mma16816(o[2 * w + i], va[w][i], b4[1][0], b4[1][1]);
          }
        }
      }
    };

    for (int t = t_lo; t < t_hi; ++t) {
      const int t0 = t0_of(t);
      if (t > t_lo && (t - t_lo) % Sh::kFlush == 0) {
        flush();
      }
      copies_wait<S - 1>();
      __syncwarp();
      if (t0 < any_end) {  // the same for the whole warp
        uint32_t absent = 0;
        const bool odd = __any_sync(0xffffffffu, lane < GR && !usual_scales(q_ks[0], q_vs[0]));
        if (odd) {
          const bool none = q_ks[0] < 0.f && __float_as_uint(q_vs[0]) == __float_as_uint(kNoPage);
          if (none) q_vs[0] = 1.f;
          else if (lane < GR) q_ks[0] = kv_scale(q_ks[0], c.status), q_vs[0] = kv_scale(q_vs[0], c.status);
          absent = __ballot_sync(0xffffffffu, lane < GR && none);
        }
#pragma unroll 1
        for (int g0 = 0; g0 < GR; g0 += GC) {
          const int tg = t0 + 16 * g0;
          if (tg >= any_end) break;
          // where every live row sees every token, the form without masks
          if (!odd && tg + 16 * GC <= all_end) compute(std::false_type(), g0, tg, absent);
          else compute(std::true_type(), g0, tg, absent);
        }
      }
      // the step's bytes are in registers: its place in the ring takes the next copies
      __syncwarp();
      stage = stage + 1 == S ? 0 : stage + 1;
#pragma unroll
      for (int i = 0; i + 1 < S; ++i) q_ks[i] = q_ks[i + 1], q_vs[i] = q_vs[i + 1];
      if (more) issue(q_ks[S - 1], q_vs[S - 1]);
      copies_commit();
    }

    // the rows' results: their output, or a partial one
#pragma unroll
    for (int j = 0; j < NR; ++j) {
#pragma unroll
      for (int k = ONE ? 1 : 4; k < 32; k *= 2) l[j] += __shfl_xor_sync(0xffffffffu, l[j], k);
      const int n = ONE ? 0 : 2 * tig + j, r = row_of(n), tok = r / a.group;
      const bool mine = r < rows_all && (!ONE || tig == 0);
      const float inv = tok >= count || l[j] == 0.f ? 0.f : 1.f / l[j];
      const int64_t at = (((int64_t)b * a.tokens + tok) * a.heads + h * a.group + r % a.group) * hd;
      // a partial result's reference is made even: the join takes half of a difference
      const float even = floorf(0.5f * m[j]) == 0.5f * m[j] ? 1.f : 0.5f;
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const int d = out_dim<HD>(w, 0, gid);
        float v[4];
        float4 *part = sums(w, j, v);
        if (!mine) continue;
        if (!done) {
          *part = make_float4(v[0] * even, v[1] * even, v[2] * even, v[3] * even);
        } else if (EXACT || d < hd) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = inv == 0.f ? 0.f : v[i] * inv;
          kv_store_out4(a.out, at + d, v);
        }
      }
      if (mine && !done && gid == 0)
        slot[kRows * HD + n] = even == 1.f ? m[j] : m[j] + 1.f, slot[kRows * HD + kRows + n] = l[j] * even;
    }
    going = use.next(a, hr, whole) && use.to_step(a, hr, whole);
    // only now: the next kernel's CTAs would take this one's places on the SMs and
    // wait there (measured: step grouped 70 us a call against 50)
    if (!going) pdl_trigger();
  }
}

// Joins the partial results of the segments that several warps shared; the others
// are done already. A thread takes 4 dims of a row, and every n-th partial result
// where there are threads to spare; their sums meet in shared memory, always in
// the same order.
constexpr int kJoinThreads = 256, kJoinItems = 64;

template <int HD, bool ONE>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(KvAttentionArgs a,
                                                                         int row_blocks, int warps) {
  using Sh = RowShape<HD, ONE>;
  __shared__ int s_c[3];             // first and last warp of the segment, count
  __shared__ float s_part[kJoinThreads][6];  // m, l, o
  pdl_wait();
  const KvView &c = a.c;
  const int tid = threadIdx.x;
  const int b = blockIdx.y, pair = blockIdx.x;
  if (tid < 32) {
    const int64_t hr = (int64_t)c.heads * row_blocks;
    int64_t before = 0, total = 0;
    int units = 0, mine = 0;
    for (int i = tid; i < c.batch; i += 32) {
      int len, count;
      const int n = units_of<HD, ONE>(a, i, len, count);
      total += n;
      if (i < b) before += n;
      if (i == b) units = n, mine = count;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    units = __shfl_sync(0xffffffffu, units, b & 31);
    mine = __shfl_sync(0xffffffffu, mine, b & 31);
    if (tid == 0) {
      const int64_t run = (total * hr + warps - 1) / warps;
      const int64_t u0 = before * hr + (int64_t)pair * units, u1 = u0 + units;
      // 64-bit divisions are long; few caches need them
      if (u1 <= INT32_MAX && run <= INT32_MAX) {
        s_c[0] = ((int)u0 + Sh::kOver) / (int)run;
        s_c[1] = ((int)u1 - 1) / (int)run;
      } else {
        s_c[0] = (int)((u0 + Sh::kOver) / run);
        s_c[1] = (int)((u1 - 1) / run);
      }
      s_c[2] = mine;
    }
  }
  __syncthreads();
  const int c0 = s_c[0], c1 = s_c[1], count = s_c[2];
  if (c0 == c1) return;
  const int h = pair / row_blocks, rb = pair % row_blocks;
  const int rows_all = a.tokens * a.group, rows = min(kRows, rows_all - rb * kRows);
  // this block's items, and the threads on one: a power of two, so that their sums
  // pair up
  const int hd4 = c.hd / 4, begin = blockIdx.z * kJoinItems;
  const int items = min(rows * hd4, begin + kJoinItems);
  if (begin >= items) return;
  int team = 1;
  while (2 * team * (items - begin) <= kJoinThreads && team < c1 - c0 + 1) team *= 2;
  for (int first = begin; first < items; first += kJoinThreads / team) {
    const int i = first + tid / team, part = tid % team;
    const bool in = i < items && tid < kJoinThreads / team * team;
    const int rr = in ? i / hd4 : 0, d = in ? i % hd4 * 4 : 0;
    const float *const base = a.ws + rr * HD + d, *const ml = a.ws + kRows * HD + rr;
    auto slot = [&](int w) { return ((int64_t)w * 2 + (w == c0 ? 1 : 0)) * Sh::kSlot; };
    float m = -CUDART_INF_F, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    // (m, l, o) += (mk, lk, v); a sum of NaN scores has m = -inf and a NaN l. The factors
    // 2^(m - mn) are squares, as l may need one below 2^-126 (rescale in kv_codes.cuh).
    auto add = [&](float mk, float lk, const float4 &v) {
      const float mn = fmaxf(m, mk);
      const float ro = m == mn || !(l == l) ? 1.f : exp2_approx(0.5f * (m - mn)), fo = ro * ro;
      const float rk = mk == mn || !(lk == lk) ? 1.f : exp2_approx(0.5f * (mk - mn)), fk = rk * rk;
      m = mn;
      l = fmaf(l * ro, ro, lk * rk * rk);
      o[0] = fmaf(o[0], fo, v.x * fk), o[1] = fmaf(o[1], fo, v.y * fk);
      o[2] = fmaf(o[2], fo, v.z * fk), o[3] = fmaf(o[3], fo, v.w * fk);
    };
    if (in) {
#pragma unroll 4
      for (int k = c0 + part; k <= c1; k += team)
        add(ml[slot(k)], ml[slot(k) + kRows], *reinterpret_cast<const float4 *>(base + slot(k)));
    }
    if (team > 1) {
      for (int step = team / 2; step > 0; step /= 2) {
        float *mine = s_part[tid];
        mine[0] = m, mine[1] = l, mine[2] = o[0], mine[3] = o[1], mine[4] = o[2], mine[5] = o[3];
        __syncthreads();
        if (part < step) {
          const float *s = s_part[tid + step];
          add(s[0], s[1], make_float4(s[2], s[3], s[4], s[5]));
        }
        __syncthreads();
      }
    }
    if (in && part == 0) {
      const int row = rb * kRows + rr, ti = row / a.group;
      const float inv = ti >= count || l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = inv == 0.f ? 0.f : o[k] * inv;
      kv_store_out4(a.out, (((int64_t)b * a.tokens + ti) * a.heads + h * a.group + row % a.group) * c.hd + d, o);
    }
  }
}

struct RowPlan {
  int row_blocks;
  int ctas;
  bool whole;
  size_t ws_bytes;
};

template <int HD, bool ONE>
int rows_plan(const KvView &c, int64_t tokens, int heads, RowPlan *p) {
  using Sh = RowShape<HD, ONE>;
  const int64_t rows = tokens * (heads / c.heads);
  const int64_t blocks = ceil_div(rows, kRows);
  if (rows > kKvMost || blocks * c.heads > INT32_MAX || c.batch > 65535)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_attention: too many rows or sequences");
  p->row_blocks = (int)blocks;
  int sms = 0;
  const int rc = kv_sm_count(&sms);
  if (rc != TT_OK) return rc;
  const int64_t steps = ceil_div((int64_t)c.columns << c.page_log2, Sh::kStep);  // of a segment, at most
  const int64_t segments = blocks * c.heads * c.batch;
  p->whole = steps <= Sh::kWhole;
  const int64_t most = p->whole ? segments : steps * segments;  // warps that could have work
  p->ctas = (int)std::min<int64_t>(sms * Sh::kCtas, ceil_div(most, kWarps));
  p->ws_bytes = p->whole ? 0 : (size_t)p->ctas * kWarps * 2 * Sh::kSlot * sizeof(float);
  return TT_OK;
}

template <int HD, int FMT, bool EXACT, bool ONE, bool TWO>
int launch_rows(const KvAttentionArgs &a, cudaStream_t stream) {
  using Sh = RowShape<HD, ONE>;
  RowPlan p;
  int rc = rows_plan<HD, ONE>(a.c, a.tokens, a.heads, &p);
  if (rc != TT_OK) return rc;
  auto *kern = kv_attention_rows_kernel<HD, FMT, EXACT, ONE, TWO>;
  static KvSmemSet set;
  if ((rc = set.ensure(reinterpret_cast<const void *>(kern), Sh::kSmem)) != TT_OK) return rc;
  TT_CUDA_TRY(launch_kernel(kern, dim3(p.ctas), dim3(kThreads), Sh::kSmem, stream, 1, a, p.row_blocks,
                            p.whole));
  if (!p.whole)
    TT_CUDA_TRY(launch_kernel(kv_attention_join_kernel<HD, ONE>,
                              dim3(p.row_blocks * a.c.heads, a.c.batch,
                                   (unsigned)ceil_div(std::min(kRows, a.tokens * a.group) * (a.c.hd / 4), kJoinItems)),
                              dim3(kJoinThreads), 0, stream, 1, a, p.row_blocks, p.ctas * kWarps));
  return TT_OK;
}

template <int HD, int FMT, bool ONE>
int launch_rows_of(const KvAttentionArgs &a, cudaStream_t stream) {
  const bool two = ONE || a.dtype == TT_DTYPE_F32;
  if (a.c.hd == HD)
    return two ? launch_rows<HD, FMT, true, ONE, true>(a, stream)
               : launch_rows<HD, FMT, true, ONE, ONE>(a, stream);
  return two ? launch_rows<HD, FMT, false, ONE, true>(a, stream)
             : launch_rows<HD, FMT, false, ONE, ONE>(a, stream);
}

// The smallest width that holds a head_dim, 32, 64, 128 or 256, and whether a key
// head has a single query row.
template <class F>
int for_rows(const KvView &c, int64_t rows, F &&f) {
  using std::integral_constant;
  auto width = [&](auto one) {
    if (c.hd <= 32) return f(integral_constant<int, 32>(), one);
    if (c.hd <= 64) return f(integral_constant<int, 64>(), one);
    if (c.hd <= 128) return f(integral_constant<int, 128>(), one);
    return f(integral_constant<int, 256>(), one);
  };
  return rows == 1 ? width(std::true_type()) : width(std::false_type());
}

// Rows of a key head from which the tile kernel takes over: it takes up to 128 rows in
// the time of one, this file's kernel goes over the codes once for every 8. Measured,
// e4m3, fp32 rows, this kernel / the tiles, us. 16 heads of 64: 16 sequences of 2000
// tokens, 48 rows 88 / 93; 4 of 20000, 48 rows 172 / 163, 32 rows 122 / 162. 32 heads
// of 128 on 4: 16 of 2000, 24 rows 35 / 42, 32 rows 41 / 41; 4 of 20000, 32 rows
// 68 / 93, 48 rows 91 / 93. (One short sequence costs 15 to 25 us either way.)
bool use_tiles(const KvView &c, int64_t tokens, int heads) {
  return tokens * (heads / c.heads) >= (c.hd <= 64 ? 56 : 40);
}

}  // namespace

int kv_sm_count(int *out) {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  TT_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (*out = cached[dev]) > 0) return TT_OK;
  TT_CUDA_TRY(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) cached[dev] = *out;
  return TT_OK;
}

int KvSmemSet::ensure(const void *kernel, size_t bytes, int regs) {
  int dev = 0;
  TT_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && done[dev]) return TT_OK;
  if (regs > 0) {
    cudaFuncAttributes at{};
    TT_CUDA_TRY(cudaFuncGetAttributes(&at, kernel));
    if (at.numRegs != regs)
      return fail(TT_ERR_UNSUPPORTED, "kernel built with " + std::to_string(at.numRegs) +
                                          " registers a thread, not " + std::to_string(regs));
  }
  TT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  if (dev < 64) done[dev] = true;
  return TT_OK;
}

size_t kv_attention_ws_bytes(const KvView &c, int dtype, int64_t tokens, int heads) {
  if (use_tiles(c, tokens, heads)) return kv_attention_tiles_ws_bytes(c, dtype, tokens, heads);
  RowPlan p{};
  const int rc = for_rows(c, tokens * (heads / c.heads), [&](auto hd, auto one) {
    return rows_plan<decltype(hd)::value, decltype(one)::value>(c, tokens, heads, &p);
  });
  return rc == TT_OK ? p.ws_bytes : 0;
}

int launch_kv_attention(const KvAttentionArgs &a, cudaStream_t stream) {
  if (use_tiles(a.c, a.tokens, a.heads)) return launch_kv_attention_tiles(a, stream);
  return for_rows(a.c, (int64_t)a.tokens * a.group, [&](auto hd, auto one) {
    constexpr int HD = decltype(hd)::value;
    constexpr bool ONE = decltype(one)::value;
    return a.c.format == TT_KV_INT8 ? launch_rows_of<HD, TT_KV_INT8, ONE>(a, stream)
                                    : launch_rows_of<HD, TT_KV_E4M3, ONE>(a, stream);
  });
}

}  // namespace tt
