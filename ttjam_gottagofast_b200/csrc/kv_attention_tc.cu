// Causal attention of new tokens over the 8-bit paged key/value cache, for many
// query rows (prompts): tcgen05 products of 128-row tiles. The mathematics is
// kv_attention.cu's: the key scale multiplies the score, the value scale 2^e
// joins the exponent, p = 2^(s' + e - M + 7) with a whole-number reference M,
// out = sum p code / sum p 2^-e; the codes, exact in fp16, are the B operands.
//
// PIECES: how many fp16 pieces q is split into. fp32 rows take two (22 significant
// bits). 16-bit rows take one: q, scaled by a power of two to have its largest element
// in [2^14, 2^15), is exact in it (bf16 elements below 2^-28 of the row's largest lose at
// most 2^-39 of that). p takes two whatever the rows' type, so that a row has fp32
// accuracy before its one rounding (one piece of p took 70 us less of the grouped prompt
// below, and was up to 2^-11 of the largest terms off); the sum of p is taken before p is
// split, in fp32.
//
// CTA = (row tile, key head, sequence, split of the tokens): MT tiles of 128 query
// rows (row = token * group + head of the group) against tiles of 64 tokens.
//   softmax   MT warpgroups: tensor-memory lane t of tile x is one thread's row. It
//             reads the 64 scores of a token tile into registers, takes their
//             maximum and writes p over them. O is rescaled in tensor memory only
//             when the maximum grows by more than 2^8.
//   conversion  a warpgroup: 16 codes a load, eight fp16 pairs, stored as
//             128-byte-swizzled rows of 64 dims, K-major for K and, the same bytes
//             read the other way, MN-major for V; the next tiles' codes are on their
//             way meanwhile. The tile's scales go to shared memory.
//   MMA       one warp of a last group allocates tensor memory; an elected lane issues the
//             products: S_x = q_x K^T into the tile's two score buffers in turn, two
//             token tiles ahead of the softmax, and O_x += P_x V (A = P from tensor
//             memory). (With one score buffer a row tile and 128 tokens a tile, a
//             softmax group waited for its own products: 355 us against 257 for
//             4 x 2048 fp32 rows behind 2048, 16 heads of 64. Two threads a row
//             instead of one: 279 us, the same work in more instructions.)
// Bound by the softmax groups' instructions, exp2 and reads of tensor memory at
// head_dim 64 (fp32, 4 x 2048 rows behind 2048, 16 heads: 103 GFLOP counted once, 265
// us), by shared memory's rate under the products of 64 columns and the converters'
// stores at 128 (bf16, 3 x 4096 rows, 32 heads on 4: 347 GFLOP, 560 us, 0.62 PFLOP/s).
// K and V tiles have a ring each. Every wait is bounded; one that gives up latches
// TT_ERR_DEVICE_TIMEOUT in the cache's status word, and the kernel frees its tensor
// memory and returns.
#include <math_constants.h>

#include <algorithm>
#include <cfloat>

#include "kv_cache.cuh"
#include "kv_codes.cuh"

namespace tt {
namespace {

// tt_test_arm_kv_wait_timeout: whether the next launch of the tile kernel takes the switch
std::atomic<bool> g_armed_timeout{false};

constexpr int kConvWarps = 4, kConvThreads = 32 * kConvWarps;

template <int HD_, int PIECES>
struct TcShape {
  static constexpr int HD = HD_;
  static constexpr int MT = HD <= 128 ? 2 : 1;    // 128-row tiles per CTA
  static constexpr int TOK = 64;                  // tokens per tile
  static constexpr bool QT = HD == 64;            // q in tensor memory (else shared memory)
  static constexpr int BOXES = HD / 64;           // 64-dim boxes of an operand tile
  static constexpr uint32_t BOX = TOK * 128;      // bytes
  static constexpr uint32_t SLOT = BOXES * BOX;
  static constexpr uint32_t QBOX = 128 * 128;
  static constexpr uint32_t QBYTES = QT ? 0 : MT * PIECES * BOXES * QBOX;
  static constexpr bool SUM_SMEM = HD == 64;  // see flush()
  static constexpr uint32_t SUMS = SUM_SMEM ? MT * 128 * HD * 4 : 0;
  // Codes on their way, AHEAD tiles: up to head_dim 64 in shared memory, every thread's
  // own chunks, copied asynchronously (in registers, loads share the few scoreboards,
  // and a wait for a page's number is one for the codes behind it: prompt 265 us, in
  // shared memory 258). Wider heads keep shared memory's bandwidth for the products
  // (prompt grouped 564 us staged, 480 in registers).
  static constexpr bool STAGED = HD <= 64;
  static constexpr int AHEAD = HD <= 128 ? 2 : 1;
  static constexpr uint32_t STAGE = STAGED ? 2 * TOK * HD : 0;  // bytes of a tile's codes
  static constexpr int SLOTS =
      (int)std::min<uint32_t>(8, (224 * 1024 - QBYTES - SUMS - AHEAD * STAGE) / SLOT);
  static constexpr int NK = SLOTS / 2, NV = SLOTS - NK;  // ring of K tiles, of V tiles
  static constexpr uint32_t V0 = QBYTES + NK * SLOT;     // first V slot
  static constexpr uint32_t SUM0 = QBYTES + SLOTS * SLOT;  // flushed sums
  static constexpr uint32_t STAGE0 = SUM0 + SUMS;          // codes on their way
  static constexpr uint32_t BARS = STAGE0 + AHEAD * STAGE;  // barriers, after all those
  static constexpr size_t SMEM = BARS + 1024 + 1024;       // alignment of the base, barriers
  static constexpr int SOFT_WARPS = 4 * MT;
  // warpgroups: softmax (MT), conversion, MMA issue (one warp of it). With two
  // softmax groups the block starts with 128 registers a thread, and they take
  // 176 (152), which the other two give up: 2 * 176 + 2 * 80 = 4 * 128.
  static constexpr int THREADS = 32 * (SOFT_WARPS + kConvWarps + 4);
  static constexpr bool SHIFT_REGS = MT == 2;
  static constexpr int START_REGS = 128;
  static constexpr int SOFT_REGS = HD == 64 ? 176 : 152, OTHER_REGS = HD == 64 ? 80 : 104;
  static_assert(!SHIFT_REGS || 2 * SOFT_REGS + 2 * OTHER_REGS <= 4 * START_REGS, "registers of the block");
  // tensor-memory columns: O, two score buffers a row tile, q
  static constexpr uint32_t T_O = 0, T_S = MT * HD, T_Q = MT * (HD + 2 * TOK);
  static_assert(T_Q + (QT ? MT * PIECES * HD / 2 : 0) <= 512, "tensor memory");
  static_assert(NK >= 1 && NV >= 2 && SMEM <= 227 * 1024, "shared memory");
  // Tile j's scales stand in place j % 8; they are written once V tile j - 1 has a
  // slot, that is, once the softmax of tile j - 1 - NV is done.
  static constexpr int SCALES = 8;
  static_assert(NV + 1 <= SCALES, "scales");
  // Tensor memory adds a product to O by rounding toward zero, so a long sum drifts:
  // 8.6e-9 of the output a token where the values have one sign. The softmax warps
  // therefore take O out every flush() tiles and start it anew. The sum stands in shared
  // memory at head_dim 64 (512 tokens); at wider heads in an fp32 row's partial result or
  // its own place of the output (1024 tokens), or for 16-bit rows in the workspace, the 128
  // rows of a tile side by side: float16 every 4096 tokens (3.5e-5, 1/14 of its half step),
  // bfloat16 every 8192 (7e-5, 1/56).
  static constexpr bool SUM_WS = PIECES == 1 && !SUM_SMEM;
  static constexpr int MIN_FLUSH = (SUM_SMEM ? 512 : SUM_WS ? 4096 : 1024) / TOK;
  __host__ __device__ static constexpr int flush(int dtype) {
    return SUM_WS && dtype == TT_DTYPE_BF16 ? 2 * MIN_FLUSH : MIN_FLUSH;  // a power of two
  }
  static constexpr int GROUPS = TOK / 16;  // of 16 tokens, each in one page
  static constexpr int NCH = TOK * HD / 16 / kConvThreads;  // 16-code chunks a converter thread
  static constexpr uint32_t IDESC_S =
      (1u << 4) | ((uint32_t)(TOK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t IDESC_PV =  // B is MN-major
      (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Bounded wait: false after about 2^28 cycles (latching TT_ERR_DEVICE_TIMEOUT and
// setting the CTA's abort word), or soon after another thread's gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_w,
                                          DeviceStatus *st, int detail) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 31) == 0) {
      if (*abort_w != 0) return false;
      if (clock64() - t0 > (1LL << 28)) {
        *abort_w = 1;
        raise_status(st, TT_ERR_DEVICE_TIMEOUT, detail);
        return false;
      }
    }
  }
}
// Shared-memory matrix descriptor, 128-byte swizzle: 8-row groups 1024 bytes
// apart, and (MN-major) 64-element blocks `lead` bytes apart.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lead) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((lead >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// The MMA warp stays converged, so that descriptors live in uniform registers; one
// elected lane issues.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Two non-negative values below 65504 to one fp16 pair, or to two (high, rest).
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// The upper 11 significant bits, exact in fp16 from 2^-14 on; below that, rounded
// there to a multiple of 2^-24.
__device__ __forceinline__ float upper11(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffffe000u);
}

template <int HD, int FMT, int PIECES>
__global__ void __launch_bounds__(TcShape<HD, PIECES>::THREADS, 1)
    kv_attention_tiles_kernel(KvAttentionArgs a, int row_tiles, int splits) {
  using Sh = TcShape<HD, PIECES>;
  constexpr int MT = Sh::MT, TOK = Sh::TOK, NK = Sh::NK, NV = Sh::NV, GROUPS = Sh::GROUPS;
  constexpr int SCALES = Sh::SCALES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float s_ks[SCALES][GROUPS], s_ve[SCALES][GROUPS];
  __shared__ float s_we[SCALES][GROUPS];  // 2^-ve, a weight over its p; 0 below kFarScale
  __shared__ uint32_t s_ok[SCALES];       // groups whose page exists; above them, whether one is below kFarScale
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *const smem = smem_raw + (base - raw);
  const uint32_t bars = base + Sh::BARS;
  auto k_full = [&](int i) { return bars + 8u * i; };
  auto k_empty = [&](int i) { return bars + 8u * (NK + i); };
  auto v_full = [&](int i) { return bars + 8u * (2 * NK + i); };
  auto v_empty = [&](int i) { return bars + 8u * (2 * NK + NV + i); };
  constexpr uint32_t XS = 2 * NK + 2 * NV;
  auto s_full = [&](int x, int buf) { return bars + 8u * (XS + 2 * x + buf); };
  auto p_full = [&](int x, int buf) { return bars + 8u * (XS + 2 * MT + 2 * x + buf); };
  auto o_done = [&](int x) { return bars + 8u * (XS + 4 * MT + x); };
  auto o_final = [&](int x) { return bars + 8u * (XS + 5 * MT + x); };
  constexpr uint32_t XB = XS + 6 * MT;
  auto sc_full = [&](int i) { return bars + 8u * (XB + i); };
  const uint32_t q_ready = bars + 8u * (XB + SCALES), drain_bar = bars + 8u * (XB + SCALES + 1);
  const uint32_t tmem_slot = bars + 8u * (XB + SCALES + 2);
  static_assert(8 * (XB + SCALES + 3) <= 1024, "barriers");
  volatile uint32_t *tmem_slot_p = reinterpret_cast<volatile uint32_t *>(smem + (tmem_slot - base));
  volatile int *abort_w = reinterpret_cast<volatile int *>(smem + (tmem_slot + 4 - base));

  const KvView &c = a.c;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  // latest row tiles (the longest, causally) first
  const int rt = row_tiles - 1 - (int)(blockIdx.x / c.heads), h = blockIdx.x % c.heads;
  const int b = blockIdx.y, split = blockIdx.z;
  const int rows_all = a.tokens * a.group, row0 = rt * 128 * MT;
  const int len = c.length(b), count = c.count(a.counts, b, a.tokens, len);
  const int live = min(rows_all, count * a.group) - row0;  // live rows from row0 on
  // tokens that the CTA's last live row sees, and this split's tiles of them
  const int any_end = live > 0 ? len - count + (row0 + min(live, 128 * MT) - 1) / a.group + 1 : 0;
  const int tiles = (any_end + TOK - 1) / TOK;
  const int j0 = (int)((int64_t)tiles * split / splits);
  const int nj = (int)((int64_t)tiles * (split + 1) / splits) - j0;
  const int active = min(MT, (live + 127) / 128);

  const int flush = Sh::flush(a.dtype);  // tiles between two flushes of O

  // results of this thread's row, written where they belong
  const int64_t rows_padded = (int64_t)row_tiles * 128 * MT;
  auto part = [&](int r) {  // partial result of row r
    return (((int64_t)split * c.batch + b) * c.heads + h) * rows_padded + r;
  };
  float *const part_ml = a.ws + (int64_t)splits * c.batch * c.heads * rows_padded * HD;
  auto out_row = [&](int r) {
    return (((int64_t)b * a.tokens + r / a.group) * a.heads + h * a.group + r % a.group) * c.hd;
  };
  if (nj <= 0) {  // no token for any row: zeros (the same for the whole CTA)
    if (warp < Sh::SOFT_WARPS) {
      const int r = row0 + threadIdx.x;
      if (splits > 1) {
        part_ml[2 * part(r)] = -CUDART_INF_F;
        part_ml[2 * part(r) + 1] = 0.f;
      } else if (r < rows_all) {
        const float z[16] = {};
        for (int d = 0; d < c.hd; d += 16) kv_store_row16(a.out, out_row(r) + d, z);
      }
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) mbar_init(k_full(i), kConvWarps), mbar_init(k_empty(i), 1);
    for (int i = 0; i < NV; ++i) mbar_init(v_full(i), kConvWarps), mbar_init(v_empty(i), 1);
    for (int x = 0; x < MT; ++x) {
      for (int buf = 0; buf < 2; ++buf) mbar_init(s_full(x, buf), 1), mbar_init(p_full(x, buf), 4);
      mbar_init(o_done(x), 1), mbar_init(o_final(x), 1);
    }
    for (int i = 0; i < SCALES; ++i) mbar_init(sc_full(i), 1);
    mbar_init(q_ready, 4 * active + a.test_hold_back);  // 1: an arrival that never comes
    mbar_init(drain_bar, 1);
    *abort_w = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  constexpr int kMmaWarp = Sh::SOFT_WARPS + kConvWarps;  // the rest of its group only waits
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, *tmem_slot_p, 0);
  if constexpr (Sh::SHIFT_REGS) {
    if (warp < Sh::SOFT_WARPS)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sh::SOFT_REGS));
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::OTHER_REGS));
  }

  if (warp >= kMmaWarp) {
    if (warp == kMmaWarp) {
      // ---- MMA issuer ------------------------------------------------------
      auto warp_wait = [&](uint32_t bar, uint32_t parity, int detail) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_w, c.status, detail)) != 0;
      };
      auto wait_k = [&](int j) {
        return warp_wait(k_full(j % NK), (j / NK) & 1, 0x6100);
      };
      auto issue_s = [&](int x, int j) {
        const uint32_t k = base + Sh::QBYTES + (uint32_t)(j % NK) * Sh::SLOT;
        const uint32_t d = tm + Sh::T_S + (uint32_t)(TOK * (2 * x + (j & 1)));
        const uint64_t kd0 = sdesc(k, 16);
        const uint64_t qd0 = sdesc(base + (uint32_t)(x * PIECES * Sh::BOXES) * Sh::QBOX, 16);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint64_t kd = kd0 + (kk / 4) * (Sh::BOX >> 4) + 2 * (kk % 4);
#pragma unroll
          for (int w = 0; w < PIECES; ++w) {
            if constexpr (Sh::QT) {
              mma_ts(d, tm + Sh::T_Q + (uint32_t)((x * PIECES + w) * (HD / 2) + 8 * kk), kd,
                     Sh::IDESC_S, (kk | w) != 0);
            } else {
              mma_ss(d, qd0 + (w * Sh::BOXES + kk / 4) * (Sh::QBOX >> 4) + 2 * (kk % 4), kd,
                     Sh::IDESC_S, (kk | w) != 0);
            }
          }
        }
        mma_commit(s_full(x, j & 1));
      };
      bool ok = warp_wait(q_ready, 0, 0x6000);
      for (int j = 0; ok && j < 2 && j < nj; ++j) {
        if (!(ok = wait_k(j))) break;
        fence_after();
        for (int x = 0; x < active; ++x) issue_s(x, j);
        mma_commit(k_empty(j % NK));
      }
      for (int j = 0; ok && j < nj; ++j) {
        ok = warp_wait(v_full(j % NV), (j / NV) & 1, 0x6110);
        const uint32_t v = base + Sh::V0 + (uint32_t)(j % NV) * Sh::SLOT;
        for (int x = 0; ok && x < active; ++x) {
          if (!(ok = warp_wait(p_full(x, j & 1), (j >> 1) & 1, 0x6200))) break;
          fence_after();
          const uint32_t p = tm + Sh::T_S + (uint32_t)(TOK * (2 * x + (j & 1)));
          const uint64_t vd0 = sdesc(v, Sh::BOX);
#pragma unroll
          for (int kk = 0; kk < TOK / 16; ++kk)
#pragma unroll
            for (int w = 0; w < 2; ++w)  // p's pieces
              mma_ts(tm + Sh::T_O + (uint32_t)(HD * x),
                     p + 32u * (kk >> 1) + 8u * (kk & 1) + 16u * w, vd0 + 128 * kk, Sh::IDESC_PV,
                     ((j & (flush - 1)) | kk | w) != 0);
          mma_commit(j + 1 < nj ? o_done(x) : o_final(x));
          if (j + 2 < nj) {  // into the buffer that this product has read
            if (x == 0 && !(ok = wait_k(j + 2))) break;
            fence_after();
            issue_s(x, j + 2);
          }
        }
        if (ok) {
          mma_commit(v_empty(j % NV));
          if (j + 2 < nj) mma_commit(k_empty((j + 2) % NK));
        }
      }
      // every MMA issued above has completed before the tensor memory is freed
      mma_commit(drain_bar);
      const long long t0 = clock64();
      for (uint32_t i = 0; !mbar_try_wait(drain_bar, 0); ++i)
        if ((i & 31) == 31 && clock64() - t0 > (1LL << 28)) {
          raise_status(c.status, TT_ERR_DEVICE_TIMEOUT, 0x6F00);
          break;
        }
    }
    __syncwarp();
  } else if (warp >= Sh::SOFT_WARPS) {
    // ---- conversion of the codes -------------------------------------------
    // Chunk u of a thread: 16 codes, dims 64 (u / 2) + 16 (ct % 4) of token ct / 4 +
    // 32 (u % 2): eight lanes' stores of 16 bytes meet different banks.
    constexpr int NCH = Sh::NCH;
    static_assert(TOK * 4 == 2 * kConvThreads, "two tokens a thread");
    const int ct = threadIdx.x - 32 * Sh::SOFT_WARPS, row = ct >> 2;
    const int cw = warp - Sh::SOFT_WARPS;
    const uint32_t put = row * 128 + (((2 * (ct & 3)) ^ (row & 7)) << 4);
    // Lane g < GROUPS looks up group g's page: the table entry a tile before its
    // check, which comes a tile or two (AHEAD) before the codes that it leads to.
    constexpr int AHEAD = Sh::AHEAD;
    auto entry_of = [&](int j) {
      const int t = (j0 + j) * TOK + 16 * lane;
      return j < nj && lane < GROUPS && t < any_end ? c.table[(int64_t)b * c.columns + (t >> c.page_log2)]
                                                    : INT32_MIN;
    };
    auto page_of = [&](int entry) {
      if ((unsigned)entry < (unsigned)c.pages) return entry;
      if (entry != INT32_MIN) raise_status(c.status, TT_ERR_DEVICE_FAULT, kKvBadPage);
      return -1;
    };
    uint4 raw_k[AHEAD][NCH], raw_v[AHEAD][NCH];  // (unless staged)
    int ids[AHEAD];
    float ks[AHEAD], vs[AHEAD];
    // where this thread's two tokens of tile j lie in the pools; bit r of `none` where
    // token r lies nowhere, or behind the last one (such a slot may hold any bits):
    // something else is read then, and zeros are stored
    auto places = [&](int id, int j, int64_t *at) -> uint32_t {
      uint32_t none = 0;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int t = row + 32 * r, pg = __shfl_sync(0xffffffffu, id, t >> 4);
        const int tok = (j0 + j) * TOK + t;
        const bool there = pg >= 0 && tok < any_end;
        at[r] = there ? c.tile(pg, h) + (tok & ((1 << c.page_log2) - 1)) * c.hd + 16 * (ct & 3) : 0;
        none |= there ? 0u : 1u << r;
      }
      return none;
    };
    auto in_head = [&](int u) { return 64 * (u >> 1) + 16 * (ct & 3) < c.hd; };
    auto load = [&](const uint8_t *pool, const int64_t *at, uint4 *r) {
#pragma unroll
      for (int u = 0; u < NCH; ++u)
        if (in_head(u)) r[u] = *reinterpret_cast<const uint4 *>(pool + at[u & 1] + 64 * (u >> 1));
    };
    // place n of the staged codes; chunk u of this thread's keys (kv 0) or values (1)
    auto staged = [&](int n, int kv, int u) {
      return Sh::STAGE0 + n * Sh::STAGE + (uint32_t)((kv * NCH + u) * kConvThreads + ct) * 16;
    };
    auto copy = [&](int n, const int64_t *at) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int u = 0; u < NCH; ++u)
          if (in_head(u))
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + staged(n, kv, u)),
                         "l"((kv ? c.v : c.k) + at[u & 1] + 64 * (u >> 1))
                         : "memory");
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const bool narrow = c.hd != HD;  // dims past head_dim are zero
    auto store = [&](uint32_t slot, uint32_t full, uint32_t none, auto &&chunk) {
      const bool clear = __any_sync(0xffffffffu, none != 0) || narrow;
      uint8_t *const dst = smem + slot;
#pragma unroll
      for (int u = 0; u < NCH; ++u) {
        uint4 r = chunk(u);
        if (clear && (((none >> (u & 1)) & 1u) || !in_head(u))) r = make_uint4(0, 0, 0, 0);
        uint32_t f[8];
        codes_along<FMT>(r.x, f[0], f[1]);
        codes_along<FMT>(r.y, f[2], f[3]);
        codes_along<FMT>(r.z, f[4], f[5]);
        codes_along<FMT>(r.w, f[6], f[7]);
        constexpr uint32_t kHalf = 32 * 128;
        uint8_t *const at = dst + (u >> 1) * Sh::BOX + (u & 1) * kHalf;
        *reinterpret_cast<uint4 *>(at + put) = make_uint4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<uint4 *>(at + (put ^ 16)) = make_uint4(f[4], f[5], f[6], f[7]);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    };
    uint32_t none[AHEAD];
    auto scales = [&](int id, float &k, float &v) {
      k = 1.f, v = 1.f;
      if (cw == 0 && id >= 0) {
        const uint32_t at = (uint32_t)id * (uint32_t)c.heads + (uint32_t)h;
        k = c.ks[at], v = c.vs[at];
      }
    };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      ids[n] = page_of(entry_of(n));
      int64_t at[2];
      none[n] = places(ids[n], n, at);
      if constexpr (Sh::STAGED) {
        copy(n, at);
      } else {
        load(c.k, at, raw_k[n]);
        load(c.v, at, raw_v[n]);
      }
      scales(ids[n], ks[n], vs[n]);
    }
    int entry = entry_of(AHEAD);
    // tile j, whose codes are in place n, and then those of tile j + AHEAD into it
    auto tile = [&](int j, auto n_c) -> bool {
      constexpr int n = decltype(n_c)::value;
      if (cw == 0) {
        float k = ks[n], e = (float)((__float_as_int(vs[n]) >> 23) - 127);
        float w = __int_as_float((254 << 23) - __float_as_int(vs[n]));  // 2^-e
        uint32_t okm = __ballot_sync(0xffffffffu, lane < GROUPS && ids[n] >= 0);
        if (__any_sync(0xffffffffu, !usual_scales(ks[n], vs[n]))) {
          const float v = kv_scale(vs[n], c.status);
          k = kv_scale(ks[n], c.status);
          e = v == v ? (float)((__float_as_int(v) >> 23) - 127) : v;
          w = v == v ? (e < kFarScale ? 0.f : exp2_approx(-e)) : v;
          if (__any_sync(0xffffffffu, e < kFarScale)) okm |= 1u << GROUPS;
        }
        if (lane < GROUPS) s_ks[j % SCALES][lane] = k, s_ve[j % SCALES][lane] = e, s_we[j % SCALES][lane] = w;
        if (lane == 0) s_ok[j % SCALES] = okm;
        __syncwarp();
        if (lane == 0) mbar_arrive(sc_full(j % SCALES));
      }
      ids[n] = page_of(entry);
      entry = entry_of(j + AHEAD + 1);
      scales(ids[n], ks[n], vs[n]);
      int64_t from[2];
      const uint32_t none_next = places(ids[n], j + AHEAD, from);
      if constexpr (Sh::STAGED) asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
      if (j >= NK && !mbar_wait(k_empty(j % NK), (j / NK - 1) & 1, abort_w, c.status, 0x6300)) return false;
      store(Sh::QBYTES + (uint32_t)(j % NK) * Sh::SLOT, k_full(j % NK), none[n], [&](int u) {
        if constexpr (Sh::STAGED) return *reinterpret_cast<const uint4 *>(smem + staged(n, 0, u));
        else return raw_k[n][u];
      });
      if constexpr (!Sh::STAGED) load(c.k, from, raw_k[n]);
      if (j >= NV && !mbar_wait(v_empty(j % NV), (j / NV - 1) & 1, abort_w, c.status, 0x6400)) return false;
      store(Sh::V0 + (uint32_t)(j % NV) * Sh::SLOT, v_full(j % NV), none[n], [&](int u) {
        if constexpr (Sh::STAGED) return *reinterpret_cast<const uint4 *>(smem + staged(n, 1, u));
        else return raw_v[n][u];
      });
      if constexpr (Sh::STAGED) copy(n, from);
      else load(c.v, from, raw_v[n]);
      none[n] = none_next;
      return true;
    };
    for (int j = 0; j < nj; j += AHEAD) {
      if (!tile(j, std::integral_constant<int, 0>())) break;
      if constexpr (AHEAD == 2)
        if (j + 1 < nj && !tile(j + 1, std::integral_constant<int, 1>())) break;
    }
    if constexpr (Sh::STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp / 4 < active) {
    // ---- softmax -----------------------------------------------------------
    const int x = warp / 4, t = threadIdx.x & 127;
    const int r = row0 + 128 * x + t;
    const int tok = r / a.group;
    const bool alive = r < rows_all && tok < count;
    const int end = alive ? len - count + tok + 1 : 0;
    const int first = row0 + 128 * x;
    const int all_end = len - count + first / a.group + 1;  // tokens that every live row sees
    const uint32_t lane_base = tm + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_o = lane_base + Sh::T_O + (uint32_t)(HD * x);
    float sc;
    {
      // q: the row's largest magnitude, then scaled and split
      const int64_t off = b * a.qs.batch + (int64_t)tok * a.qs.token +
                          (int64_t)(h * a.group + r % a.group) * a.qs.head;
      // (64 dims' loads under way at once; the second time they come from the cache)
      float mx = 0.f, v64[64];
      auto fetch = [&](int d0) {
#pragma unroll
        for (int d = 0; d < 64; d += 16) {
          if (alive && d0 + d < c.hd) {
            kv_load_row16(a.dtype, a.q, off + d0 + d, a.q_vec, v64 + d);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v64[d + i] = 0.f;
          }
        }
      };
#pragma unroll
      for (int d0 = 0; d0 < HD; d0 += 64) {
        fetch(d0);
#pragma unroll
        for (int i = 0; i < 64; ++i) mx = fmaxf(mx, fabsf(v64[i]));
      }
      const int e = q_exponent(mx);
      const float f = kv_pow2(-e);
#pragma unroll
      for (int d = 0; d < HD; d += 16) {
        if (HD > 64 && d % 64 == 0) fetch(d);
        const float *v = v64 + d % 64;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (PIECES == 2) f16_split2(v[2 * i] * f, v[2 * i + 1] * f, hi[i], lo[i]);
          else hi[i] = pack_f16(v[2 * i] * f, v[2 * i + 1] * f);
        }
#pragma unroll
        for (int w = 0; w < PIECES; ++w) {
          const uint32_t *p = w ? lo : hi;
          if constexpr (Sh::QT) {
            asm volatile(
                "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(
                    lane_base + Sh::T_Q + (uint32_t)((x * PIECES + w) * (HD / 2) + d / 2)),
                "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]), "r"(p[6]),
                "r"(p[7])
                : "memory");
          } else {
            uint8_t *row = smem + (uint32_t)((x * PIECES + w) * Sh::BOXES + d / 64) * Sh::QBOX + t * 128;
            const int c0 = (d % 64) / 8;
            *reinterpret_cast<uint4 *>(row + ((c0 ^ (t & 7)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<uint4 *>(row + (((c0 + 1) ^ (t & 7)) << 4)) = make_uint4(p[4], p[5], p[6], p[7]);
          }
        }
      }
      sc = a.scale * 1.4426950408889634f * kv_pow2(e);
      if (mx == CUDART_INF_F) sc = CUDART_NAN_F;  // also where all its scores are -inf
      if constexpr (Sh::QT) tmem_wait_st();
      else fence_async();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    // where this row's sum of flushed O stands: its partial result, or its output
    const int64_t at = out_row(r < rows_all ? r : 0);
    const KvOut sum_out = splits > 1 ? KvOut{a.ws, nullptr, TT_DTYPE_F32} : a.out;
    const int64_t sum_at = splits > 1 ? part(r) * HD : at;
    const int sum_dims = alive ? (splits > 1 ? HD : c.hd) : 0;
    // ... or, a row tile at a time with 4 dims of its rows side by side
    float4 *const sums = Sh::SUM_WS ? reinterpret_cast<float4 *>(a.ws + part(first) * HD) + t
                                    : reinterpret_cast<float4 *>(smem + Sh::SUM0) + x * 128 * (HD / 4) + t;
    float m = -CUDART_INF_F, l = 0.f, beta = 0.f;  // beta: what the sum is scaled by when read next
    // O_x holds the products up to tile j - 1's, while tile j's scores are there but
    // not yet its p: tile j - 2's product came before those scores, so one parity is
    // enough.
    auto wait_o_before = [&](int j) {
      mbar_wait(o_done(x), (j - 1) & 1, abort_w, c.status, 0x6700);
      fence_after();
    };
    // tile j's scores s[0 .. 63] to p, in the buffer that they came from
    auto softmax = [&](int j, bool open, float *s, uint32_t t_s) {
      float kc[GROUPS], ve[GROUPS], we[GROUPS], top = -CUDART_INF_F;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        kc[g] = s_ks[j % SCALES][g] * sc;
        ve[g] = s_ve[j % SCALES][g];
        we[g] = s_we[j % SCALES][g];
      }
      if (!open) {  // the same for the warp
        const int left = end - (j0 + j) * TOK;  // tokens of the tile that this row sees
        const uint32_t okm = s_ok[j % SCALES];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int n = (okm >> g) & 1u ? left - 16 * g : 0;
          // a group that the row sees nothing of: its scales, NaN perhaps, do not count
          if (n <= 0) kc[g] = 1.f, ve[g] = 0.f, we[g] = 0.f;
          // a factor that underflowed would make NaN of a masked score
          if (kc[g] < FLT_MIN) kc[g] = FLT_MIN;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[16 * g + i] = i < n ? s[16 * g + i] : -CUDART_INF_F;
        }
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const float *v = s + 16 * g;
        float a0 = fmax3(v[0], v[1], v[2]), a1 = fmax3(v[3], v[4], v[5]);
        a0 = fmax3(a0, v[6], v[7]), a1 = fmax3(a1, v[8], v[9]);
        a0 = fmax3(a0, v[10], v[11]), a1 = fmax3(a1, v[12], v[13]);
        top = fmaxf(top, fmaf(fmax3(fmaxf(a0, a1), v[14], v[15]), kc[g], ve[g]));
      }
      constexpr float kLazy = 8.f;
      const bool raise = top > m + kLazy || (m == -CUDART_INF_F && top > m);
      if (__any_sync(0xffffffffu, raise)) {
        const float mn = raise ? ceilf(top) : m;
        const float alpha = raise ? exp2_approx(m - mn) : 1.f;  // 0 from -inf
        if ((j & (flush - 1)) != 0 && __any_sync(0xffffffffu, raise && m != -CUDART_INF_F)) {
          wait_o_before(j);
#pragma unroll 1
          for (int d = 0; d < HD; d += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st16(t_o + d, o);
          }
        }
        beta *= alpha;
        l = rescale(l, m - mn, alpha);
        m = mn;
      }
      const float ref = 7.f - (m == -CUDART_INF_F ? 0.f : m);
      if (!open && s_ok[j % SCALES] >> GROUPS) {  // weights that p may not stand for
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          if (!(ve[g] < kFarScale)) continue;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += exp2_approx(fmaf(s[16 * g + i], kc[g], ref));
          l += sum;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
#pragma unroll
        for (int g2 = 0; g2 < 2; ++g2) {
          const int g = 2 * half + g2;
          const float bs = ve[g] + ref;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int col = 16 * g + 2 * i;
            const float2 y = fma_pair(make_float2(s[col], s[col + 1]), make_float2(kc[g], kc[g]),
                                      make_float2(bs, bs));
            const float2 p = make_float2(exp2_approx(y.x), exp2_approx(y.y));
            sum = add_pair(sum, p);
            const float2 hi = make_float2(upper11(p.x), upper11(p.y));
            const float2 lo = fma_pair(hi, make_float2(-1.f, -1.f), p);
            w[8 * g2 + i] = pack_f16(hi.x, hi.y);
            w[16 + 8 * g2 + i] = pack_f16(lo.x, lo.y);
          }
          l = fmaf(sum.x + sum.y, we[g], l);
        }
        tmem_st16(t_s + 32u * half, w);
        tmem_st16(t_s + 32u * half + 16u, w + 16);
      }
    };
    // o += beta times the flushed sums of dims d .. d + 15
    auto add_sums = [&](int d, bool any, uint32_t *o) {
      if (!any) return;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = sums[(d / 4 + i) * 128];
        o[4 * i] = __float_as_uint(fmaf(v.x, beta, __uint_as_float(o[4 * i])));
        o[4 * i + 1] = __float_as_uint(fmaf(v.y, beta, __uint_as_float(o[4 * i + 1])));
        o[4 * i + 2] = __float_as_uint(fmaf(v.z, beta, __uint_as_float(o[4 * i + 2])));
        o[4 * i + 3] = __float_as_uint(fmaf(v.w, beta, __uint_as_float(o[4 * i + 3])));
      }
    };
    for (int j = 0; j < nj; ++j) {
      const int t0 = (j0 + j) * TOK, buf = j & 1;
      mbar_wait(s_full(x, buf), (j >> 1) & 1, abort_w, c.status, 0x6600);
      mbar_wait(sc_full(j % SCALES), (j / SCALES) & 1, abort_w, c.status, 0x6500);
      // whether every live row sees every token (the same for the warp)
      const bool open = t0 + TOK <= all_end && s_ok[j % SCALES] == (1u << GROUPS) - 1u;
      fence_after();
      if (j > 0 && (j & (flush - 1)) == 0) {
        wait_o_before(j);
        if constexpr (Sh::SUM_WS) {
#pragma unroll 1
          for (int d = 0; d < HD; d += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + d, o);
            tmem_wait_ld();
            add_sums(d, j > flush, o);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4 *>(sums)[(d / 4 + i) * 128] =
                  make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        } else if constexpr (Sh::SUM_SMEM) {
#pragma unroll
          for (int d = 0; d < HD; d += 32) {
            float o[32];
            tmem_ld32(t_o + d, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 v = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
              if (j > flush) {
                const float4 w = sums[(d + i) / 4 * 128];
                v.x = fmaf(w.x, beta, v.x), v.y = fmaf(w.y, beta, v.y);
                v.z = fmaf(w.z, beta, v.z), v.w = fmaf(w.w, beta, v.w);
              }
              sums[(d + i) / 4 * 128] = v;
            }
          }
        } else {
#pragma unroll 1
          for (int d = 0; d < HD; d += 32) {
            float o[32], v[32];
            const bool mine = d < sum_dims, both = d + 16 < sum_dims;
            if (j > flush) {
              if (mine) kv_load_sum16(sum_out, sum_at + d, v);
              if (both) kv_load_sum16(sum_out, sum_at + d + 16, v + 16);
            }
            __syncwarp();
            tmem_ld32(t_o + d, o);
            tmem_wait_ld();
            if (j > flush) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = fmaf(v[i], beta, o[i]);
            }
            if (mine) kv_store_sum16(sum_out, sum_at + d, o);
            if (both) kv_store_sum16(sum_out, sum_at + d + 16, o + 16);
          }
        }
        beta = 1.f;
      }
      const uint32_t t_s = lane_base + Sh::T_S + (uint32_t)(TOK * (2 * x + buf));
      float s[TOK];
      tmem_ld32(t_s, s);
      tmem_ld32(t_s + 32u, s + 32);
      tmem_wait_ld();
      softmax(j, open, s, t_s);
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full(x, buf));
    }
    mbar_wait(o_final(x), 0, abort_w, c.status, 0x6800);
    fence_after();
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (Sh::SUM_WS && nj > flush) {
#pragma unroll 1
      for (int d = 0; d < HD; d += 16) {
        uint32_t o[16];
        tmem_ld16(t_o + d, o);
        tmem_wait_ld();
        add_sums(d, true, o);
        tmem_st16(t_o + d, o);
      }
      tmem_wait_st();
      // the rows' partial results go where the others' sums stand
      if (splits > 1) asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");
    }
#pragma unroll
    for (int d = 0; d < HD; d += 16) {
      uint32_t o[16];
      tmem_ld16(t_o + d, o);
      tmem_wait_ld();
      float v[16];
      if (!Sh::SUM_WS && nj > flush && (Sh::SUM_SMEM || d < sum_dims)) {
        if constexpr (Sh::SUM_SMEM) {
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 w = sums[(d + i) / 4 * 128];
            v[i] = w.x, v[i + 1] = w.y, v[i + 2] = w.z, v[i + 3] = w.w;
          }
        } else {
          kv_load_sum16(sum_out, sum_at + d, v);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(fmaf(v[i], beta, __uint_as_float(o[i])));
      }
      if (splits > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint4 *>(a.ws + part(r) * HD + d + i) =
              make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
      } else if (d < c.hd && r < rows_all) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = end > 0 && l != 0.f ? __uint_as_float(o[i]) * inv : 0.f;
        kv_store_row16(a.out, at + d, v);
      }
    }
    if (splits > 1) {
      part_ml[2 * part(r)] = m;
      part_ml[2 * part(r) + 1] = end > 0 ? l : 0.f;
    }
    fence_before();
  } else {
    // a tile without a live row: zeros
    const int r = row0 + threadIdx.x;
    if (splits > 1) {
      part_ml[2 * part(r)] = -CUDART_INF_F;
      part_ml[2 * part(r) + 1] = 0.f;
    } else if (r < rows_all) {
      const float z[16] = {};
      for (int d = 0; d < c.hd; d += 16) kv_store_row16(a.out, out_row(r) + d, z);
    }
  }
  __syncthreads();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm));
}

// Joins the splits of each row, in their order; one thread per 4 dims.
template <int HD, int FMT>
__global__ void __launch_bounds__(256) kv_attention_tiles_join_kernel(KvAttentionArgs a,
                                                                      int64_t rows_padded,
                                                                      int splits) {
  pdl_trigger();
  pdl_wait();
  const KvView &c = a.c;
  const int rows_all = a.tokens * a.group;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int d = (int)(i % (HD / 4)) * 4;
  const int64_t r64 = i / (HD / 4);
  if (r64 >= rows_all || d >= c.hd) return;
  const int r = (int)r64, h = blockIdx.y, b = blockIdx.z;
  const float *ml = a.ws + (int64_t)splits * c.batch * c.heads * rows_padded * HD;
  auto part = [&](int s) { return (((int64_t)s * c.batch + b) * c.heads + h) * rows_padded + r; };
  float m = -CUDART_INF_F;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[2 * part(s)]);
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float ms = ml[2 * part(s)], ls = ml[2 * part(s) + 1];
    if (ls == 0.f) continue;  // a split that the row sees nothing of (its O may not exist)
    const float f = ms == m || !(ls == ls) ? 1.f : exp2_approx(ms - m);
    const float4 v = *reinterpret_cast<const float4 *>(a.ws + part(s) * HD + d);
    l += rescale(ls, ms - m, f);
    o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]);
    o[2] = fmaf(v.z, f, o[2]), o[3] = fmaf(v.w, f, o[3]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = (((int64_t)b * a.tokens + r / a.group) * a.heads + h * a.group + r % a.group) * c.hd + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] *= inv;
  kv_store_out4(a.out, at, o);
}

struct TilePlan {
  int row_tiles, splits;
  int64_t rows_padded;
  size_t ws_bytes;
};

template <int HD, int PIECES>
TilePlan tile_plan(const KvView &c, int dtype, int64_t tokens, int heads, int sms) {
  using Sh = TcShape<HD, PIECES>;
  TilePlan p{};
  const int64_t rows = tokens * (heads / c.heads);
  p.row_tiles = (int)ceil_div(rows, 128 * Sh::MT);
  p.rows_padded = (int64_t)p.row_tiles * 128 * Sh::MT;
  const int64_t ctas = (int64_t)p.row_tiles * c.heads * c.batch;
  const int64_t tiles = ceil_div((int64_t)c.columns << c.page_log2, Sh::TOK);
  // one CTA an SM: too few of them share the tokens, four tiles each at least
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(sms / std::max<int64_t>(ctas, 1), tiles / 4));
  const size_t rows_all = (size_t)c.batch * c.heads * p.rows_padded;
  if (p.splits > 1) p.ws_bytes = p.splits * rows_all * (HD + 2) * sizeof(float);
  else if (Sh::SUM_WS && tiles > Sh::flush(dtype)) p.ws_bytes = rows_all * HD * sizeof(float);
  return p;
}

template <int HD, int FMT, int PIECES>
int launch_tiles(const KvAttentionArgs &a, cudaStream_t stream) {
  using Sh = TcShape<HD, PIECES>;
  int sms = 0;
  const int rc = kv_sm_count(&sms);
  if (rc != TT_OK) return rc;
  if ((int64_t)a.tokens * a.group > kKvMost || a.c.batch > 65535 || a.c.heads > 65535)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_attention: too many rows, heads or sequences");
  const TilePlan p = tile_plan<HD, PIECES>(a.c, a.dtype, a.tokens, a.heads, sms);
  if ((int64_t)p.row_tiles * a.c.heads > INT32_MAX)
    return fail(TT_ERR_UNSUPPORTED, "tt_kv_attention: too many rows");
  auto *kern = kv_attention_tiles_kernel<HD, FMT, PIECES>;
  static KvSmemSet set;
  // (a block that started with fewer registers than its warps take over would wait for good)
  const int set_rc = set.ensure(reinterpret_cast<const void *>(kern), Sh::SMEM,
                                Sh::SHIFT_REGS ? Sh::START_REGS : 0);
  if (set_rc != TT_OK) return set_rc;
  KvAttentionArgs args = a;
  args.test_hold_back = g_armed_timeout.exchange(false);  // test switch: this launch takes it
  TT_CUDA_TRY(launch_kernel(kern, dim3(p.row_tiles * a.c.heads, a.c.batch, p.splits), dim3(Sh::THREADS),
                            Sh::SMEM, stream, 1, args, p.row_tiles, p.splits));
  if (p.splits > 1)
    TT_CUDA_TRY(launch_kernel(kv_attention_tiles_join_kernel<HD, FMT>,
                              dim3((unsigned)ceil_div((int64_t)a.tokens * a.group * (HD / 4), 256),
                                   a.c.heads, a.c.batch),
                              dim3(256), 0, stream, 1, a, p.rows_padded, p.splits));
  return TT_OK;
}

template <class F>
int for_tiles(const KvView &c, int dtype, F &&f) {
  const bool i8 = c.format == TT_KV_INT8, two = dtype == TT_DTYPE_F32;
  using std::integral_constant;
#define TT_KV_TILES(HD, P)                                                                            \
  return i8 ? f(integral_constant<int, HD>(), integral_constant<int, TT_KV_INT8>(), integral_constant<int, P>()) \
            : f(integral_constant<int, HD>(), integral_constant<int, TT_KV_E4M3>(), integral_constant<int, P>())
  if (c.hd <= 64) {
    if (two) TT_KV_TILES(64, 2);
    TT_KV_TILES(64, 1);
  }
  if (c.hd <= 128) {
    if (two) TT_KV_TILES(128, 2);
    TT_KV_TILES(128, 1);
  }
  if (two) TT_KV_TILES(256, 2);
  TT_KV_TILES(256, 1);
#undef TT_KV_TILES
}

}  // namespace

size_t kv_attention_tiles_ws_bytes(const KvView &c, int dtype, int64_t tokens, int heads) {
  int sms = 0;
  if (kv_sm_count(&sms) != TT_OK) return 0;
  size_t n = 0;
  for_tiles(c, dtype, [&](auto hd, auto, auto pieces) {
    n = tile_plan<decltype(hd)::value, decltype(pieces)::value>(c, dtype, tokens, heads, sms).ws_bytes;
    return TT_OK;
  });
  return n;
}

int launch_kv_attention_tiles(const KvAttentionArgs &a, cudaStream_t stream) {
  return for_tiles(a.c, a.dtype, [&](auto hd, auto fmt, auto pieces) {
    return launch_tiles<decltype(hd)::value, decltype(fmt)::value, decltype(pieces)::value>(a, stream);
  });
}

}  // namespace tt

extern "C" int tt_test_arm_kv_wait_timeout(void) {
  tt::g_armed_timeout.store(true);
  return TT_OK;
}
