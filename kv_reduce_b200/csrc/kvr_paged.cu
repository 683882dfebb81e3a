// Paged key-value cache: append, attention of the new tokens, and the running
// sum of attention weights per cached token (sm_100a).  No reference
// counterpart: the reference keeps its target model's cache in transformers.
//
// Attention.  Query t of sequence b (length L, the T new tokens included)
// stands at i = L - T + t and sees the tokens j <= i, with a window w only
// those with j > i - w or j < sinks:
//   o_i = sum_j 2^(x_ij - m) v_j / sum_j 2^(x_ij - m),  x_ij = scale*log2(e) q_i.k_j
// in one pass over the tokens with the running maximum m and sum l in fp32.
//
// What bounds it: the bytes of K and V.  A token of one KV head is 4*D bytes
// and 4*D*R operations for the R = T*q_heads/kv_heads query rows that share
// it, so R operations per byte, below what the tensor cores do; but the
// softmax between the two products has to keep up as well, and the loads must
// never pause.  So the threads do as little per tile as they can:
//  * Work is a flat list of token tiles (sequence, KV head, row tile, tile),
//    cut into equal ranges, one per CTA.  Lengths are read on the device, so
//    a ragged batch is balanced to one tile without the host knowing it.
//  * One warp looks up pages and fills a ring of K and V tiles, on across
//    sequence boundaries.  Pages of a multiple of 4 tokens come by TMA, a box
//    or more per page; others row by row (cp.async).
//  * One thread issues the products (tcgen05).  Both are transposed: scores^T
//    = K Q^T has a tile's 128 tokens in the 128 lanes of tensor memory and
//    only as many columns as there are rows, and output^T = V^T P^T the head
//    dimension; so no lane is spent on padding the few query rows to 128, K
//    and V are read where the copies put them, and a thread of the four
//    softmax warps has one token and every row: R exponentials a tile.
//  * The next tile's scores are computed while this one's softmax runs.  The
//    output stays in tensor memory; it is read back to be rescaled only in
//    the tiles where a row's maximum has moved too far.
//  * A sequence that several CTAs share is joined by the last of them to
//    arrive, in the order of the CTAs: the result does not depend on timing.
//
// Measured (16-bit types, against a copy's 6547 GB/s, on several GPUs): 16
// sequences of 16K to 32K, 32 query and 8 KV heads of 128, 1.61 GB in 239 to
// 244 us, 6600 to 6740 GB/s; 64 of 4K to 16K with 5 new tokens each, 12 and 2
// heads of 128, 0.67 GB in 121 to 132 us, 5080 to 5530 GB/s; 32 of up to 8K, 32
// and 8 heads of 64, 0.27 GB in 51 us, 5270 GB/s; one of 32K, 12 and 2 heads
// of 128, 34 MB in 17 us, of which about 5 are the start (lengths, page
// numbers, first tiles) and 4 the join.
#include "kvr_ring.cuh"

#include <cuda.h>

#include <algorithm>
#include <cfloat>
#include <cstring>

namespace kvr {
namespace paged {

using namespace ring;

constexpr int kWarps = 4;                     // consumers
constexpr int kConsumers = 32 * kWarps;
constexpr int kLoadWarp = 4, kMmaWarp = 5;
constexpr int kThreads = kConsumers + 64;
constexpr int kGroup = 16;                    // CTAs a join takes at a time

template <bool HALF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool HALF>
__device__ __forceinline__ float to_float(uint16_t w) {
  if constexpr (HALF) return __half2float(__ushort_as_half(w));
  else return bf16_bits_to_f32(w);
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }

// A box of `rows` tokens x 64 elements of one head of one page.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int col, int row, int head,
                                        int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];\n" ::"r"(dst),
      "l"(map), "r"(bar), "r"(col), "r"(row), "r"(head), "r"(page)
      : "memory");
}

// 16 bytes from `src`, or zeros.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

struct Params {
  const uint16_t* q;
  int64_t q_b, q_h, q_t;
  const uint16_t* k;
  int64_t k_page, k_head, k_row;
  const uint16_t* v;
  int64_t v_page, v_head, v_row;
  const int* table;
  int64_t table_b;
  int num_pages, page, page_shift;
  uint32_t page_magic;   // j / page = j * page_magic >> page_shift for j < 2^30
  const int* lengths;
  const int* counts;   // [B] or null: how many of the T new tokens a sequence has, the last ones
  uint16_t* out;
  float* lse;       // [B, HQ, T] or null
  float* scores;    // [B, HKV, R, score_stride] or null: x_ij for the weights kernel
  float2* row_stat; // [B, HKV, R], with scores: reference and log2 of the sum; inf, inf for a row that is no token's
  int64_t score_stride;
  int B, HQ, HKV, T, G, R, row_tiles, window, sinks, cap;
  float scale2;     // scale * log2(e)
  int ctas;
  float* part_o;    // [3 * ctas][ROWS][D]: two parts of each CTA, group sums
  float* part_ml;   // [3 * ctas][ROWS][2]
  int* counters;    // [2 * ctas], zero on entry and on exit
  int box;          // tokens of a TMA box
};

template <int D, int N>
struct Cfg {
  static constexpr int TILE = 128;                   // tokens: the 128 lanes of a score tile
  static constexpr int HALVES = D / 64;
  static constexpr int PIECES = D / 8;
  static constexpr int HALF_BYTES = TILE * 128;      // 64 elements of every token, 128-byte rows
  static constexpr int UNIT = HALVES * HALF_BYTES;   // K or V of a tile
  static constexpr int Q_BYTES = N * D * 2;
  static constexpr int P_ROW = N == 16 ? 64 : 128;          // bytes of a token's weights (a swizzle row)
  static constexpr int P_BYTES = TILE * 4 * N;
  // Two CTAs per SM where the ring still holds three units or more; else one with a longer ring.  (One CTA and six
  // units in place of two and three each: 73 for 50 us on 32 sequences of up to 8K, 37 for 30 us on 128 windows of 1K,
  // the same on 16 sequences of 16K to 32K, and 16 for 17 us on a single one, where the join is shorter.)
  static constexpr int CTAS = N == 16 || D == 64 ? 2 : 1;
  static constexpr int UNITS = CTAS == 2 ? (D == 128 ? 3 : N == 16 ? 6 : 5) : N == 32 ? 6 : 5;
  static constexpr int DESCS = 8;
  static constexpr int OFF_Q = UNITS * UNIT;
  static constexpr int OFF_P = OFF_Q + Q_BYTES;
  static constexpr int OFF_DESC = OFF_P + P_BYTES;
  static constexpr int OFF_ROWS = OFF_DESC + DESCS * 64;   // float [12][N]: reference, alpha, position, row, 4 maxima, 4 sums
  static constexpr int OFF_BAR = OFF_ROWS + 12 * N * 4;
  static constexpr int BARS = 2 * UNITS + DESCS + 4 + 3;
  static constexpr int OFF_MISC = OFF_BAR + BARS * 8;
  static constexpr int SMEM = OFF_MISC + 80 + 1024;        // 1 KB to align the ring
  static constexpr int TMEM = 4 * N;                       // columns: two score tiles, output and its rest

  // Weight of (token t, row r), rounded (part 0) or its rest (part 1): token-major, the two parts side by side.
  static __device__ __forceinline__ int p_at(int t, int r, int part) {
    const int piece = (N == 64 ? 0 : part * (N / 8)) + (r >> 3);
    return (N == 64 ? part * TILE * 128 : 0) + t * P_ROW + ((piece ^ (N == 16 ? (t >> 1) & 3 : t & 7)) << 4) + (r & 7) * 2;
  }
};

// The reference of a row that no token has been seen by: far below any score.
constexpr float kUnseen = -FLT_MAX;

// x factor - m of two rows, the product rounded first.  Fused, it would keep the
// digits that are rounded off in m and in tiles that a mask cuts: half the
// spacing of numbers like m, which from 2^27 on is more than the exponents'
// range.  (m is taken off by a multiplication with -1 and an addition: a packed
// mul.rn and add.rn do come out fused.)
__device__ __forceinline__ void two_exponents(float& x0, float& x1, float factor, float2 m) {
  asm("{\n.reg .b64 x, f, m, one;\nmov.b64 x, {%0, %1};\nmov.b64 f, {%2, %2};\nmov.b64 m, {%3, %4};\n"
      "mov.b64 one, {%5, %5};\nmul.rn.f32x2 x, x, f;\nfma.rn.f32x2 x, m, one, x;\nmov.b64 {%0, %1}, x;\n}\n"
      : "+f"(x0), "+f"(x1)
      : "f"(factor), "f"(m.x), "f"(m.y), "f"(-1.f));
}

// The weights' range in the second product.  A reference is a maximum so far,
// less kBelow, and moves when an exponent passes kBelow + 8; the weights' rest
// is multiplied by kRest and has accumulators of its own.  bf16 has fp32's
// range and needs neither.  fp16 ends at 2^-24 (2^-25 rounds to 0): a token 17
// below the largest score, natural log, had no weight left, and a long cache
// has many of those.  With both, weights stay below 2^15, the largest is 2^7 or
// more, and hi + rest is off by 2^-36 at most: 2^-43 of the largest weight a
// token.
template <bool HALF>
constexpr float kBelow = HALF ? 7.f : 0.f;
template <bool HALF>
constexpr float kRest = HALF ? 2048.f : 1.f;

struct Desc {
  int first, last, full, token0;   // full: every row sees every token; last: 2 where the sequence is too long for its table
  int b, h, rt, len;
  int n_tiles, seg_start;          // of the segment: tiles, flat index of the first
  int whole;                       // with `last`: all of the segment's tiles are this CTA's
  uint32_t groups;                 // 16-token groups that a query sees, a bit each (one at least)
  uint32_t bad[4];   // tokens on pages outside the pool, a bit each
};
static_assert(sizeof(Desc) <= 64, "");

// The flat list counts a segment as its tiles and kHead more in front: what it
// costs beside its tiles (its queries, a first tile without a reference, its
// output or part, the join), so that a CTA does not end up with many short
// ones.  (1, 2, 3, 4: 131, 129, 128, 124 us for 64 sequences of 4K to 16K with
// 5 new tokens; 32.1, 30.0, 29.1, 27.9 us for 8 windows of 4K; others within 2%.)
constexpr int kHead = 4;

// `total` units cut into `n` ranges of equal size, the first ones a unit longer.
struct Cut {
  int q, r;
  __device__ __forceinline__ Cut(int total, int n) : q(total / n), r(total % n) {}
  __device__ __forceinline__ int begin(int c) const { return c * q + min(c, r); }
  __device__ __forceinline__ int owner(int g) const { return g < r * (q + 1) ? g / (q + 1) : r + (g - r * (q + 1)) / q; }
};

// The tiles a sequence's queries look at: with a window, `ns` tiles that hold
// the sinks, then the tiles from `lo_tile` on.
struct Span {
  int n, ns, lo_tile, lo;
};
constexpr int kTile = 128;
__device__ __forceinline__ Span span_of(const Params& p, int len) {
  Span s;
  const int total = (len + kTile - 1) / kTile;
  s.lo = p.window > 0 ? max(0, max(len - p.T, 0) - p.window + 1) : 0;
  s.lo_tile = min(s.lo / kTile, max(total - 1, 0));
  s.ns = min((p.sinks + kTile - 1) / kTile, s.lo_tile);
  s.n = max(1, s.ns + total - s.lo_tile);   // an empty sequence gets one tile, to write its zero rows
  return s;
}
__device__ __forceinline__ int length_of(const Params& p, int b) { return min(max(p.lengths[b], 0), p.cap); }

// ---- tensor memory and the 5th-generation tensor cores
// Shared-memory operand in rows of 128 (or 64) bytes with the swizzle of that
// width, patterns of 8 rows.  The rows are the operand's own (K-major) or its
// depth (transposed); `next`: bytes to the next row's width of elements of a
// transposed operand.
template <int ROW = 128>
__device__ __forceinline__ uint64_t operand(uint32_t addr, int next) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((next >> 4) & 0x3fff) << 16 | (uint64_t)(8 * ROW >> 4) << 32 |
         1ull << 46 | (ROW == 128 ? 2ull : 4ull) << 61;
}
// bf16 or fp16 operands, fp32 accumulation, M x N, both operands transposed or neither.
__device__ __forceinline__ constexpr uint32_t mma_kind(bool half, int m, int n, bool transposed) {
  return 1u << 4 | (half ? 0u : 1u) << 7 | (half ? 0u : 1u) << 10 | (transposed ? 3u : 0u) << 15 |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(kind), "r"((uint32_t)add)
      : "memory");
}
// The barrier is arrived at when all tensor-core work issued so far is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// 16 columns of this warp's 32 lanes, a lane to a thread.
__device__ __forceinline__ void tmem_load(uint32_t addr, float* x) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]),
        "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const float* x) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};\n" ::"f"(x[0]),
      "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "f"(x[8]), "f"(x[9]), "f"(x[10]),
      "f"(x[11]), "f"(x[12]), "f"(x[13]), "f"(x[14]), "f"(x[15]), "r"(addr)
      : "memory");
}
// (the registers are named so that nothing reads them before the wait)
__device__ __forceinline__ void tmem_wait_load(float* x) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]),
                 "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// Maxima or sums of NR rows over the warp's lanes, halving the rows a lane
// deals with at every exchange: NR - 1 exchanges and a few instead of 5 NR.
// Row r ends in lane r 32 / NR (NR = 64: rows 2 l and 2 l + 1 in lane l).
template <int NR, int BIT, bool SUM>
__device__ __forceinline__ void rows_join(float* v, int lane) {
  if constexpr (BIT >= 1) {
    if constexpr (NR > 1) {
      const bool up = lane & BIT;
#pragma unroll
      for (int k = 0; k < NR / 2; ++k) {
        const float mine = up ? v[k + NR / 2] : v[k], other = up ? v[k] : v[k + NR / 2];
        const float got = __shfl_xor_sync(0xffffffffu, other, BIT);
        v[k] = SUM ? mine + got : fmaxf(mine, got);
      }
      rows_join<NR / 2, BIT / 2, SUM>(v, lane);
    } else {
      const float got = __shfl_xor_sync(0xffffffffu, v[0], BIT);
      v[0] = SUM ? v[0] + got : fmaxf(v[0], got);
      rows_join<1, BIT / 2, SUM>(v, lane);
    }
  }
}
// ... written to `to` (v is used up).
template <int NR, bool SUM>
__device__ __forceinline__ void store_rows(float* v, float* to, int lane) {
  rows_join<NR, 16, SUM>(v, lane);
  if constexpr (NR >= 32) {
#pragma unroll
    for (int k = 0; k < NR / 32; ++k) to[lane * (NR / 32) + k] = v[k];
  } else {
    constexpr int SHIFT = NR == 16 ? 1 : 2;
    if ((lane & ((1 << SHIFT) - 1)) == 0) to[lane >> SHIFT] = v[0];
  }
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// Barrier of the consumers; true for all when it is for one.
__device__ __forceinline__ bool consumer_any(bool x) {
  int r;
  asm volatile("{\n.reg .pred a, b;\nsetp.ne.s32 a, %1, 0;\nbar.red.or.pred b, 1, 128, a;\nselp.s32 %0, 1, 0, b;\n}\n"
               : "=r"(r)
               : "r"((int)x)
               : "memory");
  return r != 0;
}

template <bool HALF, int D, int N, bool TMA>
__global__ void __launch_bounds__(kThreads, Cfg<D, N>::CTAS) attention_kernel(const __grid_constant__ Params p,
                                                                              const __grid_constant__ CUtensorMap kmap,
                                                                              const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D, N>;
  constexpr int TILE = C::TILE, U = C::UNITS, ROWS = N;
  extern __shared__ uint8_t raw_smem[];
  // the swizzle pattern of a tile follows address bits 7..9: align the ring to 1 KB
  uint8_t* smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto desc_at = [&](int i) { return reinterpret_cast<Desc*>(smem + C::OFF_DESC + (i & (C::DESCS - 1)) * 64); };
  float* mu_s = reinterpret_cast<float*>(smem + C::OFF_ROWS);   // references of the rows' exponents
  float* alpha_s = mu_s + N;
  int* pos_s = reinterpret_cast<int*>(alpha_s + N);
  int* row_s = pos_s + N;          // the rows of the output
  float* smax = alpha_s + 3 * N;   // [4][N]
  float* ssum = smax + 4 * N;      // [4][N]
  // (in this order)  A ring unit's data is there / is read; a tile's descriptor is there (before its data); score tile done / read;
  // P written; the output up to a tile done; a segment's queries written.
  const uint32_t full = sbase + C::OFF_BAR, empty = full + 8 * U, ready = empty + 8 * U, s_full = ready + 8 * C::DESCS,
                 s_empty = s_full + 16, p_full = s_empty + 16, o_done = p_full + 8, q_full = o_done + 8;
  int* s_start = reinterpret_cast<int*>(smem + C::OFF_MISC);   // [7]
  int* s_scan = s_start + 8;                                   // [kThreads / 32]
  int* s_last = s_scan + kThreads / 32;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_last + 1);
  int* s_add = s_last + 2;                                     // the output holds something before its first product

  if (tid < C::BARS) {
    // (s_empty and p_full are arrived at by the consumers' warps, the others by one thread)
    const uint32_t bar = full + 8 * tid;
    bar_init(bar, (bar >= s_empty && bar <= p_full) ? kWarps : 1);
    bar_init_fence();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)),
                 "r"(C::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    tc_before_sync();
  }
  auto free_tmem = [&]() {
    if (warp == kMmaWarp)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(*s_tmem), "r"(C::TMEM));
  };
  pdl_enter();

  // ---- this CTA's range of the flat tile list
  const int HR = p.HKV * p.row_tiles;
  int total, ctas, g0, count;   // units in all, CTAs that take part, this one's first unit, and its tiles
  {
    // three warps find the first unit's sequence, three the end's
    constexpr int kHalf = kThreads / 2;
    const int half = tid >= kHalf, t = tid - half * kHalf;
    const int per = (p.B + kHalf - 1) / kHalf;
    const int b0 = min(t * per, p.B), b1 = min(b0 + per, p.B);
    int mine = 0, raw0 = 0;
    for (int b = b0; b < b1; ++b) {
      const int raw = p.lengths[b];
      if (b == b0) raw0 = raw;
      mine += span_of(p, min(max(raw, 0), p.cap)).n + kHead;
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int before = incl - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kHalf / 32; ++w) {
      if (w + half * (kHalf / 32) < warp) before += s_scan[w];   // (both halves' sums are the same)
      total += s_scan[w];
    }
    total *= HR;
    ctas = min(p.ctas, total);
    const int me = blockIdx.x;
    if (me >= ctas) {
      free_tmem();
      return;
    }
    const Cut cut(total, ctas);
    g0 = cut.begin(me);
    const int g1 = cut.begin(me + 1), g = half ? g1 : g0;
    if (mine > 0 && before * HR <= g && g < (before + mine) * HR) {   // this thread's sequences hold unit g
      int b = b0, at = before, raw = raw0;
      int nb = span_of(p, min(max(raw, 0), p.cap)).n + kHead;
      while (g >= (at + nb) * HR) {
        at += nb;
        raw = p.lengths[++b];
        nb = span_of(p, min(max(raw, 0), p.cap)).n + kHead;
      }
      const int off = g - at * HR, hr = off / nb, in_seg = off - hr * nb;
      // tiles in front of unit g: the units less the heads in front
      const int tiles = g - kHead * (b * HR + hr) - min(in_seg, kHead);
      if (half) {
        s_start[6] = tiles;
      } else {
        s_start[0] = b;
        s_start[1] = raw;
        s_start[2] = hr;
        s_start[3] = max(in_seg - kHead, 0);
        s_start[4] = tiles;
      }
    }
    if (tid == 0 && g1 == total) s_start[6] = total - kHead * p.B * HR;
    __syncthreads();
    tc_after_sync();
    count = s_start[6] - s_start[4];
    if (count == 0) {   // nothing but heads
      __syncwarp();
      free_tmem();
      return;
    }
  }
  const uint32_t tmem = *s_tmem, tmem_o = tmem + 2 * N;
  bool failed = false;

  if (warp == kMmaWarp) {
    // ---------------------------------------- tensor cores: one thread issues
    // (the warp stays together around it, so that the operands are made in uniform registers)
    constexpr uint32_t s_kind = mma_kind(HALF, 128, N, false), o_kind = mma_kind(HALF, D, 2 * N, true);
    const uint64_t q_op = operand(sbase + C::OFF_Q, 16);
    const uint64_t p_op = operand<C::P_ROW>(sbase + C::OFF_P, TILE * 128);
    int queries = 0;   // segments whose queries have been waited for
    // scores^T of tile i: 128 tokens x N rows
    auto scores = [&](int i, bool first) {
      const int u = 2 * i, slot = u % U, sb = i & 1;
      if (first) bar_wait(q_full, queries++ & 1, failed);
      bar_wait(full + 8 * slot, (u / U) & 1, failed);
      if (i >= 2) bar_wait(s_empty + 8 * sb, (i / 2 - 1) & 1, failed);
      tc_after_sync();
      __syncwarp();
      const uint64_t k_op = operand(sbase + slot * C::UNIT, 16);
      if (elect_one()) {
        if (!failed)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma(tmem + sb * N, k_op + (((kk >> 2) * C::HALF_BYTES + (kk & 3) * 32) >> 4),
                q_op + (((kk >> 2) * N * 128 + (kk & 3) * 32) >> 4), s_kind, kk > 0);
        mma_commit(empty + 8 * slot);
        mma_commit(s_full + 8 * sb);
      }
      __syncwarp();
    };
    scores(0, true);
    for (int i = 0; i < count; ++i) {
      bar_wait(ready + 8 * (i & (C::DESCS - 1)), (i / C::DESCS) & 1, failed);
      const bool first = desc_at(i)->first, last = desc_at(i)->last;
      const uint32_t groups = desc_at(i)->groups;
      // the next tile's scores go first, unless its queries come after this segment's output
      if (!last && i + 1 < count) scores(i + 1, false);
      const int u = 2 * i + 1, slot = u % U;
      bar_wait(full + 8 * slot, (u / U) & 1, failed);
      bar_wait(p_full, i & 1, failed);
      tc_after_sync();
      bool add = !first || *s_add;
      __syncwarp();
      const uint64_t v_op = operand(sbase + slot * C::UNIT, C::HALF_BYTES);
      if (elect_one()) {
        // output^T: D x 2N, V^T times the rounded weights and times their rests
        if (!failed)
#pragma unroll
          for (int kk = 0; kk < TILE / 16; ++kk)
            if ((groups >> kk) & 1) {
              mma(tmem_o, v_op + (kk * 2048 >> 4), p_op + (kk * 16 * C::P_ROW >> 4), o_kind, add);
              add = true;
            }
        mma_commit(empty + 8 * slot);
        mma_commit(o_done);
      }
      __syncwarp();
      if (last && i + 1 < count) scores(i + 1, true);
    }
  } else if (warp == kLoadWarp) {
    // ------------------------------------------------------------ producer
    int ld_b = s_start[0], ld_left = count, ld_hr = s_start[2], ld_tile = s_start[3], ld_from = ld_tile;
    int ld_len = min(max(s_start[1], 0), p.cap);
    bool ld_over = s_start[1] > p.cap;
    Span ld_span = span_of(p, ld_len);
    // (the segment's first tile: the units in front of this one's, less those of the segment itself)
    int ld_seg = s_start[4] + kHead * (ld_b * HR + ld_hr + 1) - ld_tile;
    int next_raw = ld_b + 1 < p.B ? p.lengths[ld_b + 1] : 0;
    bool ld_first = true;

    // A tile's pages: a lane looks up one TMA box, or TILE / 32 rows.  The
    // page numbers loaded here are used one tile later.
    constexpr int LU = TMA ? 1 : TILE / 32;
    struct Lookup {
      int id[LU], row[LU], state[LU];   // state 0: no query sees it, 1: on page `id`, 2: past the table
      Desc d;
    };
    auto look = [&](Lookup& u) {
      if (ld_left <= 0) return;
      const int token0 = (ld_tile < ld_span.ns ? ld_tile : ld_span.lo_tile + ld_tile - ld_span.ns) * TILE;
      u.d.b = ld_b;
      u.d.h = p.row_tiles == 1 ? ld_hr : ld_hr / p.row_tiles;
      u.d.rt = ld_hr - u.d.h * p.row_tiles;
      u.d.token0 = token0;
      u.d.len = ld_len;
      u.d.first = ld_first;
      u.d.n_tiles = ld_span.n;
      u.d.seg_start = ld_seg;
      // positions run from len - T to len - 1
      u.d.full = token0 + TILE <= ld_len - p.T + 1 &&
                 (p.window == 0 || token0 > ld_len - 1 - p.window || token0 + TILE <= p.sinks);
      --ld_left;
      u.d.last = ld_left == 0 || ld_tile + 1 == ld_span.n ? (ld_over ? 2 : 1) : 0;
      u.d.whole = ld_from == 0 && ld_tile + 1 == ld_span.n;
      {
        const int j = token0 + (lane & 7) * 16;
        u.d.groups = __ballot_sync(0xffffffffu, j < ld_len && (j + 16 > ld_span.lo || j < p.sinks)) & 0xffu;
        if (u.d.groups == 0) u.d.groups = 1;
      }
      const int step = TMA ? p.box : 1;
#pragma unroll
      for (int x = 0; x < LU; ++x) {
        const int at = (x * 32 + lane) * step, j = token0 + at;
        u.state[x] = 0;
        u.id[x] = 0;
        u.row[x] = 0;
        if (at < TILE && j < ld_len && (j + step > ld_span.lo || j < p.sinks)) {
          const int pg = (int)((uint64_t)(uint32_t)j * p.page_magic >> p.page_shift);   // j / page
          u.row[x] = j - pg * p.page;
          u.state[x] = ld_over ? 2 : 1;
          u.id[x] = __ldg(p.table + (int64_t)ld_b * p.table_b + pg);
        }
      }
      ld_first = false;
      if (++ld_tile == ld_span.n && ld_left > 0) {
        ld_first = true;
        ld_tile = ld_from = 0;
        ld_seg += ld_span.n + kHead;
        if (++ld_hr == HR) {
          ld_hr = 0;
          ++ld_b;
          ld_len = min(max(next_raw, 0), p.cap);
          ld_over = next_raw > p.cap;
          ld_span = span_of(p, ld_len);
          next_raw = ld_b + 1 < p.B ? p.lengths[ld_b + 1] : 0;
        }
      }
    };
    // A unit copied row by row is announced once its copies have landed, when kBehind more are on their way.  (U - 2:
    // the unit whose slot is waited for may be a V, which is let go after the K behind it has been multiplied.)
    constexpr int kBehind = U - 2;
    auto announce = [&](int un) {
      if (un < 0) return;
      proxy_fence();
      __syncwarp();
      if (lane == 0) bar_arrive(full + 8 * (un % U));
    };
    Lookup next;
    look(next);
    for (int i = 0; i < count; ++i) {
      Lookup u = next;
      look(next);
      bool ok[LU];
#pragma unroll
      for (int w = 0; w < 4; ++w) u.d.bad[w] = 0;
      if constexpr (TMA) {
        ok[0] = u.state[0] == 1 && u.id[0] >= 0 && u.id[0] < p.num_pages;
        const uint32_t bad = __ballot_sync(0xffffffffu, u.state[0] != 0 && !ok[0]);
        if (bad)
#pragma unroll
          for (int w = 0; w < TILE / 32; ++w)
            u.d.bad[w] = __ballot_sync(0xffffffffu, (bad >> ((w * 32 + lane) / p.box)) & 1);
      } else {
#pragma unroll
        for (int x = 0; x < LU; ++x) {
          ok[x] = u.state[x] == 1 && u.id[x] >= 0 && u.id[x] < p.num_pages;
          u.d.bad[x] = __ballot_sync(0xffffffffu, u.state[x] != 0 && !ok[x]);
        }
      }
      for (int side = 0; side < 2; ++side) {   // K, V
        const int un = 2 * i + side, slot = un % U;
        if (un >= U) bar_wait(empty + 8 * slot, (un / U - 1) & 1, failed);
        if (side == 0 && lane == 0) {
          u.d.full = u.d.full && (u.d.bad[0] | u.d.bad[1] | u.d.bad[2] | u.d.bad[3]) == 0;
          *desc_at(i) = u.d;
          bar_arrive(ready + 8 * (i & (C::DESCS - 1)));
        }
        const uint32_t dst = sbase + slot * C::UNIT;
        if constexpr (TMA) {
          const uint32_t good = __ballot_sync(0xffffffffu, ok[0]);
          if (lane == 0) bar_arrive_tx(full + 8 * slot, failed ? 0 : __popc(good) * p.box * 128 * C::HALVES);
          __syncwarp();
          // (each lane its own box: one thread issuing all of them took twice the time with pages of 8)
          if (ok[0] && !failed)
#pragma unroll
            for (int hf = 0; hf < C::HALVES; ++hf)
              tma_box(dst + hf * C::HALF_BYTES + lane * p.box * 128, side ? &vmap : &kmap, full + 8 * slot, hf * 64,
                      u.row[0], u.d.h, u.id[0]);
        } else {
          constexpr int RPI = 32 / C::PIECES;   // rows per step
          const int c = lane % C::PIECES, sub = lane / C::PIECES;
          const uint16_t* base = (side ? p.v : p.k) + c * 8;
#pragma unroll
          for (int x = 0; x < LU; ++x) {
            const int64_t mine = !ok[x] ? -1
                                 : side ? (int64_t)u.id[x] * p.v_page + (int64_t)u.d.h * p.v_head + (int64_t)u.row[x] * p.v_row
                                        : (int64_t)u.id[x] * p.k_page + (int64_t)u.d.h * p.k_head + (int64_t)u.row[x] * p.k_row;
            // all the addresses first, so that the copies follow one another; a row that is not there becomes 0
            int64_t from[32 / RPI];
#pragma unroll
            for (int y = 0; y < 32 / RPI; ++y) from[y] = __shfl_sync(0xffffffffu, mine, y * RPI + sub);
#pragma unroll
            for (int y = 0; y < 32 / RPI; ++y) {
              const int r = x * 32 + y * RPI + sub;
              cp_async16_or_zero(dst + (c >> 3) * C::HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                                 base + (from[y] < 0 ? 0 : from[y]), from[y] >= 0);
            }
          }
          cp_async_commit();
          cp_async_wait<kBehind>();
          announce(un - kBehind);
        }
      }
    }
    if constexpr (!TMA) {
      cp_async_wait<0>();
      for (int un = 2 * count - kBehind; un < 2 * count; ++un) announce(un);
    }
    // after a wait that ran out, see the copies in flight off
    if (TMA && failed)
      for (int un = max(0, 2 * count - U); un < 2 * count; ++un) bar_wait_long(full + 8 * (un % U), (un / U) & 1);
  } else {
    // ------------------------------------------------------------ consumers
    const uint32_t my_lanes = (uint32_t)warp << 21;   // tensor-memory lanes 32 w ..
    float l[N];                                       // this thread's tokens' share of the rows' sums
    // A segment's query rows, row r = t * G + g; read while the segment before it is finished (N = 64: not, for
    // the registers).
    constexpr int QV = N * C::PIECES / kConsumers;
    uint4 q[QV];
    auto load_queries = [&](int b, int h, int rt) {
#pragma unroll
      for (int y = 0; y < QV; ++y) {
        const int r = (y * kConsumers + tid) / C::PIECES, c = tid % C::PIECES, R = rt * N + r;
        q[y] = make_uint4(0, 0, 0, 0);
        if (R < p.R) {
          const int t = R / p.G, g = R - t * p.G;
          q[y] = *reinterpret_cast<const uint4*>(p.q + (int64_t)b * p.q_b + (int64_t)(h * p.G + g) * p.q_h +
                                                 (int64_t)t * p.q_t + c * 8);
        }
      }
    };
    constexpr bool kAhead = N <= 32;
    load_queries(s_start[0], s_start[2] / p.row_tiles, s_start[2] % p.row_tiles);
    for (int i = 0; i < count; ++i) {
      bar_wait(ready + 8 * (i & (C::DESCS - 1)), (i / C::DESCS) & 1, failed);
      const Desc& ds = *desc_at(i);
      const int len = ds.len, token0 = ds.token0, rt = ds.rt;
      const int n_rows = min(N, p.R - rt * N);
      const int v_unit = 2 * i + 1, v_slot = v_unit % U;
      uint8_t* vs = smem + v_slot * C::UNIT;

      if (ds.first) {
        if (!kAhead && i > 0) load_queries(ds.b, ds.h, rt);
#pragma unroll
        for (int y = 0; y < QV; ++y) {
          const int r = (y * kConsumers + tid) / C::PIECES, c = tid % C::PIECES;
          *reinterpret_cast<uint4*>(smem + C::OFF_Q + (c >> 3) * N * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = q[y];
        }
        if (tid < N) {
          const int R = min(rt * N + tid, p.R - 1), t = R / p.G;
          mu_s[tid] = kUnseen;
          // a row that pads a sequence of fewer new tokens stands nowhere: tiles that every row sees are computed
          // for it too, and what it has in the end is not written
          pos_s[tid] = p.counts == nullptr || t >= p.T - p.counts[ds.b] ? len - p.T + t : -1;
          row_s[tid] = (ds.b * p.HQ + ds.h * p.G + R - t * p.G) * p.T + t;
        }
        if (tid == 0) *s_add = 0;
#pragma unroll
        for (int r = 0; r < N; ++r) l[r] = 0.f;
        proxy_fence();
        consumer_sync();
        if (tid == 0) bar_arrive(q_full);
      }
      const bool full_tile = ds.full;
      const int lo = p.window > 0 ? max(0, max(len - p.T, 0) - p.window + 1) : 0;
      if (!full_tile) {
        // Rows of V that no query sees hold whatever the page or an earlier
        // tile left there, and 0 * NaN is NaN: where their group of 16 is
        // multiplied, they are zeroed (thread = token).
        bar_wait(full + 8 * v_slot, (v_unit / U) & 1, failed);
        const int j = token0 + tid;
        if (((ds.groups >> (tid >> 4)) & 1) &&
            (!(j < len && (j >= lo || j < p.sinks)) || ((ds.bad[warp] >> lane) & 1)))
#pragma unroll
          for (int c = 0; c < C::PIECES; ++c)
            *reinterpret_cast<uint4*>(vs + (c >> 3) * C::HALF_BYTES + tid * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
      }

      // ---- scores: thread = token, registers = rows
      bar_wait(s_full + 8 * (i & 1), (i >> 1) & 1, failed);
      tc_after_sync();
      const int j = token0 + tid;
      // the scores of this thread's token, scaled (log2 units) where `factor` is 1: in a tile that some row does
      // not see whole they are also masked, -inf, or NaN on a page outside the pool for the rows that see it
      const float factor = full_tile ? p.scale2 : 1.f;
      float x[N];
      auto load_scores = [&]() {
#pragma unroll
        for (int c = 0; c < N; c += 16)
          if (c < n_rows) tmem_load(tmem + (i & 1) * N + my_lanes + c, x + c);
#pragma unroll
        for (int c = 0; c < N; c += 16)
          if (c < n_rows) tmem_wait_load(x + c);
        if (!full_tile) {
          const bool bad = (ds.bad[warp] >> lane) & 1;
#pragma unroll
          for (int r = 0; r < N; ++r) {
            if ((r & 3) == 0 && r >= n_rows) break;
            const int pos = pos_s[r];
            const bool seen = j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
            x[r] = !seen ? -INFINITY : bad ? NAN : x[r] * p.scale2;
          }
        }
      };
      // ---- exponents against the rows' references, each a maximum so far.
      // Any reference does while 2^(score - reference) stays in range: it
      // moves, and the output is rescaled, only when an exponent passes
      // kBelow + 8 or a row is seen for the first time (kUnseen makes its
      // exponents huge).
      auto exponents = [&]() {
        float hot = -INFINITY;
#pragma unroll
        for (int r = 0; r < N; r += 2) {
          if ((r & 3) == 0 && r >= n_rows) break;
          two_exponents(x[r], x[r + 1], factor, *reinterpret_cast<const float2*>(mu_s + r));
          if (r < n_rows) hot = fmaxf(hot, x[r]);
          if (r + 1 < n_rows) hot = fmaxf(hot, x[r + 1]);
        }
        return hot > kBelow<HALF> + 8.f;
      };
      load_scores();
      if (p.scores != nullptr) {
        float* dst = p.scores + ((int64_t)(ds.b * p.HKV + ds.h) * p.R + rt * N) * p.score_stride + j;
#pragma unroll
        for (int r = 0; r < N; ++r)
          if (r < n_rows) dst[r * p.score_stride] = x[r] * factor;
      }
      const bool moves = ds.first || consumer_any(exponents());
      // the product before this one is done: its P may be overwritten, its output read
      if (i > 0) bar_wait(o_done, (i - 1) & 1, failed);
      tc_after_sync();
      if (moves) {
        if (!ds.first) load_scores();
        {
          float v[N];
#pragma unroll
          for (int r = 0; r < N; ++r) v[r] = x[r] * factor;
          if (N == 16 && n_rows <= 8) store_rows<8, false>(v, smax + warp * N, lane);
          else store_rows<N, false>(v, smax + warp * N, lane);
        }
        consumer_sync();
        if (tid < n_rows) {   // thread = row
          const float before = mu_s[tid];
          float mn = before;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mn = fmaxf(mn, smax[w * N + tid] - kBelow<HALF>);
          mu_s[tid] = mn;
          alpha_s[tid] = fast_exp2(before - mn);
        }
        consumer_sync();
        if (!ds.first) {
#pragma unroll
          for (int c = 0; c < N; c += 16)
            if (c < n_rows) {
#pragma unroll
              for (int part = 0; part < 2; ++part) {
                float o[16];
                tmem_load(tmem_o + my_lanes + part * N + c, o);
                tmem_wait_load(o);
#pragma unroll
                for (int r = 0; r < 16; ++r) o[r] *= c + r < n_rows ? alpha_s[c + r] : 1.f;
                tmem_store(tmem_o + my_lanes + part * N + c, o);
              }
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (c + r < n_rows) l[c + r] *= alpha_s[c + r];
            }
          tmem_wait_store();
        }
        exponents();
      }
      tc_before_sync();
      __syncwarp();
      if (lane == 0) bar_arrive(s_empty + 8 * (i & 1));
      // ---- P.  The tensor cores take it in the pages' type: as the rounded
      // value and the rounded rest (times kRest), side by side, so that the
      // output's own rounding stays the largest error (one rounded value alone
      // doubles it).
#pragma unroll
      for (int r0 = 0; r0 < N; r0 += 8) {
        if (r0 >= n_rows) break;
        uint32_t hi[4], rest[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int r = r0 + 2 * y;
          const float p0 = fast_exp2(x[r]), p1 = fast_exp2(x[r + 1]);
          l[r] += p0;
          l[r + 1] += p1;
          hi[y] = pack2<HALF>(p0, p1);
          rest[y] = pack2<HALF>((p0 - to_float<HALF>((uint16_t)hi[y])) * kRest<HALF>,
                                (p1 - to_float<HALF>((uint16_t)(hi[y] >> 16))) * kRest<HALF>);
        }
        *reinterpret_cast<uint4*>(smem + C::OFF_P + C::p_at(tid, r0, 0)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(smem + C::OFF_P + C::p_at(tid, r0, 1)) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
      }
      // A token that some rows see and others do not has weight 0 in the
      // others, and 0 * inf is NaN in the product.  Such tokens exist for
      // T > 1 only, T - 1 of them at either end of the span.  When one of them
      // holds an infinity or NaN, they are added by hand to the rows that see
      // them and then zeroed.
      if (p.T > 1 && !full_tile) {
        const int n_part = (p.window > 0 ? 2 : 1) * (p.T - 1);
        // the n-th such token's row in the tile, or -1
        auto part_row = [&](int n) {
          const int y = n < p.T - 1 ? len - 1 - n : lo + n - (p.T - 1);
          return y >= 0 && y < len && y >= token0 && y < token0 + TILE ? y - token0 : -1;
        };
        bool odd = false;
        for (int y = tid; y < n_part * C::PIECES; y += kConsumers) {
          const int r = part_row(y / C::PIECES), c = y % C::PIECES;
          if (r < 0) continue;
          const uint4 w = *reinterpret_cast<const uint4*>(vs + (c >> 3) * C::HALF_BYTES + r * 128 + ((c & 7) << 4));
          const uint32_t ones = HALF ? 0x7c00u : 0x7f80u;
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int z = 0; z < 4; ++z) odd |= (ws[z] & ones) == ones || ((ws[z] >> 16) & ones) == ones;
        }
        if (consumer_any(odd)) {
          // thread = output element d of every row (D = 64: 16 of a warp's lanes)
          const int d = D == 128 ? tid : warp * 16 + (lane & 15);
#pragma unroll
          for (int c = 0; c < N; c += 16) {
            if (c >= n_rows) break;
            float o[16];
            tmem_load(tmem_o + my_lanes + c, o);
            tmem_wait_load(o);
            if (ds.first) {   // nothing there yet
#pragma unroll
              for (int r = 0; r < 16; ++r) o[r] = 0.f;
              tmem_store(tmem_o + my_lanes + N + c, o);
            }
            for (int n = 0; n < n_part; ++n) {
              const int tr = part_row(n), y = token0 + tr;
              if (tr < 0 || (n >= p.T - 1 && y > len - p.T)) continue;   // both ends may name it: once
              const float v = to_float<HALF>(*reinterpret_cast<const uint16_t*>(
                  vs + (d >> 6) * C::HALF_BYTES + tr * 128 + ((((d & 63) >> 3) ^ (tr & 7)) << 4) + (d & 7) * 2));
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                if (c + r >= n_rows) break;
                const int pos = pos_s[c + r];
                if (!(y <= pos && (p.window == 0 || y > pos - p.window || y < p.sinks))) continue;
                o[r] += v * (to_float<HALF>(*reinterpret_cast<const uint16_t*>(smem + C::OFF_P + C::p_at(tr, c + r, 0))) +
                             to_float<HALF>(*reinterpret_cast<const uint16_t*>(smem + C::OFF_P + C::p_at(tr, c + r, 1))) *
                                 (1.f / kRest<HALF>));
              }
            }
            tmem_store(tmem_o + my_lanes + c, o);
          }
          tmem_wait_store();
          consumer_sync();
          if (tid == 0) *s_add = 1;
          for (int y = tid; y < n_part * C::PIECES; y += kConsumers) {
            const int r = part_row(y / C::PIECES), c = y % C::PIECES;
            if (r >= 0)
              *reinterpret_cast<uint4*>(vs + (c >> 3) * C::HALF_BYTES + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      proxy_fence();
      tc_before_sync();
      __syncwarp();
      const int last = ds.last;
      const bool whole = ds.whole;
      const int sb = ds.b, sh = ds.h, n_tiles = ds.n_tiles, seg_start = ds.seg_start;
      if (lane == 0) bar_arrive(p_full);

      if (last) {
        if (kAhead && i + 1 < count) {   // the next segment's queries
          bar_wait(ready + 8 * ((i + 1) & (C::DESCS - 1)), ((i + 1) / C::DESCS) & 1, failed);
          const Desc& dn = *desc_at(i + 1);
          load_queries(dn.b, dn.h, dn.rt);
        }
        // ---- the rows' sums over the tokens' threads, while the last product runs
        if (failed || last == 2)
#pragma unroll
          for (int r = 0; r < N; ++r) l[r] = NAN;
        if (N == 16 && n_rows <= 8) store_rows<8, true>(l, ssum + warp * N, lane);
        else store_rows<N, true>(l, ssum + warp * N, lane);
        consumer_sync();
        const int64_t slot_o = blockIdx.x * 2 + (seg_start - kHead > g0 ? 1 : 0);
        if (tid < n_rows) {   // thread = row
          const float sum = ssum[tid] + ssum[N + tid] + ssum[2 * N + tid] + ssum[3 * N + tid];
          if (whole) {
            const bool none = sum == 0.f || (pos_s[tid] < 0 && last != 2);
            alpha_s[tid] = none ? 0.f : 1.f / sum;
            const float lse2 = none ? -INFINITY : mu_s[tid] + log2f(sum);
            if (p.lse) p.lse[row_s[tid]] = lse2 * 0.6931471805599453f;
            if (p.row_stat)
              p.row_stat[(int64_t)(sb * p.HKV + sh) * p.R + rt * N + tid] =
                  pos_s[tid] < 0 ? make_float2(INFINITY, INFINITY) : make_float2(mu_s[tid], none ? 0.f : log2f(sum));
          } else {
            *reinterpret_cast<float2*>(p.part_ml + (slot_o * ROWS + tid) * 2) = make_float2(mu_s[tid], sum);
          }
        }
        bar_wait(o_done, i & 1, failed);
        tc_after_sync();
        consumer_sync();
        const int d = D == 128 ? tid : warp * 16 + lane;   // (D = 64: lanes below 16 hold a row of the output each)
#pragma unroll
        for (int c = 0; c < N; c += 16) {
          if (c >= n_rows) break;
          float o[16], rest[16];
          tmem_load(tmem_o + my_lanes + c, o);
          tmem_load(tmem_o + my_lanes + N + c, rest);
          tmem_wait_load(o);
          tmem_wait_load(rest);
          if (D == 128 || lane < 16) {
            float* part = p.part_o + (slot_o * ROWS + c) * D + d;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              if (c + r >= n_rows) break;
              // (an infinite value that the row sees makes the rest, 0 or negative, NaN or of the other sign: o has it)
              const float y = rest[r] * (1.f / kRest<HALF>), x = fabsf(y) <= FLT_MAX ? o[r] + y : o[r];
              if (whole)
                p.out[(int64_t)row_s[c + r] * D + d] =
                    (uint16_t)pack2<HALF>(alpha_s[c + r] == 0.f ? 0.f : x * alpha_s[c + r], 0.f);
              else part[r * D] = x;
            }
          }
        }
        tc_before_sync();
        if (!whole) {
          // ---- join.  The CTAs c0..c1 of the segment arrive in groups of
          // kGroup; a group's last adds its parts up, the last group's last
          // adds the groups up and writes the rows: two rounds of a few
          // independent loads instead of one long chain.  The order of the
          // sums is the CTAs', whoever does them.
          const Cut cut(total, ctas);
          const int c0 = cut.owner(seg_start), c1 = cut.owner(seg_start + n_tiles - 1);
          const int n = c1 - c0 + 1, groups = (n + kGroup - 1) / kGroup;
          // part k of the segment: CTA c0 + k; CTA c0's second part when it began with another segment.
          // A group's sum: behind all parts, by its first CTA.
          const int first_slot = c0 * 2 + (cut.begin(c0) < seg_start - kHead ? 1 : 0);
          // parts [k0, k0 + cnt) of the segment, or its group sums, -> the rows, or group sum `to`
          auto join = [&](int k0, int cnt, bool of_groups, int to) {
            auto slot_of = [&](int k) {
              if (!of_groups) return k0 + k == 0 ? first_slot : (c0 + k0 + k) * 2;
              return k * kGroup + 1 == n ? c1 * 2 : 2 * p.ctas + c0 + k * kGroup;   // a group of one is its part
            };
            constexpr int PB = N == 16 || (N == 32 && D == 128) ? 8 : 4;   // as the registers allow
#pragma unroll 1
            for (int x = tid; x < n_rows * (D / 8); x += kConsumers) {   // 8 elements of a row, PB parts at a time
              const int r = x / (D / 8), col = x % (D / 8) * 8;
              float mm = kUnseen, sum = 0.f, acc[8];
#pragma unroll
              for (int z = 0; z < 8; ++z) acc[z] = 0.f;
#pragma unroll 1
              for (int kb = 0; kb < cnt; kb += PB) {
                float2 ml[PB];
                float4 f[PB][2];
#pragma unroll
                for (int y = 0; y < PB; ++y) {
                  ml[y] = make_float2(kUnseen, 0.f);
                  f[y][0] = f[y][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                  if (kb + y < cnt) {
                    const int64_t at = (int64_t)slot_of(kb + y) * ROWS + r;
                    const float4* from = reinterpret_cast<const float4*>(p.part_o + at * D + col);
                    ml[y] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
                    f[y][0] = __ldcg(from);
                    f[y][1] = __ldcg(from + 1);
                  }
                }
                float mn = mm;
#pragma unroll
                for (int y = 0; y < PB; ++y) mn = fmaxf(mn, ml[y].x);
                const float alpha = fast_exp2(mm - mn);
                mm = mn;
                sum *= alpha;
#pragma unroll
                for (int z = 0; z < 8; ++z) acc[z] *= alpha;
#pragma unroll
                for (int y = 0; y < PB; ++y) {
                  const float w = fast_exp2(ml[y].x - mn);
                  sum += w * ml[y].y;
                  acc[0] += w * f[y][0].x; acc[1] += w * f[y][0].y; acc[2] += w * f[y][0].z; acc[3] += w * f[y][0].w;
                  acc[4] += w * f[y][1].x; acc[5] += w * f[y][1].y; acc[6] += w * f[y][1].z; acc[7] += w * f[y][1].w;
                }
              }
              if (to >= 0) {
                const int64_t at = (int64_t)(2 * p.ctas + to) * ROWS + r;
                float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + col);
                dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (col == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mm, sum);
                continue;
              }
              const bool none = sum == 0.f || (pos_s[r] < 0 && last != 2);
              if (none)
#pragma unroll
                for (int z = 0; z < 8; ++z) acc[z] = 0.f;
              const float inv = none ? 0.f : 1.f / sum;
              *reinterpret_cast<uint4*>(p.out + (int64_t)row_s[r] * D + col) =
                  make_uint4(pack2<HALF>(acc[0] * inv, acc[1] * inv), pack2<HALF>(acc[2] * inv, acc[3] * inv),
                             pack2<HALF>(acc[4] * inv, acc[5] * inv), pack2<HALF>(acc[6] * inv, acc[7] * inv));
              if (col == 0) {
                const float lse2 = none ? -INFINITY : mm + log2f(sum);
                if (p.lse) p.lse[row_s[r]] = lse2 * 0.6931471805599453f;
                if (p.row_stat)
                  p.row_stat[(int64_t)(sb * p.HKV + sh) * p.R + rt * N + r] =
                      pos_s[r] < 0 ? make_float2(INFINITY, INFINITY) : make_float2(mm, none ? 0.f : log2f(sum));
              }
            }
          };
          // arrive at a counter that `of` CTAs share; true for the last one, which zeroes it
          auto arrive = [&](int* counter, int of) {
            consumer_sync();
            if (tid == 0) {
              __threadfence();   // the whole CTA's stores, which the barrier put in front of it
              const int is_last = atomicAdd(counter, 1) == of - 1;
              if (is_last) {
                *counter = 0;
                __threadfence();
              }
              *s_last = is_last;
            }
            consumer_sync();
            return *s_last != 0;
          };
          const int grp = (blockIdx.x - c0) / kGroup;
          const int in_group = min(kGroup, n - grp * kGroup);
          // (a group of one needs no counter and no sum; its CTA may begin the next segment, whose first group
          // has them there)
          if (in_group == 1 || arrive(p.counters + p.ctas + c0 + grp * kGroup, in_group)) {
            if (groups > 1 && in_group > 1) join(grp * kGroup, in_group, false, c0 + grp * kGroup);
            if (groups == 1 || arrive(p.counters + c0, groups)) join(0, groups == 1 ? n : groups, groups > 1, -1);
          }
        }
        consumer_sync();   // the row statistics and s_last are free again
      }
    }
  }
  tc_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_after_sync();
    free_tmem();
  }
}

// token_weights[b, j] += sum over the heads and new tokens of 2^((x - m) - log2 l),
// with m and l apart: their sum is rounded to the spacing of numbers like m.
// A CTA takes 256 / W tokens, 256 / W threads every W-th row; their sums are
// added in order: no atomics, a fixed order of sums.  What bounds it: round
// trips where tokens are few (W = 8), else the scores, written by the
// attention and read here out of L2, 4 bytes per row and token (W = 1).
constexpr int kWeightThreads = 256;
template <int W>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const __grid_constant__ Params p, float* weights,
                                                                 int64_t weights_b) {
  constexpr int TOKENS = kWeightThreads / W;
  __shared__ float sums[W][TOKENS];
  pdl_enter();
  const int b = blockIdx.y, rows = p.HKV * p.R, part = threadIdx.x / TOKENS, at = threadIdx.x % TOKENS;
  const int len = length_of(p, b), j0 = blockIdx.x * TOKENS, j = j0 + at;
  const Span s = span_of(p, len);
  if (j0 >= len || (j0 + TOKENS <= s.lo && j0 >= p.sinks)) return;
  const bool seen = j < len && (j >= s.lo || j < p.sinks);
  const float* src = p.scores + (int64_t)b * rows * p.score_stride + j;
  const float2* stat = p.row_stat + (int64_t)b * rows;
  float sum = 0.f;
  if (seen) {
#pragma unroll 4
    for (int r = part; r < rows; r += W) {
      const float2 y = stat[r];
      const float w = fast_exp2((src[(int64_t)r * p.score_stride] - y.x) - y.y);
      sum += y.y == INFINITY ? 0.f : w;   // (the scores of a row that is no token's may be anything)
    }
  }
  if constexpr (W > 1) {
    sums[part][at] = sum;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) sum += sums[w][at];
  }
  if (seen) weights[(int64_t)b * weights_b + j] += sum;
}

// New token t of sequence b goes to row j % page of page table[b, j / page],
// j = L - T + t; with counts, only the last of the T.  A row whose page is not in the pool is not written (the
// attention over it gives NaN).  A few KB: its time is a launch's, 2 to 4 us
// of the step.
__global__ void append_kernel(const __grid_constant__ kvr_paged_append_args a) {
  pdl_enter();
  const int pieces = a.head_dim / 8;
  const int64_t n = (int64_t)a.batch * a.kv_heads * a.new_tokens * pieces;
  for (int64_t x = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; x < 2 * n; x += (int64_t)gridDim.x * blockDim.x) {
    const bool is_v = x >= n;
    int64_t y = is_v ? x - n : x;
    const int c = (int)(y % pieces);
    y /= pieces;
    const int h = (int)(y % a.kv_heads);
    y /= a.kv_heads;
    const int t = (int)(y % a.new_tokens), b = (int)(y / a.new_tokens);
    if (a.new_counts && t < a.new_tokens - a.new_counts[b]) continue;
    const int64_t j = (int64_t)a.lengths[b] - a.new_tokens + t;
    if (j < 0 || j >= (int64_t)a.table_width * a.page_size) continue;
    const int pg = (int)(j / a.page_size), row = (int)(j - (int64_t)pg * a.page_size);
    const int id = a.block_table[(int64_t)b * a.table_stride + pg];
    if (id < 0 || id >= a.num_pages) continue;
    const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.value : a.key) +
                          (int64_t)b * (is_v ? a.value_b_stride : a.key_b_stride) +
                          (int64_t)h * (is_v ? a.value_h_stride : a.key_h_stride) +
                          (int64_t)t * (is_v ? a.value_t_stride : a.key_t_stride) + c * 8;
    uint16_t* dst = static_cast<uint16_t*>(is_v ? a.value_pages : a.key_pages) +
                    (int64_t)id * (is_v ? a.value_page_stride : a.key_page_stride) +
                    (int64_t)h * (is_v ? a.value_head_stride : a.key_head_stride) +
                    (int64_t)row * (is_v ? a.value_row_stride : a.key_row_stride) + c * 8;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  }
}

// ------------------------------------------------------------------- host
static bool mult8(int64_t x) { return (x & 7) == 0; }

static int num_sms_of(int given) {
  if (given > 0) return given;
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (sms[dev & 63] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    sms[dev & 63] = n;
  }
  return sms[dev & 63];
}

// Scores of the weights' launch are held for as many sequences at a time as
// fit here (one at least): they take 4 bytes per row and token of the table's
// width, and a pool's table may be far wider than its sequences (20 GB for 64
// sequences of 32 heads and 5 new tokens in a table of 512K tokens).  A part
// costs some 20 us: 64 sequences of 200 to 8000, 12 heads, 5 new tokens, a table
// of 512K take 237 us at once with 8 GB, 300 with this, 600 with 512 MB, which
// would also slow tables of 64K tokens (32 sequences of 2K to 16K, 32 heads: 329 for 418).
constexpr size_t kScoreBytes = 2048ull << 20;

struct Plan {
  int G, R, n, row_tiles, cap, ctas;
  int part;   // sequences per launch (with token weights)
  int64_t score_stride;
  size_t part_o, part_ml, stats, scores;
};

static int plan_of(const kvr_paged_attention_args* a, Plan* out) {
  if (!a || a->batch < 0 || a->q_heads <= 0 || a->kv_heads <= 0 || a->new_tokens <= 0 || a->page_size <= 0 ||
      a->table_width < 0 || a->num_pages < 0 || a->window < 0 || a->sinks < 0 || a->q_heads % a->kv_heads)
    return KVR_ERR_INVALID_ARGUMENT;
  if ((a->head_dim != 64 && a->head_dim != 128) || (a->dtype != 0 && a->dtype != 1)) return KVR_ERR_UNSUPPORTED;
  const int64_t cap = (int64_t)a->table_width * a->page_size;
  Plan p;
  p.G = a->q_heads / a->kv_heads;
  const int64_t R = (int64_t)p.G * a->new_tokens;
  // 2^30 keeps token positions and the rows' products inside 32 bits
  if (cap > (1 << 30) || R > (1 << 20) || (int64_t)a->batch * a->kv_heads * R > (1ll << 31) - 1)
    return KVR_ERR_UNSUPPORTED;
  // weights_kernel: the batch along the grid's y
  if (a->token_weights && a->batch > 65535) return KVR_ERR_UNSUPPORTED;
  p.R = (int)R;
  p.cap = (int)cap;
  // Rows of a tile: the fewest that hold them, since a thread's work goes with them and fewer leave room for a
  // second CTA per SM.  (4 rows in 16 and in 32: 32 sequences of up to 8K 49.8 and 52.3 us; 6 rows: 128 windows of 1K
  // 29.8 and 38.9 us; 30 rows in 32 and in 64: 64 sequences of 4K to 16K 119 and 128 us.)
  p.n = R <= 16 ? 16 : R <= 32 || a->head_dim == 64 ? 32 : 64;
  // (head dimension 64: 32 rows with two CTAs per SM in place of 64 with one take 26 for 33 us on 16 sequences of 4K
  // with 56 rows, 185 for 227 us on 64 of 16K.)
  // With little work several tiles of 16 rows beat one: K and V come from L2 again, but more CTAs share the softmax,
  // and the joins, which take longer than the tiles.  (64 rows of one sequence of 16K: 20.6 us in 16, 26.4 in 32, 45.0
  // in 64; 30 rows, 16 of 4K, 7 tiles per CTA: 25.7 in 16 and 27.7 in 32; 16 of 16K, 27 per CTA: 89 and 62;
  // 128 rows, 4 of 16K, 14 per CTA: 38.6 in 16 and 51.0 in 64; 64 rows, 16 of 16K, 27 per CTA: 74.5 and 66.4.)
  const int64_t sees = a->window > 0 ? std::min<int64_t>(cap, (int64_t)a->window + a->new_tokens + a->sinks) : cap;
  if ((sees + kTile - 1) / kTile * a->batch * a->kv_heads * ((R + 15) / 16) <=
      (p.n == 64 ? 14 : 8) * 2 * (int64_t)num_sms_of(a->num_sms))
    p.n = 16;
  p.row_tiles = (p.R + p.n - 1) / p.n;
  const int64_t tiles = std::max<int64_t>(1, (cap + kTile - 1) / kTile + 1 + kHead) * a->batch * a->kv_heads * p.row_tiles;
  if (tiles > (1ll << 31) - 1) return KVR_ERR_UNSUPPORTED;
  // one or two CTAs per SM (Cfg::CTAS); a join takes kGroup^2 parts and some
  const int per_sm = p.n == 16 || a->head_dim == 64 ? 2 : 1;
  p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(tiles, std::min(per_sm * num_sms_of(a->num_sms), kGroup * 20)));
  p.score_stride = std::max<int64_t>(128, (cap + 127) / 128 * 128);
  const size_t rows = (size_t)p.n * 3 * p.ctas;
  p.part_o = rows * a->head_dim * sizeof(float);
  p.part_ml = rows * 2 * sizeof(float);
  const size_t seq_rows = (size_t)a->kv_heads * p.R, seq_scores = seq_rows * p.score_stride * sizeof(float);
  p.part = a->token_weights ? (int)std::min<size_t>(a->batch, std::max<size_t>(1, kScoreBytes / seq_scores)) : a->batch;
  const size_t all_rows = p.part * seq_rows;
  p.stats = a->token_weights ? (all_rows * sizeof(float2) + 255) / 256 * 256 : 0;
  p.scores = a->token_weights ? all_rows * p.score_stride * sizeof(float) : 0;
  *out = p;
  return KVR_OK;
}

// Tensor maps of the pages: [page number][head][row][element] with the
// caller's strides, boxes of `box` rows x 64 elements, 128-byte swizzle.
// False where the pages do not fit one (an axis with stride 0, say).
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}
static bool page_map(CUtensorMap* map, const void* base, bool half, int D, int page, int heads, int pages,
                     int64_t row_stride, int64_t head_stride, int64_t page_stride, int box) {
  EncodeFn fn = encode_fn();
  if (!fn || pages <= 0) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)pages};
  const int64_t given[3] = {row_stride, head_stride, page_stride};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    // an axis of one element is never stepped along: any valid stride does
    strides[i] = 2 * (cuuint64_t)(dims[i + 1] == 1 ? D : given[i]);
    if (dims[i + 1] > 1 && given[i] <= 0) return false;
    if (strides[i] >= (1ull << 40)) return false;
  }
  const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
            dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Maps {
  CUtensorMap k, v;
};

template <bool HALF, int D, int N, bool TMA>
static int launch(const Params& p, const Maps& maps, cudaStream_t s) {
  using C = Cfg<D, N>;
  auto kern = attention_kernel<HALF, D, N, TMA>;
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (!ready[dev & 63]) {   // a benign race sets the same value
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
    ready[dev & 63] = true;
  }
  cudaError_t e = pdl_launch(kern, dim3(p.ctas), dim3(kThreads), C::SMEM, s, 1, p, maps.k, maps.v);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}

template <bool HALF, int D, bool TMA>
static int launch_n(int n, const Params& p, const Maps& maps, cudaStream_t s) {
  if (n == 16) return launch<HALF, D, 16, TMA>(p, maps, s);
  if constexpr (D == 128)
    if (n == 64) return launch<HALF, D, 64, TMA>(p, maps, s);
  return launch<HALF, D, 32, TMA>(p, maps, s);
}
template <bool HALF, int D>
static int launch_tma(bool tma, int n, const Params& p, const Maps& maps, cudaStream_t s) {
  return tma ? launch_n<HALF, D, true>(n, p, maps, s) : launch_n<HALF, D, false>(n, p, maps, s);
}

}  // namespace paged
}  // namespace kvr

using namespace kvr;

extern "C" int kvr_paged_attention_plan(const kvr_paged_attention_args* a, size_t* workspace_bytes,
                                        size_t* counter_count, size_t* scores_bytes) {
  paged::Plan p;
  int st = paged::plan_of(a, &p);
  if (st != KVR_OK) return st;
  if (p.part < a->batch) {   // what a part or the last, smaller one needs
    kvr_paged_attention_args part = *a;
    paged::Plan last;
    part.batch = a->batch % p.part ? a->batch % p.part : p.part;
    st = paged::plan_of(&part, &last);
    if (st != KVR_OK) return st;
    part.batch = p.part;
    st = paged::plan_of(&part, &p);
    if (st != KVR_OK) return st;
    p.part_o = std::max(p.part_o + p.part_ml, last.part_o + last.part_ml);
    p.part_ml = 0;
    p.ctas = std::max(p.ctas, last.ctas);
  }
  if (workspace_bytes) *workspace_bytes = p.part_o + p.part_ml;
  if (counter_count) *counter_count = 2 * (size_t)p.ctas;
  if (scores_bytes) *scores_bytes = p.stats + p.scores;
  return KVR_OK;
}

extern "C" int kvr_paged_attention(const kvr_paged_attention_args* a, kvr_stream_t stream) {
  paged::Plan pl;
  int st = paged::plan_of(a, &pl);
  if (st != KVR_OK) return st;
  if (a->batch == 0) return KVR_OK;
  if (pl.part < a->batch && a->query && a->out && a->lengths && a->block_table) {
    for (int b = 0; b < a->batch; b += pl.part) {
      kvr_paged_attention_args part = *a;
      const int64_t rows = (int64_t)b * a->q_heads * a->new_tokens;
      part.batch = std::min(pl.part, a->batch - b);
      part.query = static_cast<const uint16_t*>(a->query) + b * a->q_b_stride;
      part.out = static_cast<uint16_t*>(a->out) + rows * a->head_dim;
      part.lse = a->lse ? a->lse + rows : nullptr;
      part.block_table = a->block_table + b * a->table_stride;
      part.lengths = a->lengths + b;
      part.new_counts = a->new_counts ? a->new_counts + b : nullptr;
      part.token_weights = a->token_weights + b * a->weights_b_stride;
      st = kvr_paged_attention(&part, stream);
      if (st != KVR_OK) return st;
    }
    return KVR_OK;
  }
  if (!a->query || !a->out || !a->lengths || (pl.cap > 0 && !a->block_table) ||
      (a->num_pages > 0 && (!a->key_pages || !a->value_pages)))
    return KVR_ERR_INVALID_ARGUMENT;
  if (!aligned16(a->query) || !aligned16(a->key_pages) || !aligned16(a->value_pages) || !aligned16(a->out))
    return KVR_ERR_MISALIGNED;
  const int64_t strides[] = {a->q_b_stride, a->q_h_stride, a->q_t_stride, a->key_page_stride, a->key_head_stride,
                             a->key_row_stride, a->value_page_stride, a->value_head_stride, a->value_row_stride};
  for (int64_t x : strides)
    if (!paged::mult8(x)) return KVR_ERR_MISALIGNED;
  if (!a->workspace || a->workspace_bytes < pl.part_o + pl.part_ml || !a->counters) return KVR_ERR_WORKSPACE;
  if (!aligned16(a->workspace)) return KVR_ERR_MISALIGNED;
  if (a->token_weights && (!a->scores || a->scores_bytes < pl.stats + pl.scores)) return KVR_ERR_WORKSPACE;
  if (a->token_weights && !aligned16(a->scores)) return KVR_ERR_MISALIGNED;

  paged::Params p;
  p.q = static_cast<const uint16_t*>(a->query);
  p.q_b = a->q_b_stride; p.q_h = a->q_h_stride; p.q_t = a->q_t_stride;
  p.k = static_cast<const uint16_t*>(a->key_pages);
  p.k_page = a->key_page_stride; p.k_head = a->key_head_stride; p.k_row = a->key_row_stride;
  p.v = static_cast<const uint16_t*>(a->value_pages);
  p.v_page = a->value_page_stride; p.v_head = a->value_head_stride; p.v_row = a->value_row_stride;
  p.table = a->block_table; p.table_b = a->table_stride;
  p.num_pages = a->num_pages; p.page = a->page_size;
  // Division by the page size as a product: with 2^s >= page and m = ceil(2^(30+s) / page), m page exceeds 2^(30+s)
  // by less than 2^s, so j m / 2^(30+s) exceeds j / page by less than 1 / page for j < 2^30.  m < 2^32.
  int shift = 0;
  while ((1ll << shift) < a->page_size) ++shift;
  p.page_shift = 30 + shift;
  p.page_magic = (uint32_t)(((1ull << p.page_shift) + a->page_size - 1) / a->page_size);
  p.lengths = a->lengths;
  p.counts = a->new_counts;
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.row_stat = a->token_weights ? static_cast<float2*>(a->scores) : nullptr;
  p.scores = a->token_weights ? reinterpret_cast<float*>(static_cast<uint8_t*>(a->scores) + pl.stats) : nullptr;
  p.score_stride = pl.score_stride;
  p.B = a->batch; p.HQ = a->q_heads; p.HKV = a->kv_heads; p.T = a->new_tokens;
  p.G = pl.G; p.R = pl.R; p.row_tiles = pl.row_tiles;
  // (no more than what a table can hold, 2^30: the sums with positions stay inside 32 bits)
  p.window = std::min(a->window, 1 << 30); p.sinks = a->window > 0 ? std::min(a->sinks, pl.cap) : 0; p.cap = pl.cap;
  p.scale2 = a->scale * 1.4426950408889634f;
  p.ctas = pl.ctas;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + pl.part_o);
  p.counters = a->counters;
  cudaStream_t s = as_stream(stream);
  const bool half = a->dtype == 1;
  // TMA boxes: the largest number of tokens that divides both a page and a
  // tile; below 4 (a lane's box each) the rows are copied one by one.  32
  // sequences of 2K to 8K, 12 query and 2 KV heads of 128: pages of 16 or more
  // 38 us, of 8 39 us, of 4 53 us by TMA, row by row 59 us whatever the page.
  int box = paged::kTile;
  while (a->page_size % box) box /= 2;
  p.box = box;
  paged::Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  const bool tma = box >= 4 &&
                   paged::page_map(&maps.k, a->key_pages, half, a->head_dim, a->page_size, a->kv_heads, a->num_pages,
                                   a->key_row_stride, a->key_head_stride, a->key_page_stride, box) &&
                   paged::page_map(&maps.v, a->value_pages, half, a->head_dim, a->page_size, a->kv_heads, a->num_pages,
                                   a->value_row_stride, a->value_head_stride, a->value_page_stride, box);
  if (a->head_dim == 64)
    st = half ? paged::launch_tma<true, 64>(tma, pl.n, p, maps, s) : paged::launch_tma<false, 64>(tma, pl.n, p, maps, s);
  else
    st = half ? paged::launch_tma<true, 128>(tma, pl.n, p, maps, s) : paged::launch_tma<false, 128>(tma, pl.n, p, maps, s);
  if (st != KVR_OK || !a->token_weights || pl.cap == 0) return st;
  // Few CTAs: the rows split over eight warps (their share of a step with one sequence of 4K and 64 rows: 6 us, with
  // one thread for all rows 12; with 256 rows 11 and 32).  More CTAs than the GPU holds at a time only cost: 16 sequences
  // of 1K to 8K with 12 rows, 25 us a step for 23.
  const int wide = (pl.cap + paged::kWeightThreads - 1) / paged::kWeightThreads;
  cudaError_t e;
  if ((int64_t)wide * p.B < 2 * paged::num_sms_of(a->num_sms))
    e = pdl_launch(paged::weights_kernel<8>, dim3((pl.cap + 31) / 32, p.B), dim3(paged::kWeightThreads), 0, s, 1, p,
                   a->token_weights, a->weights_b_stride);
  else
    e = pdl_launch(paged::weights_kernel<1>, dim3(wide, p.B), dim3(paged::kWeightThreads), 0, s, 1, p, a->token_weights,
                   a->weights_b_stride);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}

extern "C" int kvr_paged_append(const kvr_paged_append_args* a, kvr_stream_t stream) {
  if (!a || a->batch < 0 || a->kv_heads <= 0 || a->new_tokens < 0 || a->page_size <= 0 || a->table_width < 0 ||
      a->num_pages < 0 || a->head_dim <= 0)
    return KVR_ERR_INVALID_ARGUMENT;
  if (a->head_dim % 8) return KVR_ERR_UNSUPPORTED;
  const int64_t n = 2ll * a->batch * a->kv_heads * a->new_tokens * (a->head_dim / 8);
  if (n == 0) return KVR_OK;
  if (!a->key || !a->value || !a->lengths || (a->table_width > 0 && !a->block_table) ||
      (a->num_pages > 0 && (!a->key_pages || !a->value_pages)))
    return KVR_ERR_INVALID_ARGUMENT;
  const int64_t strides[] = {a->key_b_stride, a->key_h_stride, a->key_t_stride, a->value_b_stride, a->value_h_stride,
                             a->value_t_stride, a->key_page_stride, a->key_head_stride, a->key_row_stride,
                             a->value_page_stride, a->value_head_stride, a->value_row_stride};
  for (int64_t x : strides)
    if (!paged::mult8(x)) return KVR_ERR_MISALIGNED;
  if (!aligned16(a->key) || !aligned16(a->value) || !aligned16(a->key_pages) || !aligned16(a->value_pages))
    return KVR_ERR_MISALIGNED;
  const int grid = (int)std::min<int64_t>((n + 127) / 128, 4096);
  cudaError_t e = pdl_launch(paged::append_kernel, dim3(grid), dim3(128), 0, as_stream(stream), 1, *a);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}
