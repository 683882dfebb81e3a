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
// it, so R operations per byte, far below the tensor cores' rate for the few
// rows of a decode step.  The kernel is therefore laid out around keeping
// loads in flight and the instructions per tile few:
//  * Work is a flat list of token tiles (sequence, KV head, row tile, tile),
//    cut into equal ranges, one per CTA.  Lengths are read on the device, so
//    a ragged batch is balanced to one tile without the host knowing it.
//  * A producer warp looks up pages and fills a ring of tiles, on across
//    sequence boundaries; four consumer warps compute.  Pages of a multiple
//    of 8 tokens come by TMA, a box per page; others row by row (cp.async).
//  * The consumers share each tile: for the scores a warp owns a quarter of
//    the tokens, for the output a quarter of the head dimension, so every
//    byte of K and V is read from shared memory once and the accumulator is
//    complete in the CTA: nothing is merged between warps.
//  * A sequence that several CTAs share is joined by the last of them to
//    arrive, in the order of the CTAs: the result does not depend on timing.
#include "kvr_ring.cuh"

#include <cuda.h>

#include <algorithm>
#include <cstring>

namespace kvr {
namespace paged {

using namespace ring;

constexpr int kWarps = 4;                     // consumers
constexpr int kConsumers = 32 * kWarps;
constexpr int kThreads = kConsumers + 32;     // and the producer warp
constexpr int kGroup = 16;                    // CTAs a join takes at a time

// Rows that no mask leaves anything to keep m = -inf; 0 stands in for it
// wherever it would be subtracted.
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

template <bool HALF>
__device__ __forceinline__ void mma_e(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (HALF) mma_f16(d, a0, a1, a2, a3, b0, b1);
  else mma_bf16(d, a0, a1, a2, a3, b0, b1);
}

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

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
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

struct Params {
  const uint16_t* q;
  int64_t q_b, q_h, q_t;
  const uint16_t* k;
  int64_t k_page, k_head, k_row;
  const uint16_t* v;
  int64_t v_page, v_head, v_row;
  const int* table;
  int64_t table_b;
  int table_width, num_pages, page;
  const int* lengths;
  uint16_t* out;
  float* lse;       // [B, HQ, T] or null
  float* scores;    // [B, HKV, R, score_stride] or null: x_ij for the weights kernel
  float* row_lse2;  // [B, HKV, R], with scores
  int64_t score_stride;
  int B, HQ, HKV, T, G, R, row_tiles, window, sinks, cap;
  float scale2;     // scale * log2(e)
  int ctas, min_tiles;
  float* part_o;    // [3 * ctas][ROWS][D]: two parts of each CTA, group sums
  float* part_ml;   // [3 * ctas][ROWS][2]
  int* counters;    // [2 * ctas], zero on entry and on exit
  int box;          // tokens of a TMA box
};

template <int D, int MT>
struct Cfg {
  static constexpr int TILE = D == 64 ? 128 : 64;   // tokens: 16 KB of K and 16 KB of V either way
  static constexpr int ROWS = 16 * MT;
  static constexpr int HALVES = D / 64;
  static constexpr int PIECES = D / 8;
  static constexpr int HALF_BYTES = TILE * 128;     // 64 elements of every token, 128-byte rows
  static constexpr int KV_BYTES = HALVES * HALF_BYTES;
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int STAGES = MT == 4 ? 2 : 3;    // two CTAs per SM in every case
  static constexpr int NT = TILE / kWarps / 8;      // 8-token score tiles of a warp
  static constexpr int DW = D / kWarps;             // output columns of a warp
  static constexpr int DT = DW / 8;
  // shared memory: ring, Q (MT <= 2 keeps it in registers and lets P take its place), P, descriptors, row
  // statistics, barriers
  static constexpr int Q_BYTES = ROWS * D * 2, P_HALF = ROWS * TILE * 2, P_BYTES = 2 * P_HALF;
  static constexpr int OFF_Q = STAGES * STAGE;
  static constexpr int OFF_P = MT <= 2 ? OFF_Q : OFF_Q + Q_BYTES;
  static constexpr int OFF_DESC = OFF_Q + (MT <= 2 ? (Q_BYTES > P_BYTES ? Q_BYTES : P_BYTES) : Q_BYTES + P_BYTES);
  static constexpr int OFF_MAX = OFF_DESC + STAGES * 64;
  static constexpr int OFF_SUM = OFF_MAX + kWarps * ROWS * 4;
  static constexpr int OFF_BAR = OFF_SUM + kWarps * ROWS * 4;
  static constexpr int OFF_MISC = OFF_BAR + 3 * STAGES * 8;
  static constexpr int SMEM = OFF_MISC + 64 + 1024;   // 1 KB to align the ring
};

struct Desc {
  int b, h, rt, token0, len, first, last, n_tiles;
  int seg_start;
  uint32_t bad[4];   // tokens on pages outside the pool, a bit each
};
static_assert(sizeof(Desc) <= 64, "");

// `total` tiles cut into `n` ranges of equal size, the first ones a tile longer.
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
template <int TILE>
__device__ __forceinline__ Span span_of(const Params& p, int len) {
  Span s;
  const int total = (len + TILE - 1) / TILE;
  s.lo = p.window > 0 ? max(0, max(len - p.T, 0) - p.window + 1) : 0;
  s.lo_tile = min(s.lo / TILE, max(total - 1, 0));
  s.ns = min((p.sinks + TILE - 1) / TILE, s.lo_tile);
  s.n = max(1, s.ns + total - s.lo_tile);   // an empty sequence gets one tile, to write its zero rows
  return s;
}
__device__ __forceinline__ int length_of(const Params& p, int b) { return min(max(p.lengths[b], 0), p.cap); }

template <bool HALF, int D, int MT, bool TMA>
__global__ void __launch_bounds__(kThreads, 2) attention_kernel(const __grid_constant__ Params p,
                                                                const __grid_constant__ CUtensorMap kmap,
                                                                const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D, MT>;
  constexpr int TILE = C::TILE, ROWS = C::ROWS, S = C::STAGES;
  extern __shared__ uint8_t raw_smem[];
  // the swizzle pattern of a tile follows address bits 7..9: align the ring to 1 KB
  uint8_t* smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Desc* descs = reinterpret_cast<Desc*>(smem + C::OFF_DESC);
  float* smax = reinterpret_cast<float*>(smem + C::OFF_MAX);
  float* ssum = reinterpret_cast<float*>(smem + C::OFF_SUM);
  // a slot's data is there / is read / its descriptor is there (before the data)
  const uint32_t full = sbase + C::OFF_BAR, empty = full + S * 8, ready = empty + S * 8;
  int* s_start = reinterpret_cast<int*>(smem + C::OFF_MISC);   // [3]
  int* s_scan = s_start + 4;                                   // [kThreads / 32]
  int* s_last = s_scan + kThreads / 32;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      bar_init(full + 8 * i, TMA ? 1 : 33);
      bar_init(empty + 8 * i, kWarps);
      bar_init(ready + 8 * i, 1);
    }
    bar_init_fence();
  }
  pdl_wait();

  // ---- this CTA's range of the flat tile list
  const int HR = p.HKV * p.row_tiles;
  int total, ctas, g0, count;   // tiles in all, CTAs that take part, this one's first tile and how many
  {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += span_of<TILE>(p, length_of(p, b)).n;
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
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    total *= HR;
    ctas = min(p.ctas, max(1, total / p.min_tiles));
    const int me = blockIdx.x;
    if (me >= ctas) return;
    const Cut cut(total, ctas);
    g0 = cut.begin(me);
    count = cut.begin(me + 1) - g0;
    // the thread whose sequences hold tile g0 finds the sequence
    if (mine > 0 && before * HR <= g0 && g0 < (before + mine) * HR) {
      int b = b0;
      if (per > 1)
        for (;; ++b) {
          const int nb = span_of<TILE>(p, length_of(p, b)).n;
          if (g0 < (before + nb) * HR) break;
          before += nb;
        }
      s_start[0] = b;
      s_start[1] = before;
      s_start[2] = p.lengths[b];
    }
    __syncthreads();
  }
  bool failed = false;

  if (warp == kWarps) {
    // ------------------------------------------------------------ producer
    int ld_b = s_start[0], ld_left = count, ld_hr, ld_tile;
    int ld_len = min(max(s_start[2], 0), p.cap);
    bool ld_over = s_start[2] > p.cap;
    Span ld_span = span_of<TILE>(p, ld_len);
    int ld_seg = s_start[1] * HR;
    {
      const int off = g0 - ld_seg;
      ld_hr = off / ld_span.n;
      ld_tile = off - ld_hr * ld_span.n;
      ld_seg += ld_hr * ld_span.n;
    }
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
      u.d.h = ld_hr / p.row_tiles;
      u.d.rt = ld_hr - u.d.h * p.row_tiles;
      u.d.token0 = token0;
      u.d.len = ld_len;
      u.d.first = ld_first;
      u.d.n_tiles = ld_span.n;
      u.d.seg_start = ld_seg;
      --ld_left;
      u.d.last = ld_left == 0 || ld_tile + 1 == ld_span.n;
      const int step = TMA ? p.box : 1;
#pragma unroll
      for (int x = 0; x < LU; ++x) {
        const int at = (x * 32 + lane) * step, j = token0 + at;
        u.state[x] = 0;
        u.id[x] = 0;
        u.row[x] = 0;
        if (at < TILE && j < ld_len && (j + step > ld_span.lo || j < p.sinks)) {
          const int pg = j / p.page;
          u.row[x] = j - pg * p.page;
          u.state[x] = ld_over ? 2 : 1;
          u.id[x] = __ldg(p.table + (int64_t)ld_b * p.table_b + pg);
        }
      }
      ld_first = false;
      if (++ld_tile == ld_span.n && ld_left > 0) {
        ld_first = true;
        ld_tile = 0;
        ld_seg += ld_span.n;
        if (++ld_hr == HR) {
          ld_hr = 0;
          ++ld_b;
          ld_len = min(max(next_raw, 0), p.cap);
          ld_over = next_raw > p.cap;
          ld_span = span_of<TILE>(p, ld_len);
          next_raw = ld_b + 1 < p.B ? p.lengths[ld_b + 1] : 0;
        }
      }
    };
    Lookup next;
    look(next);
    for (int i = 0; i < count; ++i) {
      Lookup u = next;
      look(next);
      const int slot = i % S;
      if (i >= S) bar_wait(empty + 8 * slot, (i / S - 1) & 1, failed);
      const uint32_t kdst = sbase + slot * C::STAGE, vdst = kdst + C::KV_BYTES;
      if constexpr (TMA) {
        const bool ok = u.state[0] == 1 && u.id[0] >= 0 && u.id[0] < p.num_pages;
        const uint32_t good = __ballot_sync(0xffffffffu, ok);
        const uint32_t bad = __ballot_sync(0xffffffffu, u.state[0] != 0 && !ok);
#pragma unroll
        for (int w = 0; w < 4; ++w) u.d.bad[w] = 0;
        if (bad)
#pragma unroll
          for (int w = 0; w < TILE / 32; ++w)
            u.d.bad[w] = __ballot_sync(0xffffffffu, (bad >> ((w * 32 + lane) / p.box)) & 1);
        if (lane == 0) {
          descs[slot] = u.d;
          bar_arrive(ready + 8 * slot);
          bar_arrive_tx(full + 8 * slot, __popc(good) * p.box * 128 * C::HALVES * 2);
        }
        __syncwarp();
        if (ok && !failed) {
          const uint32_t at = lane * p.box * 128;
#pragma unroll
          for (int hf = 0; hf < C::HALVES; ++hf) {
            tma_box(kdst + hf * C::HALF_BYTES + at, &kmap, full + 8 * slot, hf * 64, u.row[0], u.d.h, u.id[0]);
            tma_box(vdst + hf * C::HALF_BYTES + at, &vmap, full + 8 * slot, hf * 64, u.row[0], u.d.h, u.id[0]);
          }
        }
      } else {
        int64_t ko[LU], vo[LU];
#pragma unroll
        for (int w = 0; w < 4; ++w) u.d.bad[w] = 0;
#pragma unroll
        for (int x = 0; x < LU; ++x) {
          const bool ok = u.state[x] == 1 && u.id[x] >= 0 && u.id[x] < p.num_pages;
          u.d.bad[x] = __ballot_sync(0xffffffffu, u.state[x] != 0 && !ok);
          ko[x] = !ok ? -1 : (int64_t)u.id[x] * p.k_page + (int64_t)u.d.h * p.k_head + (int64_t)u.row[x] * p.k_row;
          vo[x] = !ok ? -1 : (int64_t)u.id[x] * p.v_page + (int64_t)u.d.h * p.v_head + (int64_t)u.row[x] * p.v_row;
        }
        if (lane == 0) {
          descs[slot] = u.d;
          bar_arrive(ready + 8 * slot);
        }
        constexpr int RPI = 32 / C::PIECES;   // rows per step
        const int c = lane % C::PIECES, sub = lane / C::PIECES;
#pragma unroll
        for (int x = 0; x < LU; ++x)
#pragma unroll 4
          for (int r0 = 0; r0 < 32; r0 += RPI) {
            const int64_t k_at = __shfl_sync(0xffffffffu, ko[x], r0 + sub), v_at = __shfl_sync(0xffffffffu, vo[x], r0 + sub);
            const int r = x * 32 + r0 + sub;
            const uint32_t at = (c >> 3) * C::HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            if (k_at >= 0) {
              cp_async16(kdst + at, p.k + k_at + c * 8);
              cp_async16(vdst + at, p.v + v_at + c * 8);
            }
          }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(full + 8 * slot) : "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(full + 8 * slot);
      }
    }
    // consumers wait for every tile; after a wait that ran out, see the copies in flight off
    if (failed)
      for (int i = max(0, count - S); i < count; ++i) bar_wait_long(full + 8 * (i % S), (i / S) & 1);
    return;
  }

  // -------------------------------------------------------------- consumers
  uint32_t qf[MT <= 2 ? MT : 1][D / 16][4];   // query fragments (MT = 4 reads them from shared memory)
  float o[MT][C::DT][4];
  float m[MT][2], l[MT][2];
  int back[MT][2];                            // T - t of the thread's rows: position = len - back
  // Fragment addresses: 128-byte rows, 16-byte piece c of row r at c ^ (r & 7); the rows of a thread's
  // ldmatrix lanes all have r & 7 = lane & 7.
  const uint32_t swz = (lane & 7) << 4;
  const uint32_t k_row = (warp * (TILE / kWarps) + ((lane >> 4) << 3) + (lane & 7)) * 128, k_col = ((lane >> 3) & 1) << 4;
  const uint32_t v_at = (lane & 15) * 128 + ((warp * C::DW) >> 6) * C::HALF_BYTES;
  const uint32_t v_col = ((warp * C::DW) & 63) * 2 + ((lane >> 4) << 4);
  const uint32_t a_row = lane & 15, a_col = (lane >> 4) << 4;   // Q and P operands

  for (int i = 0; i < count; ++i) {
    const int slot = i % S;
    bar_wait(ready + 8 * slot, (i / S) & 1, failed);
    const Desc& ds = descs[slot];
    const int len = ds.len, token0 = ds.token0, rt = ds.rt;

    if (ds.first) {
      // query rows of this segment, while its first tile is on the way: row r = t * G + g
      for (int x = tid; x < ROWS * C::PIECES; x += kConsumers) {
        const int r = x / C::PIECES, c = x % C::PIECES;
        const int R = rt * ROWS + r;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (R < p.R) {
          const int t = R / p.G, g = R - t * p.G;
          w = *reinterpret_cast<const uint4*>(p.q + (int64_t)ds.b * p.q_b + (int64_t)(ds.h * p.G + g) * p.q_h +
                                              (int64_t)t * p.q_t + c * 8);
        }
        *reinterpret_cast<uint4*>(smem + C::OFF_Q + r * D * 2 + ((c ^ (r & 7)) << 4)) = w;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int R = rt * ROWS + mt * 16 + e * 8 + lane / 4;
          back[mt][e] = p.T - min(R, p.R - 1) / p.G;
          m[mt][e] = -INFINITY;
          l[mt][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < C::DT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
      }
      consumer_sync();
      if constexpr (MT <= 2) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            ldsm_x4(sbase + C::OFF_Q + (mt * 16 + a_row) * D * 2 + ((kk * 32 + a_col) ^ swz), qf[mt][kk][0],
                    qf[mt][kk][1], qf[mt][kk][2], qf[mt][kk][3]);
      }
    }

    bar_wait(full + 8 * slot, (i / S) & 1, failed);

    // ---- scores: this warp's TILE/4 tokens x all rows
    const uint32_t kb = sbase + slot * C::STAGE, vb = kb + C::KV_BYTES;
    float s[MT][C::NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t bf[C::NT][2];
#pragma unroll
      for (int n2 = 0; n2 < C::NT / 2; ++n2)
        ldsm_x4(kb + k_row + n2 * 2048 + (kk >> 2) * C::HALF_BYTES + (((kk & 3) * 32 + k_col) ^ swz), bf[2 * n2][0],
                bf[2 * n2][1], bf[2 * n2 + 1][0], bf[2 * n2 + 1][1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a[4];
        if constexpr (MT <= 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = qf[mt][kk][e];
        } else {
          ldsm_x4(sbase + C::OFF_Q + (mt * 16 + a_row) * D * 2 + ((kk * 32 + a_col) ^ swz), a[0], a[1], a[2], a[3]);
        }
#pragma unroll
        for (int n = 0; n < C::NT; ++n) mma_e<HALF>(s[mt][n], a[0], a[1], a[2], a[3], bf[n][0], bf[n][1]);
      }
    }
    const int in_tile = warp * (TILE / kWarps) + (lane & 3) * 2;   // token of n-tile 0, element 0
    const int tok = token0 + in_tile;
    // every row sees every token of the tile: positions run from len - T to len - 1
    const bool full_tile = token0 + TILE <= len - p.T + 1 &&
                           (p.window == 0 || token0 > len - 1 - p.window || token0 + TILE <= p.sinks) &&
                           (ds.bad[0] | ds.bad[1] | ds.bad[2] | ds.bad[3]) == 0;
    float mx[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      mx[mt][0] = mx[mt][1] = -INFINITY;
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[mt][n][e] * p.scale2;
          if (!full_tile) {
            const int at = in_tile + n * 8 + (e & 1), j = token0 + at, pos = len - back[mt][e >> 1];
            const bool seen = j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
            // a page outside the pool: the rows that see it say so
            x = !seen ? -INFINITY : (ds.bad[at >> 5] >> (at & 31)) & 1 ? NAN : x;
          }
          s[mt][n][e] = x;
          mx[mt][e >> 1] = fmaxf(mx[mt][e >> 1], x);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[mt][e] = fmaxf(mx[mt][e], __shfl_xor_sync(0xffffffffu, mx[mt][e], 1));
        mx[mt][e] = fmaxf(mx[mt][e], __shfl_xor_sync(0xffffffffu, mx[mt][e], 2));
        if ((lane & 3) == 0) smax[warp * ROWS + mt * 16 + e * 8 + lane / 4] = mx[mt][e];
      }
    }
    if (p.scores != nullptr) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int R = rt * ROWS + mt * 16 + e * 8 + lane / 4;
          if (R < p.R) {
            float* dst = p.scores + ((int64_t)(ds.b * p.HKV + ds.h) * p.R + R) * p.score_stride + tok;
#pragma unroll
            for (int n = 0; n < C::NT; ++n)
              *reinterpret_cast<float2*>(dst + n * 8) = make_float2(s[mt][n][2 * e], s[mt][n][2 * e + 1]);
          }
        }
    }
    if (!full_tile) {
      // rows of V that no query sees hold whatever the page or an earlier
      // tile left there, and 0 * NaN is NaN: zero them
      const int lo = p.window > 0 ? max(0, max(len - p.T, 0) - p.window + 1) : 0;
      for (int x = tid; x < TILE * C::PIECES; x += kConsumers) {
        const int r = x / C::PIECES, c = x % C::PIECES, j = token0 + r;
        if (j < len && (j >= lo || j < p.sinks) && !((ds.bad[r >> 5] >> (r & 31)) & 1)) continue;
        *reinterpret_cast<uint4*>(smem + slot * C::STAGE + C::KV_BYTES + (c >> 3) * C::HALF_BYTES + r * 128 +
                                  ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
      }
    }
    consumer_sync();

    // ---- running maximum and sum; P to shared memory.  The tensor cores
    // take it in the pages' type: as the rounded value and the rounded rest,
    // two products, so that the output's own rounding stays the largest error
    // (one rounded value alone doubles it).
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = mt * 16 + e * 8 + lane / 4;
        float mn = m[mt][e];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mn = fmaxf(mn, smax[w * ROWS + r]);
        const float mu = finite_or_zero(mn);
        const float alpha = fast_exp2(m[mt][e] - mu);
        m[mt][e] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          const float p0 = fast_exp2(s[mt][n][2 * e] - mu), p1 = fast_exp2(s[mt][n][2 * e + 1] - mu);
          sum += p0 + p1;
          const int c = warp * (TILE / kWarps / 8) + n;   // 8-token piece of the row
          const uint32_t hi = pack2<HALF>(p0, p1);
          const uint32_t lo = pack2<HALF>(p0 - to_float<HALF>((uint16_t)hi), p1 - to_float<HALF>((uint16_t)(hi >> 16)));
          uint8_t* dst = smem + C::OFF_P + r * TILE * 2 + ((c ^ (r & 7)) << 4) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(dst) = hi;
          *reinterpret_cast<uint32_t*>(dst + C::P_HALF) = lo;
        }
        l[mt][e] = l[mt][e] * alpha + sum;
#pragma unroll
        for (int n = 0; n < C::DT; ++n) {
          o[mt][n][2 * e] *= alpha;
          o[mt][n][2 * e + 1] *= alpha;
        }
      }
    consumer_sync();

    // A token that some rows see and others do not has weight 0 in the
    // others, and 0 * inf is NaN in the product below.  Such tokens exist for
    // T > 1 only, T - 1 of them at either end of the span.  When one of them
    // holds an infinity or NaN, they are added by hand to the rows that see
    // them and then zeroed.
    if (p.T > 1 && !full_tile) {
      const int lo = p.window > 0 ? max(0, max(len - p.T, 0) - p.window + 1) : 0;
      const int n_part = (p.window > 0 ? 2 : 1) * (p.T - 1);
      // the n-th such token's row in the tile, or -1
      auto part_row = [&](int n) {
        const int j = n < p.T - 1 ? len - 1 - n : lo + n - (p.T - 1);
        return j >= 0 && j < len && j >= token0 && j < token0 + TILE ? j - token0 : -1;
      };
      uint8_t* vs = smem + slot * C::STAGE + C::KV_BYTES;
      int odd = 0;
      for (int x = tid; x < n_part * C::PIECES; x += kConsumers) {
        const int r = part_row(x / C::PIECES), c = x % C::PIECES;
        if (r < 0) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(vs + (c >> 3) * C::HALF_BYTES + r * 128 + ((c & 7) << 4));
        const uint32_t ones = HALF ? 0x7c00u : 0x7f80u;
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) odd |= (ws[y] & ones) == ones || ((ws[y] >> 16) & ones) == ones;
      }
      int any;
      asm volatile("{\n.reg .pred a, b;\nsetp.ne.s32 a, %1, 0;\nbar.red.or.pred b, 1, 128, a;\nselp.s32 %0, 1, 0, b;\n}\n"
                   : "=r"(any)
                   : "r"(odd)
                   : "memory");
      if (any) {
        for (int n = 0; n < n_part; ++n) {
          const int r = part_row(n), j = token0 + r;
          if (r < 0 || (n >= p.T - 1 && j > len - p.T)) continue;   // both ends may name it: once
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int pos = len - back[mt][e], row = mt * 16 + e * 8 + lane / 4;
              if (!(j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks))) continue;
              const uint8_t* pw = smem + C::OFF_P + row * TILE * 2 + (((r >> 3) ^ (row & 7)) << 4) + (r & 7) * 2;
              const float w = to_float<HALF>(*reinterpret_cast<const uint16_t*>(pw)) +
                              to_float<HALF>(*reinterpret_cast<const uint16_t*>(pw + C::P_HALF));
#pragma unroll
              for (int x = 0; x < C::DT; ++x) {
                const int col = warp * C::DW + x * 8 + (lane & 3) * 2;
                const uint32_t vv = *reinterpret_cast<const uint32_t*>(
                    vs + (col >> 6) * C::HALF_BYTES + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4) + (col & 7) * 2);
                o[mt][x][2 * e] += w * to_float<HALF>((uint16_t)vv);
                o[mt][x][2 * e + 1] += w * to_float<HALF>((uint16_t)(vv >> 16));
              }
            }
        }
        consumer_sync();
        for (int x = tid; x < n_part * C::PIECES; x += kConsumers) {
          const int r = part_row(x / C::PIECES), c = x % C::PIECES;
          if (r >= 0)
            *reinterpret_cast<uint4*>(vs + (c >> 3) * C::HALF_BYTES + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        consumer_sync();
      }
    }

    // ---- output: all tokens x this warp's D/4 columns
#pragma unroll
    for (int kk = 0; kk < TILE / 16; ++kk) {
      uint32_t bf[C::DT][2];
#pragma unroll
      for (int n2 = 0; n2 < C::DT / 2; ++n2)
        ldsm_x4_trans(vb + v_at + kk * 2048 + ((n2 * 32 + v_col) ^ swz), bf[2 * n2][0], bf[2 * n2][1],
                      bf[2 * n2 + 1][0], bf[2 * n2 + 1][1]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t at = sbase + C::OFF_P + (mt * 16 + a_row) * TILE * 2 + ((kk * 32 + a_col) ^ swz);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t a[4];
          ldsm_x4(at + part * C::P_HALF, a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < C::DT; ++n) mma_e<HALF>(o[mt][n], a[0], a[1], a[2], a[3], bf[n][0], bf[n][1]);
        }
      }
    }

    const bool last = ds.last;
    const int sb = ds.b, sh = ds.h, n_tiles = ds.n_tiles;
    const int seg_start = ds.seg_start;
    // the tile is read: hand it back (zeroed rows are ordinary stores, which the TMA must not overtake)
    if (!full_tile) asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncwarp();
    if (lane == 0) bar_arrive(empty + 8 * slot);

    if (last) {
      // ---- the rows' sums over the four warps
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = failed ? NAN : l[mt][e];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if ((lane & 3) == 0) ssum[warp * ROWS + mt * 16 + e * 8 + lane / 4] = x;
        }
      consumer_sync();
      const bool whole = g0 <= seg_start && g0 + i == seg_start + n_tiles - 1;
      const int64_t slot_o = blockIdx.x * 2 + (seg_start > g0 ? 1 : 0);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = mt * 16 + e * 8 + lane / 4, R = rt * ROWS + r;
          if (R >= p.R) continue;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) sum += ssum[w * ROWS + r];
          const int col = warp * C::DW + (lane & 3) * 2;
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int t = R / p.G, g = R - t * p.G;
            const int64_t row = ((int64_t)sb * p.HQ + sh * p.G + g) * p.T + t;
#pragma unroll
            for (int n = 0; n < C::DT; ++n)
              *reinterpret_cast<uint32_t*>(p.out + row * D + col + n * 8) =
                  pack2<HALF>(o[mt][n][2 * e] * inv, o[mt][n][2 * e + 1] * inv);
            if (warp == 0 && (lane & 3) == 0) {
              const float lse2 = sum == 0.f ? -INFINITY : finite_or_zero(m[mt][e]) + log2f(sum);
              if (p.lse) p.lse[row] = lse2 * 0.6931471805599453f;
              if (p.row_lse2) p.row_lse2[(int64_t)(sb * p.HKV + sh) * p.R + R] = lse2;
            }
          } else {
            float* po = p.part_o + (slot_o * ROWS + r) * D + col;
#pragma unroll
            for (int n = 0; n < C::DT; ++n)
              *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
            if (warp == 0 && (lane & 3) == 0)
              *reinterpret_cast<float2*>(p.part_ml + (slot_o * ROWS + r) * 2) = make_float2(m[mt][e], sum);
          }
        }
      if (!whole) {
        // ---- join.  The CTAs c0..c1 of the segment arrive in groups of
        // kGroup; a group's last adds its parts up, the last group's last
        // adds the groups up and writes the rows: two rounds of a few
        // independent loads instead of one long chain.  The order of the
        // sums is the CTAs', whoever does them.
        const Cut cut(total, ctas);
        const int c0 = cut.owner(seg_start), c1 = cut.owner(seg_start + n_tiles - 1);
        const int n = c1 - c0 + 1, groups = (n + kGroup - 1) / kGroup;
        const int n_rows = min(ROWS, p.R - rt * ROWS);
        // part k of the segment: CTA c0 + k; CTA c0's second part when it began with another segment.
        // A group's sum: behind all parts, by its first CTA.
        const int first_slot = c0 * 2 + (cut.begin(c0) < seg_start ? 1 : 0);
        // parts [k0, k0 + cnt) of the segment, or its group sums, -> the rows, or group sum `to`
        auto join = [&](int k0, int cnt, bool of_groups, int to) {
          auto slot_of = [&](int k) {
            if (!of_groups) return k0 + k == 0 ? first_slot : (c0 + k0 + k) * 2;
            return k * kGroup + 1 == n ? c1 * 2 : 2 * p.ctas + c0 + k * kGroup;   // a group of one is its part
          };
#pragma unroll 1
          for (int x = tid; x < n_rows * (D / 4); x += kConsumers) {
            const int r = x / (D / 4), col = x % (D / 4) * 4;
            float mm = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int kb = 0; kb < cnt; kb += 8) {
              float2 ml[8];
              float4 f[8];
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                ml[y] = make_float2(-INFINITY, 0.f);
                f[y] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (kb + y < cnt) {
                  const int64_t at = (int64_t)slot_of(kb + y) * ROWS + r;
                  ml[y] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
                  f[y] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + col));
                }
              }
              float mn = mm;
#pragma unroll
              for (int y = 0; y < 8; ++y) mn = fmaxf(mn, ml[y].x);
              const float mu = finite_or_zero(mn), alpha = fast_exp2(mm - mu);
              mm = mn;
              sum *= alpha;
              acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
#pragma unroll
              for (int y = 0; y < 8; ++y) {
                const float w = fast_exp2(ml[y].x - mu);
                sum += w * ml[y].y;
                acc.x += w * f[y].x; acc.y += w * f[y].y; acc.z += w * f[y].z; acc.w += w * f[y].w;
              }
            }
            if (to >= 0) {
              const int64_t at = (int64_t)(2 * p.ctas + to) * ROWS + r;
              *reinterpret_cast<float4*>(p.part_o + at * D + col) = acc;
              if (col == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mm, sum);
              continue;
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int R = rt * ROWS + r, t = R / p.G, g = R - t * p.G;
            const int64_t row = ((int64_t)sb * p.HQ + sh * p.G + g) * p.T + t;
            *reinterpret_cast<uint2*>(p.out + row * D + col) =
                make_uint2(pack2<HALF>(acc.x * inv, acc.y * inv), pack2<HALF>(acc.z * inv, acc.w * inv));
            if (col == 0) {
              const float lse2 = sum == 0.f ? -INFINITY : finite_or_zero(mm) + log2f(sum);
              if (p.lse) p.lse[row] = lse2 * 0.6931471805599453f;
              if (p.row_lse2) p.row_lse2[(int64_t)(sb * p.HKV + sh) * p.R + R] = lse2;
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
        consumer_sync();   // s_last and the statistics are free again
      }
    }
  }
}

// token_weights[b, j] += sum over the heads and new tokens of 2^(x - lse2).
// One thread per token, the rows in order: no atomics, a fixed order of sums.
template <int TILE>
__global__ void weights_kernel(const __grid_constant__ Params p, float* weights, int64_t weights_b) {
  extern __shared__ float lse2[];
  pdl_wait();
  const int b = blockIdx.y, rows = p.HKV * p.R;
  const int len = length_of(p, b);
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if ((int)(blockIdx.x * blockDim.x) >= len) return;
  for (int r = threadIdx.x; r < rows; r += blockDim.x) lse2[r] = finite_or_zero(p.row_lse2[(int64_t)b * rows + r]);
  __syncthreads();
  if (j >= len) return;
  const Span s = span_of<TILE>(p, len);
  if (j < s.lo && j >= p.sinks) return;
  const float* src = p.scores + (int64_t)b * rows * p.score_stride + j;
  float sum = 0.f;
#pragma unroll 4
  for (int r = 0; r < rows; ++r) sum += fast_exp2(src[(int64_t)r * p.score_stride] - lse2[r]);
  weights[(int64_t)b * weights_b + j] += sum;
}

// New token t of sequence b goes to row j % page of page table[b, j / page],
// j = L - T + t.  A row whose page is not in the pool is not written (the
// attention over it gives NaN).
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

struct Plan {
  int G, R, mt, row_tiles, cap, ctas;
  int64_t score_stride;
  size_t part_o, part_ml, lse2, scores;
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
  const int tile = a->head_dim == 64 ? 128 : 64;
  // 2^30 keeps token positions and the rows' products inside 32 bits
  if (cap > (1 << 30) || R > (1 << 20) || (int64_t)a->batch * a->kv_heads * R > (1ll << 31) - 1)
    return KVR_ERR_UNSUPPORTED;
  // weights_kernel: 48 KB of row statistics, the batch along the grid's y
  if (a->token_weights && (a->kv_heads * R > 12000 || a->batch > 65535)) return KVR_ERR_UNSUPPORTED;
  p.R = (int)R;
  p.cap = (int)cap;
  p.mt = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  p.row_tiles = (p.R + 16 * p.mt - 1) / (16 * p.mt);
  const int64_t tiles = std::max<int64_t>(1, (cap + tile - 1) / tile + 1) * a->batch * a->kv_heads * p.row_tiles;
  if (tiles > (1ll << 31) - 1) return KVR_ERR_UNSUPPORTED;
  // two CTAs per SM; a join takes kGroup^2 parts and some
  p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(tiles, std::min(2 * num_sms_of(a->num_sms), kGroup * 20)));
  p.score_stride = std::max<int64_t>(128, (cap + 127) / 128 * 128);
  const size_t rows = (size_t)16 * p.mt * 3 * p.ctas;
  p.part_o = rows * a->head_dim * sizeof(float);
  p.part_ml = rows * 2 * sizeof(float);
  const size_t all_rows = (size_t)a->batch * a->kv_heads * p.R;
  p.lse2 = a->token_weights ? (all_rows * sizeof(float) + 255) / 256 * 256 : 0;
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

template <bool HALF, int D, int MT, bool TMA>
static int launch(const Params& p, const Maps& maps, cudaStream_t s) {
  using C = Cfg<D, MT>;
  auto kern = attention_kernel<HALF, D, MT, TMA>;
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
static int launch_mt(int mt, const Params& p, const Maps& maps, cudaStream_t s) {
  if (mt == 1) return launch<HALF, D, 1, TMA>(p, maps, s);
  if (mt == 2) return launch<HALF, D, 2, TMA>(p, maps, s);
  return launch<HALF, D, 4, TMA>(p, maps, s);
}
template <bool HALF, int D>
static int launch_tma(bool tma, int mt, const Params& p, const Maps& maps, cudaStream_t s) {
  return tma ? launch_mt<HALF, D, true>(mt, p, maps, s) : launch_mt<HALF, D, false>(mt, p, maps, s);
}

}  // namespace paged
}  // namespace kvr

using namespace kvr;

extern "C" int kvr_paged_attention_plan(const kvr_paged_attention_args* a, size_t* workspace_bytes,
                                        size_t* counter_count, size_t* scores_bytes) {
  paged::Plan p;
  const int st = paged::plan_of(a, &p);
  if (st != KVR_OK) return st;
  if (workspace_bytes) *workspace_bytes = p.part_o + p.part_ml;
  if (counter_count) *counter_count = 2 * (size_t)p.ctas;
  if (scores_bytes) *scores_bytes = p.lse2 + p.scores;
  return KVR_OK;
}

extern "C" int kvr_paged_attention(const kvr_paged_attention_args* a, kvr_stream_t stream) {
  paged::Plan pl;
  int st = paged::plan_of(a, &pl);
  if (st != KVR_OK) return st;
  if (a->batch == 0) return KVR_OK;
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
  if (a->token_weights && (!a->scores || a->scores_bytes < pl.lse2 + pl.scores)) return KVR_ERR_WORKSPACE;
  if (a->token_weights && !aligned16(a->scores)) return KVR_ERR_MISALIGNED;

  paged::Params p;
  p.q = static_cast<const uint16_t*>(a->query);
  p.q_b = a->q_b_stride; p.q_h = a->q_h_stride; p.q_t = a->q_t_stride;
  p.k = static_cast<const uint16_t*>(a->key_pages);
  p.k_page = a->key_page_stride; p.k_head = a->key_head_stride; p.k_row = a->key_row_stride;
  p.v = static_cast<const uint16_t*>(a->value_pages);
  p.v_page = a->value_page_stride; p.v_head = a->value_head_stride; p.v_row = a->value_row_stride;
  p.table = a->block_table; p.table_b = a->table_stride;
  p.table_width = a->table_width; p.num_pages = a->num_pages; p.page = a->page_size;
  p.lengths = a->lengths;
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.row_lse2 = a->token_weights ? static_cast<float*>(a->scores) : nullptr;
  p.scores = a->token_weights ? reinterpret_cast<float*>(static_cast<uint8_t*>(a->scores) + pl.lse2) : nullptr;
  p.score_stride = pl.score_stride;
  p.B = a->batch; p.HQ = a->q_heads; p.HKV = a->kv_heads; p.T = a->new_tokens;
  p.G = pl.G; p.R = pl.R; p.row_tiles = pl.row_tiles;
  p.window = a->window; p.sinks = a->window > 0 ? a->sinks : 0; p.cap = pl.cap;
  p.scale2 = a->scale * 1.4426950408889634f;
  p.ctas = pl.ctas; p.min_tiles = 1;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + pl.part_o);
  p.counters = a->counters;
  cudaStream_t s = as_stream(stream);
  const bool half = a->dtype == 1;
  // TMA boxes: the largest number of tokens that divides both a page and a
  // tile; below 8 rows (one swizzle pattern) the rows are copied one by one.
  const int tile = a->head_dim == 64 ? 128 : 64;
  int box = tile;
  while (a->page_size % box) box /= 2;
  p.box = box;
  paged::Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  const bool tma = box >= 8 &&
                   paged::page_map(&maps.k, a->key_pages, half, a->head_dim, a->page_size, a->kv_heads, a->num_pages,
                                   a->key_row_stride, a->key_head_stride, a->key_page_stride, box) &&
                   paged::page_map(&maps.v, a->value_pages, half, a->head_dim, a->page_size, a->kv_heads, a->num_pages,
                                   a->value_row_stride, a->value_head_stride, a->value_page_stride, box);
  if (a->head_dim == 64)
    st = half ? paged::launch_tma<true, 64>(tma, pl.mt, p, maps, s) : paged::launch_tma<false, 64>(tma, pl.mt, p, maps, s);
  else
    st = half ? paged::launch_tma<true, 128>(tma, pl.mt, p, maps, s) : paged::launch_tma<false, 128>(tma, pl.mt, p, maps, s);
  if (st != KVR_OK || !a->token_weights || pl.cap == 0) return st;
  const int rows = p.HKV * p.R;
  const dim3 grid((pl.cap + 255) / 256, p.B);
  cudaError_t e = a->head_dim == 64
                      ? pdl_launch(paged::weights_kernel<128>, grid, dim3(256), rows * sizeof(float), s, 1, p,
                                   a->token_weights, a->weights_b_stride)
                      : pdl_launch(paged::weights_kernel<64>, grid, dim3(256), rows * sizeof(float), s, 1, p,
                                   a->token_weights, a->weights_b_stride);
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
