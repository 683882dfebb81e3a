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
// loads in flight:
//  * Work is a flat list of token tiles (sequence, KV head, row tile, tile),
//    cut into equal ranges, one per CTA.  Lengths are read on the device, so
//    a ragged batch is balanced to one tile without the host knowing it.
//  * The tiles stream through a cp.async ring that runs on across sequence
//    boundaries; page numbers are looked up one step ahead of the copies.
//  * The four warps of a CTA share each tile: for the scores a warp owns a
//    quarter of the tokens, for the output a quarter of the head dimension,
//    so every byte of K and V is read from shared memory once and the
//    accumulator is complete in the CTA: nothing is merged between warps.
//  * A sequence that several CTAs share is joined by the last of them to
//    arrive, in the order of the CTAs: the result does not depend on timing.
#include "kvr_common.cuh"

#include <algorithm>

namespace kvr {
namespace paged {

constexpr int kThreads = 128;
constexpr int kWarps = 4;

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
  float* part_o;    // [2 * ctas][ROWS][D]
  float* part_ml;   // [2 * ctas][ROWS][2]
  int* counters;    // [ctas], zero on entry and on exit
};

template <int D, int MT>
struct Cfg {
  static constexpr int TILE = D == 64 ? 128 : 64;   // tokens: 16 KB of K and 16 KB of V either way
  static constexpr int ROWS = 16 * MT;
  static constexpr int ROW_BYTES = 2 * D;
  static constexpr int PIECES = D / 8;
  static constexpr int KV_BYTES = TILE * ROW_BYTES;
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int STAGES = MT == 4 ? 2 : 3;    // two CTAs per SM in every case
  static constexpr int NT = TILE / kWarps / 8;      // 8-token score tiles of a warp
  static constexpr int DW = D / kWarps;             // output columns of a warp
  static constexpr int DT = DW / 8;
  static constexpr int DESCS = 4;
  // shared memory: ring, Q, P, row offsets, descriptors, row statistics
  // (MT <= 2 keeps Q in registers and lets P take its place)
  static constexpr int Q_BYTES = ROWS * ROW_BYTES, P_HALF = ROWS * TILE * 2, P_BYTES = 2 * P_HALF;
  static constexpr int OFF_Q = STAGES * STAGE;
  static constexpr int OFF_P = MT <= 2 ? OFF_Q : OFF_Q + Q_BYTES;
  static constexpr int OFF_ROW = OFF_Q + (MT <= 2 ? (Q_BYTES > P_BYTES ? Q_BYTES : P_BYTES) : Q_BYTES + P_BYTES);
  static constexpr int OFF_DESC = OFF_ROW + STAGES * TILE * 16;
  static constexpr int OFF_MAX = OFF_DESC + DESCS * 64;
  static constexpr int OFF_SUM = OFF_MAX + kWarps * ROWS * 4;
  static constexpr int SMEM = OFF_SUM + kWarps * ROWS * 4 + 64;
};

struct Desc {
  int b, h, rt, token0, len, first, last, n_tiles;
  int64_t seg_start;
};
static_assert(sizeof(Desc) <= 64, "");

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

template <bool HALF, int D, int MT>
__global__ void __launch_bounds__(kThreads) attention_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D, MT>;
  constexpr int TILE = C::TILE, ROWS = C::ROWS, S = C::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t* row_off = reinterpret_cast<int64_t*>(smem + C::OFF_ROW);   // [S][TILE][2]
  Desc* descs = reinterpret_cast<Desc*>(smem + C::OFF_DESC);
  float* smax = reinterpret_cast<float*>(smem + C::OFF_MAX);
  float* ssum = reinterpret_cast<float*>(smem + C::OFF_SUM);

  pdl_wait();

  // ---- this CTA's range of the flat tile list
  const int HR = p.HKV * p.row_tiles;
  __shared__ int64_t s_start[4];   // {sequence, tiles before it, total}
  __shared__ int64_t s_scan[kWarps];
  __shared__ int s_last;
  int64_t total, g0, g1;
  {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += span_of<TILE>(p, length_of(p, b)).n;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int64_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += s_scan[w];
      total += s_scan[w];
    }
    total *= HR;
    const int64_t want = max((int64_t)1, total / p.min_tiles);
    const int64_t n = min((int64_t)p.ctas, want);
    if ((int64_t)blockIdx.x >= n) return;
    g0 = total * blockIdx.x / n;
    g1 = total * (blockIdx.x + 1) / n;
    // the thread whose sequences hold tile g0 finds the sequence
    int64_t before = base + incl - mine;
    if (mine > 0 && before * HR <= g0 && g0 < (before + mine) * HR) {
      int b = b0;
      for (;; ++b) {
        const int64_t nb = span_of<TILE>(p, length_of(p, b)).n;
        if (g0 < (before + nb) * HR) break;
        before += nb;
      }
      s_start[0] = b;
      s_start[1] = before;
      s_start[2] = n;
    }
    __syncthreads();
  }
  const int64_t ctas = s_start[2];
  const int count = (int)(g1 - g0);

  // ---- loader state: the next tile to look up
  int ld_b = (int)s_start[0], ld_left = count, ld_hr, ld_tile;
  int ld_len = length_of(p, ld_b);
  bool ld_over = p.lengths[ld_b] > p.cap;
  Span ld_span = span_of<TILE>(p, ld_len);
  int64_t ld_seg = s_start[1] * HR;
  {
    const int64_t off = g0 - ld_seg;
    ld_hr = (int)(off / ld_span.n);
    ld_tile = (int)(off - (int64_t)ld_hr * ld_span.n);
    ld_seg += (int64_t)ld_hr * ld_span.n;
  }
  int next_raw = ld_b + 1 < p.B ? p.lengths[ld_b + 1] : 0;
  bool ld_first = true;

  // One lookup: thread `tid` < TILE finds the page of token tid of the tile.
  // The page number is loaded here and used in `finish`, one iteration later.
  struct Lookup {
    int page_id, row, state;   // state 0: not needed, 1: page_id is valid once loaded, 2: outside the table
    Desc d;
    bool any;
  };
  auto look = [&]() {
    Lookup u;
    u.any = ld_left > 0;
    u.page_id = 0;
    u.row = 0;
    u.state = 0;
    if (!u.any) return u;
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
    if (tid < TILE) {
      const int j = token0 + tid;
      if (j < ld_len && (j >= ld_span.lo || j < p.sinks)) {
        const int pg = j / p.page;
        u.row = j - pg * p.page;
        u.state = ld_over ? 2 : 1;
        u.page_id = __ldg(p.table + (int64_t)ld_b * p.table_b + pg);
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
    return u;
  };
  auto finish = [&](const Lookup& u, int slot, int dslot) {
    if (!u.any) return;
    if (tid < TILE) {
      int64_t ko = -1, vo = -1;
      if (u.state) {
        const bool bad = u.state == 2 || u.page_id < 0 || u.page_id >= p.num_pages;
        ko = bad ? -2 : (int64_t)u.page_id * p.k_page + (int64_t)u.d.h * p.k_head + (int64_t)u.row * p.k_row;
        vo = bad ? -1 : (int64_t)u.page_id * p.v_page + (int64_t)u.d.h * p.v_head + (int64_t)u.row * p.v_row;
      }
      row_off[(slot * TILE + tid) * 2] = ko;
      row_off[(slot * TILE + tid) * 2 + 1] = vo;
    }
    if (tid == 0) descs[dslot] = u.d;
  };
  // Copies of one tile: rows of D elements in 16-byte pieces, piece c of row
  // r at c ^ (r & 7), so that the 8 rows of an ldmatrix hit 8 bank groups.
  auto issue = [&](int slot) {
    constexpr int RPI = kThreads / C::PIECES;   // rows per step
    const int c = tid % C::PIECES;
    const uint32_t kdst = sbase + slot * C::STAGE, vdst = kdst + C::KV_BYTES;
#pragma unroll
    for (int i = 0; i < TILE / RPI; ++i) {
      const int r = tid / C::PIECES + i * RPI;
      const longlong2 off = *reinterpret_cast<const longlong2*>(&row_off[(slot * TILE + r) * 2]);
      const uint32_t at = r * C::ROW_BYTES + ((c ^ (r & 7)) << 4);
      if (off.x >= 0) {
        cp_async16(kdst + at, p.k + off.x + c * 8);
        cp_async16(vdst + at, p.v + off.y + c * 8);
      } else {
        // no query sees this token: zeros, whatever the page holds there.  A
        // page outside the pool: NaN keys, so that the rows that see it say so.
        const uint32_t f = off.x == -2 ? 0x7fff7fffu : 0u;
        *reinterpret_cast<uint4*>(smem + slot * C::STAGE + at) = make_uint4(f, f, f, f);
        *reinterpret_cast<uint4*>(smem + slot * C::STAGE + C::KV_BYTES + at) = make_uint4(0, 0, 0, 0);
      }
    }
  };

  {
    Lookup u[S];
#pragma unroll
    for (int s = 0; s < S; ++s) u[s] = look();
#pragma unroll
    for (int s = 0; s < S; ++s) finish(u[s], s, s);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      if (s < count) issue(s);
      cp_async_commit();
    }
  }

  // ---- compute state
  uint32_t qf[MT <= 2 ? MT : 1][D / 16][4];   // query fragments (MT = 4 reads them from shared memory)
  float o[MT][C::DT][4];
  float m[MT][2], l[MT][2];
  int back[MT][2];                            // T - t of the thread's rows: position = len - back

  const int64_t part_rows = ROWS;
  for (int i = 0; i < count; ++i) {
    cp_async_wait<S - 2>();
    __syncthreads();
    const int slot = i % S;
    if (i + S - 1 < count) issue((i + S - 1) % S);
    cp_async_commit();
    const Lookup ahead = look();
    const Desc d = descs[i & (C::DESCS - 1)];

    if (d.first) {
      // query rows of this segment: row r = t * G + g
      for (int x = tid; x < ROWS * C::PIECES; x += kThreads) {
        const int r = x / C::PIECES, c = x % C::PIECES;
        const int R = d.rt * ROWS + r;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (R < p.R) {
          const int t = R / p.G, g = R - t * p.G;
          w = *reinterpret_cast<const uint4*>(p.q + (int64_t)d.b * p.q_b + (int64_t)(d.h * p.G + g) * p.q_h +
                                              (int64_t)t * p.q_t + c * 8);
        }
        *reinterpret_cast<uint4*>(smem + C::OFF_Q + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4)) = w;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int R = d.rt * ROWS + mt * 16 + e * 8 + lane / 4;
          back[mt][e] = p.T - min(R, p.R - 1) / p.G;
          m[mt][e] = -INFINITY;
          l[mt][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < C::DT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
      }
      __syncthreads();
      if constexpr (MT <= 2) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int r = mt * 16 + (lane & 15), c = kk * 2 + (lane >> 4);
            ldsm_x4(sbase + C::OFF_Q + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4), qf[mt][kk][0], qf[mt][kk][1],
                    qf[mt][kk][2], qf[mt][kk][3]);
          }
      }
    }

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
      for (int n2 = 0; n2 < C::NT / 2; ++n2) {
        const int r = warp * (TILE / kWarps) + n2 * 16 + ((lane >> 4) << 3) + (lane & 7);
        const int c = kk * 2 + ((lane >> 3) & 1);
        ldsm_x4(kb + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4), bf[2 * n2][0], bf[2 * n2][1], bf[2 * n2 + 1][0],
                bf[2 * n2 + 1][1]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a[4];
        if constexpr (MT <= 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = qf[mt][kk][e];
        } else {
          const int r = mt * 16 + (lane & 15), c = kk * 2 + (lane >> 4);
          ldsm_x4(sbase + C::OFF_Q + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4), a[0], a[1], a[2], a[3]);
        }
#pragma unroll
        for (int n = 0; n < C::NT; ++n) mma_e<HALF>(s[mt][n], a[0], a[1], a[2], a[3], bf[n][0], bf[n][1]);
      }
    }
    const int tok = d.token0 + warp * (TILE / kWarps) + (lane & 3) * 2;   // token of n-tile 0, element 0
    // every row sees every token of the tile: positions run from len - T to len - 1
    const bool full = d.token0 + TILE <= d.len - p.T + 1 &&
                      (p.window == 0 || d.token0 > d.len - 1 - p.window || d.token0 + TILE <= p.sinks);
    float mx[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      mx[mt][0] = mx[mt][1] = -INFINITY;
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[mt][n][e] * p.scale2;
          if (!full) {
            const int j = tok + n * 8 + (e & 1), pos = d.len - back[mt][e >> 1];
            const bool seen = j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks);
            x = seen ? x : -INFINITY;
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
          const int R = d.rt * ROWS + mt * 16 + e * 8 + lane / 4;
          if (R < p.R) {
            float* dst = p.scores + ((int64_t)(d.b * p.HKV + d.h) * p.R + R) * p.score_stride + tok;
#pragma unroll
            for (int n = 0; n < C::NT; ++n)
              *reinterpret_cast<float2*>(dst + n * 8) = make_float2(s[mt][n][2 * e], s[mt][n][2 * e + 1]);
          }
        }
    }
    __syncthreads();

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
    __syncthreads();

    // A token that some rows see and others do not has weight 0 in the
    // others, and 0 * inf is NaN in the product below.  Such tokens exist for
    // T > 1 only, T - 1 of them at either end of the span.  When one of them
    // holds an infinity or NaN, they are added by hand to the rows that see
    // them and then zeroed.
    if (p.T > 1 && !full) {
      const int lo = p.window > 0 ? max(0, max(d.len - p.T, 0) - p.window + 1) : 0;
      const int n_part = (p.window > 0 ? 2 : 1) * (p.T - 1);
      // the n-th such token's row in the tile, or -1
      auto part_row = [&](int n) {
        const int j = n < p.T - 1 ? d.len - 1 - n : lo + n - (p.T - 1);
        return j >= 0 && j < d.len && j >= d.token0 && j < d.token0 + TILE ? j - d.token0 : -1;
      };
      uint8_t* vs = smem + slot * C::STAGE + C::KV_BYTES;
      int odd = 0;
      for (int x = tid; x < n_part * C::PIECES; x += kThreads) {
        const int r = part_row(x / C::PIECES);
        if (r < 0) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(vs + r * C::ROW_BYTES + (x % C::PIECES << 4));
        const uint32_t ones = HALF ? 0x7c00u : 0x7f80u;
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) odd |= (ws[y] & ones) == ones || ((ws[y] >> 16) & ones) == ones;
      }
      if (__syncthreads_or(odd)) {
        for (int n = 0; n < n_part; ++n) {
          const int r = part_row(n), j = d.token0 + r;
          if (r < 0 || (n >= p.T - 1 && j > d.len - p.T)) continue;   // both ends may name it: once
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int pos = d.len - back[mt][e], row = mt * 16 + e * 8 + lane / 4;
              if (!(j <= pos && (p.window == 0 || j > pos - p.window || j < p.sinks))) continue;
              const uint8_t* pw = smem + C::OFF_P + row * TILE * 2 + (((r >> 3) ^ (row & 7)) << 4) + (r & 7) * 2;
              const float w = to_float<HALF>(*reinterpret_cast<const uint16_t*>(pw)) +
                              to_float<HALF>(*reinterpret_cast<const uint16_t*>(pw + C::P_HALF));
#pragma unroll
              for (int x = 0; x < C::DT; ++x) {
                const int col = warp * C::DW + x * 8 + (lane & 3) * 2;
                const uint32_t vv = *reinterpret_cast<const uint32_t*>(
                    vs + r * C::ROW_BYTES + (((col >> 3) ^ (r & 7)) << 4) + (col & 7) * 2);
                o[mt][x][2 * e] += w * to_float<HALF>((uint16_t)vv);
                o[mt][x][2 * e + 1] += w * to_float<HALF>((uint16_t)(vv >> 16));
              }
            }
        }
        __syncthreads();
        for (int x = tid; x < n_part * C::PIECES; x += kThreads) {
          const int r = part_row(x / C::PIECES);
          if (r >= 0)
            *reinterpret_cast<uint4*>(vs + r * C::ROW_BYTES + (x % C::PIECES << 4)) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
      }
    }

    // ---- output: all tokens x this warp's D/4 columns
#pragma unroll
    for (int kk = 0; kk < TILE / 16; ++kk) {
      uint32_t bf[C::DT][2];
#pragma unroll
      for (int n2 = 0; n2 < C::DT / 2; ++n2) {
        const int r = kk * 16 + (lane & 15);
        const int c = warp * (C::DW / 8) + n2 * 2 + (lane >> 4);
        ldsm_x4_trans(vb + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4), bf[2 * n2][0], bf[2 * n2][1], bf[2 * n2 + 1][0],
                      bf[2 * n2 + 1][1]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int r = mt * 16 + (lane & 15), c = kk * 2 + (lane >> 4);
        const uint32_t at = sbase + C::OFF_P + r * TILE * 2 + ((c ^ (r & 7)) << 4);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t a[4];
          ldsm_x4(at + part * C::P_HALF, a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < C::DT; ++n) mma_e<HALF>(o[mt][n], a[0], a[1], a[2], a[3], bf[n][0], bf[n][1]);
        }
      }
    }

    if (d.last) {
      // ---- the rows' sums over the four warps
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = l[mt][e];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if ((lane & 3) == 0) ssum[warp * ROWS + mt * 16 + e * 8 + lane / 4] = x;
        }
      __syncthreads();
      const int64_t at = g0 + i;                            // flat index of this tile
      const bool begins = g0 <= d.seg_start;                // the segment's first tile is ours
      const bool whole = begins && at == d.seg_start + d.n_tiles - 1;
      const int64_t slot_o = (int64_t)blockIdx.x * 2 + (d.seg_start > g0 ? 1 : 0);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = mt * 16 + e * 8 + lane / 4, R = d.rt * ROWS + r;
          if (R >= p.R) continue;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) sum += ssum[w * ROWS + r];
          const int col = warp * C::DW + (lane & 3) * 2;
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int t = R / p.G, g = R - t * p.G;
            const int64_t row = ((int64_t)d.b * p.HQ + d.h * p.G + g) * p.T + t;
#pragma unroll
            for (int n = 0; n < C::DT; ++n)
              *reinterpret_cast<uint32_t*>(p.out + row * D + col + n * 8) =
                  pack2<HALF>(o[mt][n][2 * e] * inv, o[mt][n][2 * e + 1] * inv);
            if (warp == 0 && (lane & 3) == 0) {
              const float lse2 = sum == 0.f ? -INFINITY : finite_or_zero(m[mt][e]) + log2f(sum);
              if (p.lse) p.lse[row] = lse2 * 0.6931471805599453f;
              if (p.row_lse2) p.row_lse2[(int64_t)(d.b * p.HKV + d.h) * p.R + R] = lse2;
            }
          } else {
            float* po = p.part_o + (slot_o * part_rows + r) * D + col;
#pragma unroll
            for (int n = 0; n < C::DT; ++n)
              *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
            if (warp == 0 && (lane & 3) == 0)
              *reinterpret_cast<float2*>(p.part_ml + (slot_o * part_rows + r) * 2) = make_float2(m[mt][e], sum);
          }
        }
      if (!whole) {
        // ---- join: the last of the segment's CTAs to arrive adds the parts
        // up in the order of the CTAs
        const int64_t c0 = ((d.seg_start + 1) * ctas - 1) / total;
        const int64_t c1 = ((d.seg_start + d.n_tiles) * ctas - 1) / total;
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const int seen = atomicAdd(p.counters + c0, 1);
          s_last = seen == (int)(c1 - c0);
          if (s_last) p.counters[c0] = 0;
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          const int n = (int)(c1 - c0) + 1;
          // part k of the segment: CTA c0 + k; its second slot when it began with another segment
          const int64_t first_slot = c0 * 2 + (total * c0 / ctas < d.seg_start ? 1 : 0);
          auto slot_of = [&](int k) { return k == 0 ? first_slot : (c0 + k) * 2; };
          for (int r = warp; r < ROWS; r += kWarps) {
            if (d.rt * ROWS + r >= p.R) break;
            float mm = -INFINITY;
            for (int k = lane; k < n; k += 32) mm = fmaxf(mm, __ldcg(p.part_ml + (slot_of(k) * part_rows + r) * 2));
#pragma unroll
            for (int off = 16; off; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
            const float mu = finite_or_zero(mm);
            float sum = 0.f;
            for (int k = lane; k < n; k += 32) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (slot_of(k) * part_rows + r) * 2));
              sum += ml.y * fast_exp2(ml.x - mu);
            }
#pragma unroll
            for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            float acc[D / 32];
#pragma unroll
            for (int x = 0; x < D / 32; ++x) acc[x] = 0.f;
#pragma unroll 8
            for (int k = 0; k < n; ++k) {
              const float w = fast_exp2(__ldcg(p.part_ml + (slot_of(k) * part_rows + r) * 2) - mu);
              const float* src = p.part_o + (slot_of(k) * part_rows + r) * D + lane * (D / 32);
              if constexpr (D == 128) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
                acc[0] += w * f.x; acc[1] += w * f.y; acc[2] += w * f.z; acc[3] += w * f.w;
              } else {
                const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
                acc[0] += w * f.x; acc[1] += w * f.y;
              }
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int R = d.rt * ROWS + r, t = R / p.G, g = R - t * p.G;
            const int64_t row = ((int64_t)d.b * p.HQ + d.h * p.G + g) * p.T + t;
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + row * D + lane * (D / 32));
#pragma unroll
            for (int x = 0; x < D / 64; ++x) dst[x] = pack2<HALF>(acc[2 * x] * inv, acc[2 * x + 1] * inv);
            if (lane == 0) {
              const float lse2 = sum == 0.f ? -INFINITY : mu + log2f(sum);
              if (p.lse) p.lse[row] = lse2 * 0.6931471805599453f;
              if (p.row_lse2) p.row_lse2[(int64_t)(d.b * p.HKV + d.h) * p.R + R] = lse2;
            }
          }
        }
      }
    }
    finish(ahead, slot, (i + S) & (C::DESCS - 1));
  }
  cp_async_wait<0>();
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
  const int64_t tiles = std::max<int64_t>(1, (cap + tile - 1) / tile) * a->batch * a->kv_heads * p.row_tiles;
  p.ctas = (int)std::max<int64_t>(1, std::min<int64_t>(tiles, 2 * num_sms_of(a->num_sms)));
  p.score_stride = std::max<int64_t>(128, (cap + 127) / 128 * 128);
  const size_t rows = (size_t)16 * p.mt * 2 * p.ctas;
  p.part_o = rows * a->head_dim * sizeof(float);
  p.part_ml = rows * 2 * sizeof(float);
  const size_t all_rows = (size_t)a->batch * a->kv_heads * p.R;
  p.lse2 = a->token_weights ? (all_rows * sizeof(float) + 255) / 256 * 256 : 0;
  p.scores = a->token_weights ? all_rows * p.score_stride * sizeof(float) : 0;
  *out = p;
  return KVR_OK;
}

template <bool HALF, int D, int MT>
static int launch(const Params& p, cudaStream_t s) {
  using C = Cfg<D, MT>;
  auto kern = attention_kernel<HALF, D, MT>;
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (!ready[dev & 63]) {   // a benign race sets the same value
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
    ready[dev & 63] = true;
  }
  cudaError_t e = pdl_launch(kern, dim3(p.ctas), dim3(kThreads), C::SMEM, s, 1, p);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}

template <bool HALF, int D>
static int launch_mt(int mt, const Params& p, cudaStream_t s) {
  if (mt == 1) return launch<HALF, D, 1>(p, s);
  if (mt == 2) return launch<HALF, D, 2>(p, s);
  return launch<HALF, D, 4>(p, s);
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
  if (counter_count) *counter_count = (size_t)p.ctas;
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
  if (a->head_dim == 64) st = half ? paged::launch_mt<true, 64>(pl.mt, p, s) : paged::launch_mt<false, 64>(pl.mt, p, s);
  else st = half ? paged::launch_mt<true, 128>(pl.mt, p, s) : paged::launch_mt<false, 128>(pl.mt, p, s);
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
