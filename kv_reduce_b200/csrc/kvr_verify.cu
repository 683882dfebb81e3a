// Verification of drafted tokens against the target model's probabilities,
// from given random numbers (sm_100a).  No reference counterpart: the
// reference compares the target's argmax on the host
// (kv_reduce/experiments/packed_review.py:101-137).
//
// p = softmax(target / t), q = softmax(draft / t).  Token x_k is accepted
// while u_k < a_k = min(1, p_k(x_k) / q_k(x_k)); at the first refusal j the
// next token is drawn from max(p_j - q_j, 0), after a full acceptance from
// p_K.  A draw is a race (Gumbel-max in another form): the token with the
// largest weight / e, e the given exponential numbers.  Unlike a search in a
// running sum it needs no normalisation and does not depend on an order of
// summation, so it is one more pass over one row, in any order, with a maximum
// at its end.
//
// What bounds it: the logits' bytes, 2 K rows (up to the first refusal) of
// 2*V bytes and one race row per sequence, with one exponential per logit
// close behind (16 per clock and SM).  Rows are cut into segments, one to a
// warp, and the warps have nothing to do with one another: no barrier holds
// a warp back, so that the loads, the exponentials and the round trips at a
// segment's end of 32 and more warps per SM overlap.  A row pair's last
// segment decides its position.  The segments come position by position, and
// in a large batch one whose sequence is already refused earlier is left
// unread: that changes the work, never the result, since no row behind the
// first refusal is used.
//
// Measured (bf16): 64 sequences of 5 drafted tokens over 128000 entries, each
// accepted with probability 0.75, 137 MB that count, 47 us; greedy, 4 of 4
// over 32000, 0.8 MB, 6.6 us of device time, all of it round trips.
#include "kvr_common.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace kvr {
namespace verify {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;      // blocks a lane has in hand, and as many on their way

struct Params {
  const void* target;
  int64_t t_b, t_k;
  const void* draft;
  int64_t d_b, d_k;
  const int64_t* tokens;
  int64_t tok_b;
  const float* uniforms;
  int64_t u_b;
  const float* noise;
  int64_t n_b;
  const int* draft_lengths;
  int64_t* out_tokens;
  int* accepted;
  float* accept_prob;
  int B, K, V;
  int segments, seg_blocks;            // of a row in the first pass: how many, and blocks of 16 bytes in one
  int race_segments, race_blocks;
  float c;                 // log2(e) / temperature
  bool skip;               // look for earlier refusals before reading
  // zero on entry and on exit
  unsigned long long* best;   // greedy [B, K + 1], else [B]
  int* arrived;               // [B, K + 1]
  int* done;                  // [B]
  int* refused;               // [B]: K + 1 - (first refused position), 0 while none is known
  // scratch
  float2* part;               // [B, K, 2, segments]: (max, sum) of the target's and the draft's segments
  float4* stats;              // [B, K]: the same of the rows, target then draft
  int4* raced;                // [B, race_segments]: the segments' winners (Racer) where the race is over the target alone
};

__device__ __forceinline__ float zero_if_none(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[8]) {
    f[0] = bf16lo(w.x); f[1] = bf16hi(w.x); f[2] = bf16lo(w.y); f[3] = bf16hi(w.y);
    f[4] = bf16lo(w.z); f[5] = bf16hi(w.z); f[6] = bf16lo(w.w); f[7] = bf16hi(w.w);
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {   // of two pairs; a NaN gives way
    asm("max.bf16x2 %0, %0, %1;\n" : "+r"(a) : "r"(b));
    return a;
  }
  static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(bf16lo(w), bf16hi(w)); }
  static constexpr uint32_t kLowest = 0xff80ff80u;   // -inf, -inf
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    asm("max.f16x2 %0, %0, %1;\n" : "+r"(a) : "r"(b));
    return a;
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return fmaxf(v.x, v.y);
  }
  static constexpr uint32_t kLowest = 0xfc00fc00u;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static constexpr uint32_t kLowest = 0xff800000u;
};

// Rows start anywhere (an odd vocabulary), 16-byte loads do not.  Block g is
// elements [g*N, g*N + N) whatever the alignment, so that sums and draws do
// not depend on it: a block that lies across two 16-byte granules is put
// together from both, and one at the row's end element by element, with -inf
// (no weight) behind the end.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* p;
  int shift;   // bytes the row starts behind a 16-byte boundary
  __device__ __forceinline__ explicit Row(const T* row) : p(row), shift((int)(reinterpret_cast<uintptr_t>(row) & 15)) {}
  __device__ __forceinline__ uint4 load(int g, int V) const {
    const int e = g * N, s = shift / (int)sizeof(T);
    if (shift == 0 && e + N <= V) return __ldg(reinterpret_cast<const uint4*>(p + e));
    if (shift != 0 && e >= s && e - s + 2 * N <= V) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p + e - s));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(p + e - s + N));
      uint32_t x0 = a.x, x1 = a.y, x2 = a.z, x3 = a.w, x4 = b.x, x5 = b.y, x6 = b.z, x7 = b.w;
      if (shift & 8) { x0 = x2; x1 = x3; x2 = x4; x3 = x5; x4 = x6; x5 = x7; }
      if (shift & 4) { x0 = x1; x1 = x2; x2 = x3; x3 = x4; x4 = x5; }
      const int bits = (shift & 2) * 8;
      return make_uint4(__funnelshift_r(x0, x1, bits), __funnelshift_r(x1, x2, bits), __funnelshift_r(x2, x3, bits),
                        __funnelshift_r(x3, x4, bits));
    }
    union {
      uint4 w;
      T t[N];
    } u;
    u.w = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
    for (int i = 0; i < N; ++i)
      if (e + i < V) u.t[i] = p[e + i];
    return u.w;
  }
};
template <typename T>
__device__ __forceinline__ int blocks_of(int V) { return (V + Vec<T>::N - 1) / Vec<T>::N; }

// 2^((x - m) c): x - m is exact or nearly so, the product the one rounding,
// and the largest gives 1 whatever c is.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float c) {
  const float mm = fmaxf(m, m2), mu = zero_if_none(mm);
  s = s * fast_exp2((m - mu) * c) + s2 * fast_exp2((m2 - mu) * c);
  m = mm;
}
// The same over the warp's lanes, one exponential a lane.
__device__ __forceinline__ void lanes_merge(float& m, float& s, float c) {
  float mm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
  s *= fast_exp2((m - zero_if_none(mm)) * c);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  m = mm;
}

// Two fp32 operations to an instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void halves(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Takes UN blocks into a running (max, sum of 2^((x - max) c)).
template <typename T, int UN>
__device__ __forceinline__ void take(const uint4 (&w)[UN], float c, float& m, float& s) {
  uint32_t top = Vec<T>::kLowest;
#pragma unroll
  for (int i = 0; i < UN; ++i)
    top = Vec<T>::max2(top, Vec<T>::max2(Vec<T>::max2(w[i].x, w[i].y), Vec<T>::max2(w[i].z, w[i].w)));
  const float mm = fmaxf(m, Vec<T>::top(top)), mu = zero_if_none(mm);
  const uint64_t mu2 = pair(-mu, -mu), c2 = pair(c, c);
  uint64_t sum[2] = {pair(s * fast_exp2((m - mu) * c), 0.f), pair(0.f, 0.f)};
  m = mm;
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    float f[Vec<T>::N];
    Vec<T>::get(w[i], f);
#pragma unroll
    for (int j = 0; j < Vec<T>::N; j += 2) {
      float a, b;
      halves(mul2(add2(pair(f[j], f[j + 1]), mu2), c2), a, b);
      sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], pair(fast_exp2(a), fast_exp2(b)));
    }
  }
  float a, b;
  halves(add2(sum[0], sum[1]), a, b);
  s = a + b;
}

__device__ __forceinline__ int drafted(const Params& p, int b) {
  return p.draft_lengths ? min(max(p.draft_lengths[b], 0), p.K) : p.K;
}
__device__ __forceinline__ int refused_at(const Params& p, int b) {   // K + 1: nowhere so far
  return p.K + 1 - *reinterpret_cast<volatile int*>(p.refused + b);
}

// Larger is better; equal weights: the lowest index.
__device__ __forceinline__ unsigned long long race_key(float score, int index) {
  uint32_t u = __float_as_uint(score + 0.f);
  u = (u >> 31) ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ int64_t race_index(unsigned long long key) {
  return key == 0 ? -1 : (int64_t)(0xffffffffu - (uint32_t)key);
}
__device__ __forceinline__ unsigned long long lanes_best(unsigned long long best) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(~0u, best, o);
    best = x > best ? x : best;
  }
  return best;
}

// One segment of a row through `use(blocks in hand, first block)`, the next
// blocks on their way.  Lane l has blocks first + 32 i + l.
template <typename T, typename Use>
__device__ __forceinline__ void stream(const Row<T>& row, int begin, int end, int V, Use use) {
  const int lane = threadIdx.x & 31;
  const uint4 none = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
  uint4 w[kUnroll], next[kUnroll];
  auto load = [&](int g, uint4 (&x)[kUnroll]) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) x[i] = g + 32 * i + lane < end ? row.load(g + 32 * i + lane, V) : none;
  };
  load(begin, w);
  for (int g = begin; g < end; g += 32 * kUnroll) {
    if (g + 32 * kUnroll < end) load(g + 32 * kUnroll, next);
    use(w, g);
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) w[i] = next[i];
  }
}

// Rows in the order of their positions: (k, b, target | draft, segment).
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) stats_kernel(const __grid_constant__ Params p) {
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int seg = unit % p.segments, row = unit / p.segments;   // row = (k * B + b) * 2 + (draft)
  const int side = row & 1, k = (row >> 1) / p.B, b = (row >> 1) - k * p.B;
  if (k >= p.K) return;
  pdl_enter();
  const int n_draft = drafted(p, b);
  if (k >= n_draft) return;
  if (p.skip && k > 0 && refused_at(p, b) < k) return;   // an earlier position of this sequence is refused already
  const T* trow = static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)k * p.t_k;
  const T* drow = static_cast<const T*>(p.draft) + (int64_t)b * p.d_b + (int64_t)k * p.d_k;
  float m = -INFINITY, s = 0.f;
  const int begin = seg * p.seg_blocks, end = min(begin + p.seg_blocks, blocks_of<T>(p.V));
  stream<T>(Row<T>(side ? drow : trow), begin, end, p.V,
            [&](const uint4(&w)[kUnroll], int) { take<T, kUnroll>(w, p.c, m, s); });
  lanes_merge(m, s, p.c);
  const int at = b * p.K + k;
  float2* part = p.part + (int64_t)at * 2 * p.segments;   // [2][segments]
  int last = 0;
  if (lane == 0) {
    part[side * p.segments + seg] = make_float2(m, s);
    __threadfence();
    last = atomicAdd(p.arrived + b * (p.K + 1) + k, 1) == 2 * p.segments - 1;
    if (last) __threadfence();
  }
  if (!__shfl_sync(~0u, last, 0)) return;
  // ---- the position's last segment: join them in order and decide
  float mt = -INFINITY, st = 0.f, md = -INFINITY, sd = 0.f;
  for (int i = lane; i < p.segments; i += 32) {
    const float2 x = __ldcg(part + i), y = __ldcg(part + p.segments + i);
    merge(mt, st, x.x, x.y, p.c);
    merge(md, sd, y.x, y.y, p.c);
  }
  lanes_merge(mt, st, p.c);
  lanes_merge(md, sd, p.c);
  if (lane == 0) {
    p.stats[at] = make_float4(mt, st, md, sd);
    const int64_t x = p.tokens[(int64_t)b * p.tok_b + k];
    float a = 0.f;   // a token outside the vocabulary is refused
    if (x >= 0 && x < p.V) {
      const float lt = Vec<T>::one(trow + x), ld = Vec<T>::one(drow + x);
      const float r = exp2f(((lt - zero_if_none(mt)) - (ld - zero_if_none(md))) * p.c) * (sd / st);
      a = r >= 1.f ? 1.f : r > 0.f ? r : 0.f;   // 0 / 0: not in the target's support
    }
    p.accept_prob[at] = a;
    if (!(p.uniforms[(int64_t)b * p.u_b + k] < a)) atomicMax(p.refused + b, p.K + 1 - k);
  }
}

// The sequence's outputs, and its zeros for the next call, by one warp.
// `drafted_token`: tokens[lane], read ahead (the first 32).
__device__ __forceinline__ void write_out(const Params& p, int b, int n_draft, int at, int64_t token,
                                          int64_t drafted_token, int best_rows) {
  const int lane = threadIdx.x & 31;
  for (int k = lane; k <= p.K; k += 32) {
    const int64_t old = k == lane ? drafted_token : k < at ? p.tokens[(int64_t)b * p.tok_b + k] : -1;
    p.out_tokens[(int64_t)b * (p.K + 1) + k] = k < at ? old : k == at ? token : -1;
    if (k < p.K && (k > at || k >= n_draft)) p.accept_prob[b * p.K + k] = 0.f;
    p.arrived[b * (p.K + 1) + k] = 0;
    if (k < best_rows) p.best[(int64_t)b * best_rows + k] = 0;
  }
  if (lane == 0) {
    p.accepted[b] = at;
    p.done[b] = 0;
    p.refused[b] = 0;
  }
}
__device__ __forceinline__ int64_t token_ahead(const Params& p, int b) {
  const int lane = threadIdx.x & 31;
  return lane < p.K ? p.tokens[(int64_t)b * p.tok_b + lane] : -1;
}

// The noise of a block of N elements.
template <int N>
__device__ __forceinline__ void load_noise(const float* p, int e, int V, float (&f)[N]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && e + N <= V) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(p + e + i));
      f[i] = x.x; f[i + 1] = x.y; f[i + 2] = x.z; f[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = e + i < V ? __ldg(p + e + i) : 1.f;
  }
}

// The best entry so far of a race over the target alone.  Weight / e of two
// entries compares as (x - y) c with log2 e_x - log2 e_y: the row's maximum and
// sum, which nothing has computed for this row, are not needed.  Only the
// difference is scaled: x c by itself overflows for small temperatures and for
// masks of the type's lowest value, and loses the bits that decide between
// equal logits.
struct Racer {
  float x = -INFINITY, l = 0.f;   // logit, log2 of its exponential number
  int at = -1;
  __device__ __forceinline__ void take(float f, float le, int i, float c) {   // in rising order of i
    if ((f - x) * c > le - l) {   // (-inf, no weight, and NaN never are; anything else beats the initial -inf)
      x = f;
      l = le;
      at = i;
    }
  }
  __device__ __forceinline__ void merge(const Racer& o, float c) {   // the same winner whichever is merged into which
    if (o.at < 0) return;
    const float d = (o.x - x) * c, t = o.l - l;
    if (at < 0 || d > t || (!(d < t) && o.at < at)) *this = o;
  }
};
__device__ __forceinline__ Racer lanes_race(Racer r, float c) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Racer other;
    other.x = __shfl_xor_sync(~0u, r.x, o);
    other.l = __shfl_xor_sync(~0u, r.l, o);
    other.at = __shfl_xor_sync(~0u, r.at, o);
    r.merge(other, c);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void race_target(const uint4& w, const float (&e)[Vec<T>::N], float c, int at, Racer& r) {
  float f[Vec<T>::N];
  Vec<T>::get(w, f);
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) r.take(f[j], __log2f(e[j]), at + j, c);
}

constexpr int kRaceUnroll = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads, 8) race_kernel(const __grid_constant__ Params p) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * kWarps + (threadIdx.x >> 5), b = unit / p.race_segments;
  if (b >= p.B) return;
  const int begin = (unit - b * p.race_segments) * p.race_blocks, end = min(begin + p.race_blocks, blocks_of<T>(p.V));
  pdl_enter();
  const int n_draft = drafted(p, b), at = min(refused_at(p, b), n_draft);
  const bool residual = at < n_draft;
  const float* noise = p.noise + (int64_t)b * p.n_b;
  const Row<T> rt(static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)at * p.t_k);
  float mt = 0.f, md = 0.f, it = 0.f, id = 0.f, top = 0.f;
  int where = -1;
  Racer racer;
  if (residual) {
    const Row<T> rd(static_cast<const T*>(p.draft) + (int64_t)b * p.d_b + (int64_t)at * p.d_k);
    const float4 st = p.stats[b * p.K + at];
    mt = zero_if_none(st.x);
    md = zero_if_none(st.z);
    it = st.y > 0.f ? 1.f / st.y : 0.f;
    id = st.w > 0.f ? 1.f / st.w : 0.f;
#pragma unroll kRaceUnroll
    for (int g = begin + lane; g < end; g += 32) {
      float f[N], d[N], e[N];
      Vec<T>::get(rt.load(g, p.V), f);
      Vec<T>::get(rd.load(g, p.V), d);
      load_noise(noise, g * N, p.V, e);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        // (each product rounded: contracted into one fused operation, equal p and q would leave a rounding error)
        const float x = __fsub_rn(__fmul_rn(fast_exp2((f[j] - mt) * p.c), it), __fmul_rn(fast_exp2((d[j] - md) * p.c), id));
        const float score = __fdividef(x, e[j]);
        if (score > top) {
          top = score;
          where = g * N + j;
        }
      }
    }
  } else {
#pragma unroll kRaceUnroll
    for (int g = begin + lane; g < end; g += 32) {
      float e[N];
      const uint4 w = rt.load(g, p.V);
      load_noise(noise, g * N, p.V, e);
      race_target<T>(w, e, p.c, g * N, racer);
    }
  }
  unsigned long long best = 0;
  if (residual) best = lanes_best(where < 0 ? 0ull : race_key(top, where));
  else racer = lanes_race(racer, p.c);
  const int64_t ahead = token_ahead(p, b);
  int4* raced = p.raced + (int64_t)b * p.race_segments;
  int last = 0;
  if (lane == 0) {
    if (best) atomicMax(p.best + b, best);
    if (!residual)
      raced[unit - b * p.race_segments] = make_int4(__float_as_int(racer.x), __float_as_int(racer.l), racer.at, 0);
    __threadfence();
    last = atomicAdd(p.done + b, 1) == p.race_segments - 1;
    if (last) __threadfence();
  }
  if (!__shfl_sync(~0u, last, 0)) return;
  int64_t token = -1;
  if (residual) token = race_index(*reinterpret_cast<volatile unsigned long long*>(p.best + b));
  if (token < 0) {
    racer = Racer();
    if (residual) {   // p = q up to rounding leaves nothing to draw from: draw from p
      for (int g = lane; g < blocks_of<T>(p.V); g += 32) {
        float e[N];
        const uint4 w = rt.load(g, p.V);
        load_noise(noise, g * N, p.V, e);
        race_target<T>(w, e, p.c, g * N, racer);
      }
    } else {   // the segments' winners, in order
      for (int i = lane; i < p.race_segments; i += 32) {
        const int4 x = __ldcg(raced + i);
        Racer other;
        other.x = __int_as_float(x.x);
        other.l = __int_as_float(x.y);
        other.at = x.z;
        racer.merge(other, p.c);
      }
    }
    token = lanes_race(racer, p.c).at;
  }
  write_out(p, b, n_draft, at, token, ahead, 1);
}

// t = 0: x_k is accepted while it is the argmax of target_k (the lowest index
// of the largest logit; NaN is never the largest).  A CTA's warps take
// neighbouring segments of a row and count as one: with a maximum in place of
// the exponentials the warps are done together, and the counts are what takes
// time in a small batch.
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) greedy_kernel(const __grid_constant__ Params p) {
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 31;
  const int chunks = (p.segments + kWarps - 1) / kWarps;   // CTAs of a row
  const int row = blockIdx.x / chunks, k = row / p.B, b = row - k * p.B;
  const int seg = (blockIdx.x - row * chunks) * kWarps + (threadIdx.x >> 5);
  __shared__ unsigned long long buf[kWarps];
  __shared__ int s_unread;
  pdl_enter();
  const int n_draft = drafted(p, b);
  bool unread = k > n_draft;
  if (p.skip && k > 0) {   // one look for the whole CTA
    if (threadIdx.x == 0) s_unread = refused_at(p, b) < k;
    __syncthreads();
    unread |= s_unread != 0;
  }
  unsigned long long best = 0;
  if (!unread) {
    float top = -INFINITY;
    int where = -1;
    const int begin = seg * p.seg_blocks, end = min(begin + p.seg_blocks, blocks_of<T>(p.V));
    stream<T>(Row<T>(static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)k * p.t_k), begin, end, p.V,
              [&](const uint4(&w)[kUnroll], int g) {
#pragma unroll
                for (int i = 0; i < kUnroll; ++i) {
                  // most blocks hold nothing new: their largest pair tells
                  const uint32_t high = Vec<T>::max2(Vec<T>::max2(w[i].x, w[i].y), Vec<T>::max2(w[i].z, w[i].w));
                  if (!(Vec<T>::top(high) > top || where < 0)) continue;
                  float f[N];
                  Vec<T>::get(w[i], f);
                  const int e = (g + 32 * i + lane) * N;
#pragma unroll
                  for (int j = 0; j < N; ++j)
                    if (f[j] > top || (where < 0 && f[j] == top && e + j < p.V)) {
                      top = f[j];
                      where = e + j;
                    }
                }
              });
    best = lanes_best(where < 0 ? 0ull : race_key(top, where));
  }
  if (lane == 0) buf[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int64_t ahead = token_ahead(p, b);
  int last = 0;
  if (lane == 0) {
#pragma unroll
    for (int w = 1; w < kWarps; ++w) best = buf[w] > best ? buf[w] : best;
    unsigned long long* slot = p.best + (int64_t)b * (p.K + 1) + k;
    if (best) atomicMax(slot, best);
    __threadfence();
    if (p.skip && !unread && k < n_draft && atomicAdd(p.arrived + b * (p.K + 1) + k, 1) == chunks - 1) {
      __threadfence();
      if (race_index(*reinterpret_cast<volatile unsigned long long*>(slot)) != p.tokens[(int64_t)b * p.tok_b + k])
        atomicMax(p.refused + b, p.K + 1 - k);
      __threadfence();
    }
    last = atomicAdd(p.done + b, 1) == (p.K + 1) * chunks - 1;
    if (last) __threadfence();
  }
  if (!__shfl_sync(~0u, last, 0)) return;
  // the sequence's last CTA: the first token that is not its row's argmax (rows behind it may be unread)
  const volatile unsigned long long* rows = p.best + (int64_t)b * (p.K + 1);
  const unsigned long long mine = lane <= n_draft ? rows[lane] : 0ull;
  int at = n_draft;
  for (int i = lane; i < n_draft; i += 32) {
    const int64_t x = race_index(i == lane ? mine : rows[i]);
    if (x < 0 || x != (i == lane ? ahead : p.tokens[(int64_t)b * p.tok_b + i])) at = min(at, i);
  }
  at = __reduce_min_sync(~0u, at);
  for (int i = lane; i < at; i += 32) p.accept_prob[b * p.K + i] = 1.f;
  if (lane == 0 && at < n_draft) p.accept_prob[b * p.K + at] = 0.f;
  const unsigned long long here = __shfl_sync(~0u, mine, at & 31);
  const int64_t token = race_index(at < 32 ? here : rows[at]);
  __syncwarp();
  write_out(p, b, n_draft, at, token, ahead, p.K + 1);
}

// ------------------------------------------------------------------- host
struct Plan {
  int segments, seg_blocks, race_segments, race_blocks;
  bool skip;
  size_t zeroed, scratch;
};

static int plan_of(const kvr_verify_args* a, Plan* out) {
  if (!a || a->batch < 0 || a->draft_tokens < 0 || a->vocab <= 0 || !(a->temperature >= 0.f) ||
      !std::isfinite(a->temperature))
    return KVR_ERR_INVALID_ARGUMENT;
  if (a->dtype < 0 || a->dtype > 2) return KVR_ERR_UNSUPPORTED;
  if (a->temperature > 0.f && a->temperature < FLT_MIN) return KVR_ERR_UNSUPPORTED;   // its reciprocal may overflow
  if (a->vocab > (1 << 30) || a->draft_tokens > 4095 || (int64_t)a->batch * (a->draft_tokens + 1) > (1 << 24))
    return KVR_ERR_UNSUPPORTED;
  const int n = a->dtype == 2 ? 4 : 8;
  const int64_t blocks = (a->vocab + n - 1) / n;
  const bool greedy = a->temperature == 0.f;
  const int64_t rows = std::max<int64_t>(1, (int64_t)a->batch * (greedy ? a->draft_tokens + 1 : 2 * a->draft_tokens));
  Plan p;
  // A warp's segment: at most 4 steps of kUnroll blocks a lane (longer ones are under way when their sequence is
  // refused, shorter ones spend more of their time on the count: 64 x 5 of 128K took 51, 48, 45.5, 46, 52 us with 2,
  // 3, 4, 8, 16), fewer while they leave warps out (32 on each of 148 SMs).
  p.seg_blocks = 4 * 32 * kUnroll;
  while (p.seg_blocks > 32 * kUnroll && rows * ((blocks + p.seg_blocks - 1) / p.seg_blocks) < 148 * 32) p.seg_blocks /= 2;
  p.segments = (int)((blocks + p.seg_blocks - 1) / p.seg_blocks);
  // the race: 8 blocks a lane (2, 4, 16, 32 took 7, 2, 4 and 16 us longer on the same), fewer while that leaves
  // half of the warps out
  p.race_blocks = 8 * 32;
  while (p.race_blocks > 32 * kRaceUnroll &&
         (int64_t)a->batch * ((blocks + p.race_blocks - 1) / p.race_blocks) < 148 * 16)
    p.race_blocks /= 2;
  p.race_segments = (int)((blocks + p.race_blocks - 1) / p.race_blocks);
  if (rows * p.segments > (1ll << 31) - 1 || (int64_t)a->batch * p.race_segments > (1ll << 31) - 1)
    return KVR_ERR_UNSUPPORTED;
  // Looking for an earlier refusal costs every warp a round trip to L2 and saves reading: not for logits that
  // 5 us read anyway.
  p.skip = rows * a->vocab * (a->dtype == 2 ? 4 : 2) > (32 << 20);
  const size_t B = a->batch, K1 = a->draft_tokens + 1;
  p.zeroed = B * K1 * 8 + B * K1 * 4 + 2 * B * 4;
  p.scratch = greedy ? 0
                     : B * p.race_segments * sizeof(int4) +
                           B * (K1 - 1) * (sizeof(float4) + 2 * (size_t)p.segments * sizeof(float2));
  *out = p;
  return KVR_OK;
}

template <typename T>
static cudaError_t launch(const Params& p, bool greedy, cudaStream_t s) {
  auto grid = [](int64_t warps) { return dim3((unsigned)((warps + kWarps - 1) / kWarps)); };
  if (greedy)
    return pdl_launch(greedy_kernel<T>, dim3((unsigned)((int64_t)p.B * (p.K + 1) * ((p.segments + kWarps - 1) / kWarps))),
                      dim3(kThreads), 0, s, 1, p);
  if (p.K > 0) {
    const cudaError_t e = pdl_launch(stats_kernel<T>, grid(2ll * p.B * p.K * p.segments), dim3(kThreads), 0, s, 1, p);
    if (e != cudaSuccess) return e;
  }
  return pdl_launch(race_kernel<T>, grid((int64_t)p.B * p.race_segments), dim3(kThreads), 0, s, 1, p);
}

}  // namespace verify
}  // namespace kvr

using namespace kvr;

extern "C" int kvr_verify_plan(const kvr_verify_args* a, size_t* zeroed_bytes, size_t* workspace_bytes) {
  verify::Plan p;
  const int st = verify::plan_of(a, &p);
  if (st != KVR_OK) return st;
  if (zeroed_bytes) *zeroed_bytes = p.zeroed;
  if (workspace_bytes) *workspace_bytes = p.scratch;
  return KVR_OK;
}

extern "C" int kvr_verify(const kvr_verify_args* a, kvr_stream_t stream) {
  verify::Plan pl;
  const int st = verify::plan_of(a, &pl);
  if (st != KVR_OK) return st;
  if (a->batch == 0) return KVR_OK;
  const bool greedy = a->temperature == 0.f;
  const int K = a->draft_tokens;
  if (!a->target || !a->out_tokens || !a->accepted || (K > 0 && (!a->tokens || !a->accept_prob))) return KVR_ERR_INVALID_ARGUMENT;
  if (!greedy && (!a->noise || (K > 0 && (!a->draft || !a->uniforms)))) return KVR_ERR_INVALID_ARGUMENT;
  if (!a->zeroed || a->zeroed_bytes < pl.zeroed || (pl.scratch > 0 && (!a->workspace || a->workspace_bytes < pl.scratch)))
    return KVR_ERR_WORKSPACE;
  if (!aligned16(a->zeroed) || !aligned16(a->workspace)) return KVR_ERR_MISALIGNED;
  verify::Params p;
  p.target = a->target; p.t_b = a->target_b_stride; p.t_k = a->target_k_stride;
  p.draft = a->draft; p.d_b = a->draft_b_stride; p.d_k = a->draft_k_stride;
  p.tokens = a->tokens; p.tok_b = a->tokens_b_stride;
  p.uniforms = a->uniforms; p.u_b = a->uniforms_b_stride;
  p.noise = a->noise; p.n_b = a->noise_b_stride;
  p.draft_lengths = a->draft_lengths;
  p.out_tokens = a->out_tokens; p.accepted = a->accepted; p.accept_prob = a->accept_prob;
  p.B = a->batch; p.K = K; p.V = a->vocab; 
  p.segments = pl.segments; p.seg_blocks = pl.seg_blocks;
  p.race_segments = pl.race_segments; p.race_blocks = pl.race_blocks;
  p.skip = pl.skip;
  p.c = greedy ? 1.f : 1.4426950408889634f / a->temperature;
  const size_t rows = (size_t)p.B * (K + 1);
  p.best = static_cast<unsigned long long*>(a->zeroed);
  p.arrived = reinterpret_cast<int*>(p.best + rows);
  p.done = p.arrived + rows;
  p.refused = p.done + p.B;
  p.raced = static_cast<int4*>(a->workspace);
  p.stats = reinterpret_cast<float4*>(p.raced + (greedy ? 0 : (size_t)p.B * p.race_segments));
  p.part = reinterpret_cast<float2*>(p.stats + (size_t)p.B * K);
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = a->dtype == 0   ? verify::launch<__nv_bfloat16>(p, greedy, s)
                        : a->dtype == 1 ? verify::launch<__half>(p, greedy, s)
                                        : verify::launch<float>(p, greedy, s);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}
