// Verification of drafted tokens against the target model's probabilities,
// from given random numbers (sm_100a).  No reference counterpart: the
// reference compares the target's argmax on the host
// (kv_reduce/experiments/packed_review.py:101-137).
//
// p = softmax(target / t), q = softmax(draft / t).  Token x_k is accepted
// while u_k < a_k = min(1, p_k(x_k) / q_k(x_k)); at the first refusal j the
// next token is drawn from max(p_j - q_j, 0), after a full acceptance from
// p_K.  A draw is a race: the token with the largest weight / e, e the given
// exponential numbers.  Unlike a search in a running sum it needs no
// normalisation and does not depend on an order of summation, so it is one
// more pass over one row, in any order, with a maximum at its end.
//
// What bounds it: the logits' bytes, 2 K rows (up to the first refusal) of
// 2*V bytes and one race row per sequence, with one exponential per logit
// close behind (16 per clock and SM).  Every row is cut into chunks, a CTA
// takes the same chunk of p_k and q_k and keeps it in registers: one read for
// maximum and sum.  CTAs run through the positions in order, and in a large
// batch one that finds its sequence already refused earlier leaves its rows
// unread: that changes the work, never the result, since no row behind the
// first refusal is used.
#include "kvr_common.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace kvr {
namespace verify {

constexpr int kThreads = 256;

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
  int B, K, V, chunks;     // chunks of a row in the first pass
  int race_chunks;
  float c;                 // log2(e) / temperature
  bool skip;               // look for earlier refusals before reading
  // zero on entry and on exit
  unsigned long long* best;   // greedy [B, K + 1], else [B]
  int* arrived;               // [B, K + 1]
  int* done;                  // [B]
  int* refused;               // [B]: K + 1 - (first refused position), 0 while none is known
  // scratch
  float4* part;               // [B, K, chunks]: (max * c, sum) of the target's and the draft's chunk
  float4* stats;              // [B, K]: the same of the rows
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

// Maxima are kept times c, rounded once: m in 2^(x c - m) is one number for
// the whole row and its rounding falls out of every ratio.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float mm = fmaxf(m, m2), mu = zero_if_none(mm);
  s = s * fast_exp2(m - mu) + s2 * fast_exp2(m2 - mu);
  m = mm;
}

// (max c, sum of 2^(x c - max c)) of the thread's UN blocks
template <typename T, int UN>
__device__ __forceinline__ void chunk_stats(const uint4 (&w)[UN], float c, float& m, float& s) {
  uint32_t top = Vec<T>::kLowest;
#pragma unroll
  for (int i = 0; i < UN; ++i)
    top = Vec<T>::max2(top, Vec<T>::max2(Vec<T>::max2(w[i].x, w[i].y), Vec<T>::max2(w[i].z, w[i].w)));
  m = Vec<T>::top(top) * c;
  const float mu = zero_if_none(m);
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < UN; ++i) {
    float f[Vec<T>::N];
    Vec<T>::get(w[i], f);
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) part[j & 3] += fast_exp2(__fmaf_rn(f[j], c, -mu));
  }
  s = (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ void warp_merge(float& m, float& s, float2* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) merge(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o));
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(m, s);
}

__device__ __forceinline__ int drafted(const Params& p, int b) {
  return p.draft_lengths ? min(max(p.draft_lengths[b], 0), p.K) : p.K;
}
__device__ __forceinline__ int refused_at(const Params& p, int b) {   // K + 1: nowhere so far
  return p.K + 1 - *reinterpret_cast<volatile int*>(p.refused + b);
}

template <typename T, int UN>
__global__ void __launch_bounds__(kThreads) stats_kernel(const __grid_constant__ Params p) {
  __shared__ float2 buf[2][kThreads / 32];
  __shared__ int s_flag;
  pdl_wait();
  const int per_k = p.B * p.chunks;
  const int k = blockIdx.x / per_k, b = (blockIdx.x - k * per_k) / p.chunks, ch = blockIdx.x % p.chunks;
  const int n_draft = drafted(p, b);
  if (k >= n_draft) return;
  if (p.skip && k > 0) {
    if (threadIdx.x == 0) s_flag = refused_at(p, b) < k;
    __syncthreads();
    if (s_flag) return;   // an earlier position of this sequence is refused already
  }
  const T* trow = static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)k * p.t_k;
  const T* drow = static_cast<const T*>(p.draft) + (int64_t)b * p.d_b + (int64_t)k * p.d_k;
  const Row<T> rt(trow), rd(drow);
  const int g0 = ch * UN * kThreads + threadIdx.x, blocks = blocks_of<T>(p.V);
  uint4 wt[UN], wd[UN];
  const uint4 none = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
#pragma unroll
  for (int i = 0; i < UN; ++i) wt[i] = g0 + i * kThreads < blocks ? rt.load(g0 + i * kThreads, p.V) : none;
#pragma unroll
  for (int i = 0; i < UN; ++i) wd[i] = g0 + i * kThreads < blocks ? rd.load(g0 + i * kThreads, p.V) : none;
  float mt, st, md, sd;
  chunk_stats<T, UN>(wt, p.c, mt, st);
  chunk_stats<T, UN>(wd, p.c, md, sd);
  warp_merge(mt, st, buf[0]);
  warp_merge(md, sd, buf[1]);
  __syncthreads();
  const int row = b * p.K + k;
  if (threadIdx.x == 0) {
    mt = buf[0][0].x; st = buf[0][0].y; md = buf[1][0].x; sd = buf[1][0].y;
    for (int w = 1; w < kThreads / 32; ++w) {
      merge(mt, st, buf[0][w].x, buf[0][w].y);
      merge(md, sd, buf[1][w].x, buf[1][w].y);
    }
    p.part[(int64_t)row * p.chunks + ch] = make_float4(mt, st, md, sd);
    __threadfence();
    s_flag = atomicAdd(p.arrived + b * (p.K + 1) + k, 1) == p.chunks - 1;
  }
  __syncthreads();
  if (!s_flag || threadIdx.x >= 32) return;
  // ---- the row's last chunk: join them in order and decide
  __threadfence();
  mt = md = -INFINITY;
  st = sd = 0.f;
  for (int i = threadIdx.x; i < p.chunks; i += 32) {
    const float4 q = __ldcg(p.part + (int64_t)row * p.chunks + i);
    merge(mt, st, q.x, q.y);
    merge(md, sd, q.z, q.w);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    merge(mt, st, __shfl_xor_sync(~0u, mt, o), __shfl_xor_sync(~0u, st, o));
    merge(md, sd, __shfl_xor_sync(~0u, md, o), __shfl_xor_sync(~0u, sd, o));
  }
  if (threadIdx.x == 0) {
    p.stats[row] = make_float4(mt, st, md, sd);
    const int64_t x = p.tokens[(int64_t)b * p.tok_b + k];
    float a = 0.f;   // a token outside the vocabulary is refused
    if (x >= 0 && x < p.V) {
      const float lt = Vec<T>::one(trow + x), ld = Vec<T>::one(drow + x);
      const float r = exp2f(__fmaf_rn(lt, p.c, -zero_if_none(mt)) - __fmaf_rn(ld, p.c, -zero_if_none(md))) * (sd / st);
      a = r >= 1.f ? 1.f : r > 0.f ? r : 0.f;   // 0 / 0: not in the target's support
    }
    p.accept_prob[row] = a;
    if (!(p.uniforms[(int64_t)b * p.u_b + k] < a)) atomicMax(p.refused + b, p.K + 1 - k);
  }
}

// Larger is better; equal weights: the lowest index.
__device__ __forceinline__ unsigned long long race_key(float score, int index) {
  uint32_t u = __float_as_uint(score + 0.f);
  u = (u >> 31) ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ unsigned long long block_best(unsigned long long best, unsigned long long* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(~0u, best, o);
    best = x > best ? x : best;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) best = buf[w] > best ? buf[w] : best;
  return best;
}

// The sequence's outputs, and its zeros for the next call.
__device__ __forceinline__ void write_out(const Params& p, int b, int at, int64_t token, int best_rows) {
  for (int k = threadIdx.x; k <= p.K; k += kThreads) {
    p.out_tokens[(int64_t)b * (p.K + 1) + k] =
        k < at ? p.tokens[(int64_t)b * p.tok_b + k] : k == at ? token : -1;
    if (k < p.K && (k > at || k >= drafted(p, b))) p.accept_prob[b * p.K + k] = 0.f;
    p.arrived[b * (p.K + 1) + k] = 0;
    if (k < best_rows) p.best[(int64_t)b * best_rows + k] = 0;
  }
  if (threadIdx.x == 0) {
    p.accepted[b] = at;
    p.done[b] = 0;
    p.refused[b] = 0;
  }
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

// weight / e over one block, in logarithms: x c - log2 e has the same order
// and needs neither the row's maximum nor its sum.
template <typename T>
__device__ __forceinline__ void race_target(const uint4& w, const float (&e)[Vec<T>::N], float c, int at, float& top,
                                            int& where) {
  float f[Vec<T>::N];
  Vec<T>::get(w, f);
#pragma unroll
  for (int j = 0; j < Vec<T>::N; ++j) {
    const float key = f[j] * c - __log2f(e[j]);
    if (key > top) {
      top = key;
      where = at + j;
    }
  }
}

constexpr int kRaceBlocks = 2;   // blocks of a thread: all its loads are issued at once

template <typename T>
__global__ void __launch_bounds__(kThreads) race_kernel(const __grid_constant__ Params p) {
  __shared__ unsigned long long buf[kThreads / 32];
  __shared__ int s_last;
  pdl_wait();
  const int b = blockIdx.x / p.race_chunks, ch = blockIdx.x % p.race_chunks;
  const int n_draft = drafted(p, b), at = min(refused_at(p, b), n_draft);
  const float* noise = p.noise + (int64_t)b * p.n_b;
  constexpr int N = Vec<T>::N;
  const Row<T> rt(static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)at * p.t_k);
  const int blocks = blocks_of<T>(p.V), g0 = ch * kRaceBlocks * kThreads + threadIdx.x;
  const uint4 none = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
  uint4 wt[kRaceBlocks], wd[kRaceBlocks];
  float e[kRaceBlocks][N];
#pragma unroll
  for (int i = 0; i < kRaceBlocks; ++i) {
    const int g = g0 + i * kThreads;
    wt[i] = g < blocks ? rt.load(g, p.V) : none;
    if (g < blocks) load_noise(noise, g * N, p.V, e[i]);
    else
      for (int j = 0; j < N; ++j) e[i][j] = 1.f;
  }
  float top = -INFINITY;
  int where = -1;
  if (at < n_draft) {
    const Row<T> rd(static_cast<const T*>(p.draft) + (int64_t)b * p.d_b + (int64_t)at * p.d_k);
#pragma unroll
    for (int i = 0; i < kRaceBlocks; ++i) wd[i] = g0 + i * kThreads < blocks ? rd.load(g0 + i * kThreads, p.V) : none;
    const float4 st = p.stats[b * p.K + at];
    const float mt = zero_if_none(st.x), md = zero_if_none(st.z);
    const float it = st.y > 0.f ? 1.f / st.y : 0.f, id = st.w > 0.f ? 1.f / st.w : 0.f;
    top = 0.f;
#pragma unroll
    for (int i = 0; i < kRaceBlocks; ++i) {
      float f[N], d[N];
      Vec<T>::get(wt[i], f);
      Vec<T>::get(wd[i], d);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float w = fast_exp2(__fmaf_rn(f[j], p.c, -mt)) * it - fast_exp2(__fmaf_rn(d[j], p.c, -md)) * id;
        const float score = __fdividef(w, e[i][j]);
        if (score > top) {
          top = score;
          where = (g0 + i * kThreads) * N + j;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRaceBlocks; ++i) race_target<T>(wt[i], e[i], p.c, (g0 + i * kThreads) * N, top, where);
  }
  unsigned long long best = block_best(where < 0 ? 0ull : race_key(top, where), buf);
  if (threadIdx.x == 0) {
    if (best) atomicMax(p.best + b, best);
    __threadfence();
    s_last = atomicAdd(p.done + b, 1) == p.race_chunks - 1;
    if (s_last) __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  best = *reinterpret_cast<volatile unsigned long long*>(p.best + b);
  if (best == 0 && at < n_draft) {   // p = q up to rounding leaves nothing to draw from: draw from p
    top = -INFINITY;
    where = -1;
    for (int g = threadIdx.x; g < blocks; g += kThreads) {
      load_noise(noise, g * N, p.V, e[0]);
      race_target<T>(rt.load(g, p.V), e[0], p.c, g * N, top, where);
    }
    best = block_best(where < 0 ? 0ull : race_key(top, where), buf);
  }
  __syncthreads();
  write_out(p, b, at, best == 0 ? -1 : (int64_t)(0xffffffffu - (uint32_t)best), 1);
}

// t = 0: x_k is accepted while it is the argmax of target_k (the lowest index
// of the largest logit; NaN is never the largest).
template <typename T, int UN>
__global__ void __launch_bounds__(kThreads) greedy_kernel(const __grid_constant__ Params p) {
  __shared__ unsigned long long buf[kThreads / 32];
  __shared__ int s_flag, s_at;
  pdl_wait();
  const int per_k = p.B * p.chunks;
  const int k = blockIdx.x / per_k, b = (blockIdx.x - k * per_k) / p.chunks, ch = blockIdx.x % p.chunks;
  const int n_draft = drafted(p, b);
  bool skip = k > n_draft;
  if (p.skip && k > 0) {
    if (threadIdx.x == 0) s_flag = refused_at(p, b) < k;
    __syncthreads();
    skip |= s_flag != 0;
    __syncthreads();
  }
  unsigned long long best = 0;
  if (!skip) {
    const Row<T> rt(static_cast<const T*>(p.target) + (int64_t)b * p.t_b + (int64_t)k * p.t_k);
    const int g0 = ch * UN * kThreads + threadIdx.x, blocks = blocks_of<T>(p.V);
    uint4 w[UN];
    const uint4 none = make_uint4(Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest, Vec<T>::kLowest);
#pragma unroll
    for (int i = 0; i < UN; ++i) w[i] = g0 + i * kThreads < blocks ? rt.load(g0 + i * kThreads, p.V) : none;
    float top = -INFINITY;
    int where = -1;
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      float f[Vec<T>::N];
      Vec<T>::get(w[i], f);
      const int e = (g0 + i * kThreads) * Vec<T>::N;
#pragma unroll
      for (int j = 0; j < Vec<T>::N; ++j)
        if (e + j < p.V && (f[j] > top || (where < 0 && f[j] == top))) {
          top = f[j];
          where = e + j;
        }
    }
    best = block_best(where < 0 ? 0ull : race_key(top, where), buf);
  }
  if (threadIdx.x == 0) {
    unsigned long long* slot = p.best + (int64_t)b * (p.K + 1) + k;
    if (best) atomicMax(slot, best);
    __threadfence();
    if (p.skip && !skip && k < n_draft && atomicAdd(p.arrived + b * (p.K + 1) + k, 1) == p.chunks - 1) {
      __threadfence();
      const unsigned long long x = *reinterpret_cast<volatile unsigned long long*>(slot);
      if (x == 0 || (int64_t)(0xffffffffu - (uint32_t)x) != p.tokens[(int64_t)b * p.tok_b + k])
        atomicMax(p.refused + b, p.K + 1 - k);
    }
    s_flag = atomicAdd(p.done + b, 1) == (p.K + 1) * p.chunks - 1;
    if (s_flag) __threadfence();
    s_at = n_draft;
  }
  __syncthreads();
  if (!s_flag) return;
  // the sequence's last CTA: the first token that is not its row's argmax (rows behind it may be unread)
  const volatile unsigned long long* rows = p.best + (int64_t)b * (p.K + 1);
  for (int i = threadIdx.x; i < n_draft; i += kThreads) {
    const unsigned long long x = rows[i];
    if (x == 0 || (int64_t)(0xffffffffu - (uint32_t)x) != p.tokens[(int64_t)b * p.tok_b + i]) atomicMin(&s_at, i);
  }
  __syncthreads();
  const int at = s_at;
  for (int i = threadIdx.x; i < at; i += kThreads) p.accept_prob[b * p.K + i] = 1.f;
  if (threadIdx.x == 0 && at < n_draft) p.accept_prob[b * p.K + at] = 0.f;
  const unsigned long long x = rows[at];
  __syncthreads();
  write_out(p, b, at, x == 0 ? -1 : (int64_t)(0xffffffffu - (uint32_t)x), p.K + 1);
}

// ------------------------------------------------------------------- host
struct Plan {
  int un, chunks, race_chunks;
  bool skip;
  size_t zeroed, scratch;
};

static int plan_of(const kvr_verify_args* a, Plan* out) {
  if (!a || a->batch < 0 || a->draft_tokens < 0 || a->vocab <= 0 || !(a->temperature >= 0.f) ||
      !std::isfinite(a->temperature))
    return KVR_ERR_INVALID_ARGUMENT;
  if (a->dtype < 0 || a->dtype > 2) return KVR_ERR_UNSUPPORTED;
  if (a->temperature > 0.f && a->temperature < FLT_MIN) return KVR_ERR_UNSUPPORTED;   // its reciprocal may overflow
  if (a->draft_tokens > 4095 || (int64_t)a->batch * (a->draft_tokens + 1) > (1 << 24)) return KVR_ERR_UNSUPPORTED;
  const int n = a->dtype == 2 ? 4 : 8;
  const int64_t blocks = (a->vocab + n - 1) / n;
  const int64_t rows = std::max<int64_t>(1, (int64_t)a->batch * (a->draft_tokens + (a->temperature > 0.f ? 0 : 1)));
  Plan p;
  // 4 blocks of a row to a thread keep the registers at 64 (four CTAs per SM); fewer where that fills the GPU
  p.un = 4;
  for (; p.un > 1; p.un /= 2)
    if (rows * ((blocks + p.un * kThreads - 1) / (p.un * kThreads)) >= 296) break;
  p.chunks = (int)((blocks + p.un * kThreads - 1) / (p.un * kThreads));
  if (rows * p.chunks > (1ll << 31) - 1) return KVR_ERR_UNSUPPORTED;
  // Looking for an earlier refusal costs every CTA a round trip to L2 and saves reading: not for logits that
  // 5 us read anyway.
  p.skip = rows * a->vocab * (a->dtype == 2 ? 4 : 2) > (32 << 20);
  p.race_chunks = (int)((blocks + kRaceBlocks * kThreads - 1) / (kRaceBlocks * kThreads));
  if ((int64_t)a->batch * p.race_chunks > (1ll << 31) - 1) return KVR_ERR_UNSUPPORTED;
  const size_t B = a->batch, K1 = a->draft_tokens + 1;
  p.zeroed = B * K1 * 8 + B * K1 * 4 + 2 * B * 4;
  p.scratch = B * (K1 - 1) * ((size_t)p.chunks + 1) * sizeof(float4);
  *out = p;
  return KVR_OK;
}

template <typename T>
static cudaError_t launch(const Params& p, const Plan& pl, bool greedy, cudaStream_t s) {
  auto grid = [&](int rows) { return dim3((unsigned)((int64_t)rows * p.B * pl.chunks)); };
  if (greedy) {
    auto kern = pl.un == 4 ? greedy_kernel<T, 4> : pl.un == 2 ? greedy_kernel<T, 2> : greedy_kernel<T, 1>;
    return pdl_launch(kern, grid(p.K + 1), dim3(kThreads), 0, s, 1, p);
  }
  if (p.K > 0) {
    auto kern = pl.un == 4 ? stats_kernel<T, 4> : pl.un == 2 ? stats_kernel<T, 2> : stats_kernel<T, 1>;
    cudaError_t e = pdl_launch(kern, grid(p.K), dim3(kThreads), 0, s, 1, p);
    if (e != cudaSuccess) return e;
  }
  return pdl_launch(race_kernel<T>, dim3((unsigned)((int64_t)p.B * pl.race_chunks)), dim3(kThreads), 0, s, 1, p);
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
  p.B = a->batch; p.K = K; p.V = a->vocab; p.chunks = pl.chunks; p.race_chunks = pl.race_chunks;
  p.skip = pl.skip;
  p.c = greedy ? 1.f : 1.4426950408889634f / a->temperature;
  const size_t rows = (size_t)p.B * (K + 1);
  p.best = static_cast<unsigned long long*>(a->zeroed);
  p.arrived = reinterpret_cast<int*>(p.best + rows);
  p.done = p.arrived + rows;
  p.refused = p.done + p.B;
  p.stats = static_cast<float4*>(a->workspace);
  p.part = p.stats + (size_t)p.B * K;
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = a->dtype == 0   ? verify::launch<__nv_bfloat16>(p, pl, greedy, s)
                        : a->dtype == 1 ? verify::launch<__half>(p, pl, greedy, s)
                                        : verify::launch<float>(p, pl, greedy, s);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}
