// Eviction from a paged cache by accumulated attention weight (sm_100a).  No
// reference counterpart.
//
// A sequence longer than `keep` keeps its first `first` tokens, its last
// `recent` ones and, of those between, the heaviest, ties to the lowest
// index.  Two launches:
//  * select_kernel: one cluster of CTAs per sequence, each with a slice of
//    the weights in shared memory.  The weight of the last token to be kept
//    is found digit by digit (11 + 11 + 10 bits of the weight as an ordered
//    integer): a histogram per CTA, added up over distributed shared memory.
//    Then every CTA knows how many tokens the slices before it keep, and
//    writes its own in order.  What bounds it is the latency of the three
//    rounds, not the 4 bytes per token.
//  * copy_kernel: the kept rows into the new pages, all heads of a token by
//    the same CTA.  What bounds it is the rows' bytes, read once and written
//    once; the new pages are others than the old, so the order of copies does
//    not matter and pages that sequences share stay as they are.
#include "kvr_common.cuh"

#include <algorithm>

namespace kvr {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 2048;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}
// Word of another CTA's shared memory.
__device__ __forceinline__ uint32_t peer_word(const void* p, int rank) {
  uint32_t a, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Weights as integers in the same order (-0 as 0; NaN above all others).
__device__ __forceinline__ uint32_t ordered(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block; *total the whole.
__device__ __forceinline__ int block_scan(int x, int* buf, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += buf[w];
    all += buf[w];
  }
  *total = all;
  return before + incl - x;
}

struct Params {
  const float* weights;
  int64_t weights_b;
  const int* lengths;
  int* kept;            // [B, keep]
  int* new_lengths;     // [B]
  float* new_weights;   // [B, keep]
  int cap, keep, recent, first, slice, cluster;
};

__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint32_t keys[];   // [slice]
  __shared__ uint32_t hist[2][kBins];
  __shared__ int buf[kThreads / 32];
  __shared__ uint32_t s_counts[2];     // tokens kept for certain, ties
  __shared__ int s_digit[2];
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x % p.cluster, b = blockIdx.x / p.cluster;
  const int len = min(max(p.lengths[b], 0), p.cap);
  const float* w = p.weights + (int64_t)b * p.weights_b;
  int* kept = p.kept + (int64_t)b * p.keep;
  float* new_w = p.new_weights + (int64_t)b * p.keep;
  const int n_new = min(len, p.keep);
  if (rank == 0 && tid == 0) p.new_lengths[b] = n_new;
  // slots behind the last kept token
  for (int i = n_new + rank * kThreads + tid; i < p.keep; i += p.cluster * kThreads) {
    kept[i] = -1;
    new_w[i] = 0.f;
  }
  if (len <= p.keep) {   // all of them (the whole cluster takes this way out)
    for (int i = rank * kThreads + tid; i < len; i += p.cluster * kThreads) {
      kept[i] = i;
      new_w[i] = w[i];
    }
    return;
  }
  // candidates: [first, len - recent); this CTA's slice of the sequence
  const int c0 = p.first, c1 = len - p.recent;
  const int part = (len + p.cluster - 1) / p.cluster;   // <= slice
  const int s0 = min(rank * part, len), n = min(part, len - s0);
  for (int i = tid; i < n; i += kThreads) keys[i] = ordered(w[s0 + i]);
  const int lo = max(c0 - s0, 0), hi = min(c1 - s0, n);   // candidates of the slice
  int need = p.keep - p.first - p.recent;                 // heaviest candidates to keep
  uint32_t prefix = 0;                                    // digits of the need-th heaviest found so far
  int shift = 32;
  if (need > 0) {
    for (int round = 0; round < 3; ++round) {
      const int bits = round == 2 ? 10 : 11, bins = 1 << bits;
      uint32_t* h = hist[round & 1];
      for (int i = tid; i < bins; i += kThreads) h[i] = 0;
      __syncthreads();
      const int down = shift - bits;
      for (int i = lo + tid; i < hi; i += kThreads) {
        const uint32_t k = keys[i];
        if (round == 0 || (k >> shift) == prefix) atomicAdd(&h[(k >> down) & (bins - 1)], 1u);
      }
      if (p.cluster > 1) cluster_sync();
      else __syncthreads();
      // thread t adds up 4 (2 in the last round) bins, the highest first
      const int per = bins / kThreads, top = bins - 1 - tid * per;
      uint32_t c[4];
      int mine = 0;
      for (int j = 0; j < per; ++j) {
        c[j] = 0;
        if (p.cluster == 1) c[j] = h[top - j];
        else
          for (int r = 0; r < p.cluster; ++r) c[j] += peer_word(&h[top - j], r);
        mine += (int)c[j];
      }
      int total;
      int before = block_scan(mine, buf, &total);
      if (before < need && need <= before + mine) {
        for (int j = 0; j < per; ++j) {
          if (need <= before + (int)c[j]) {
            s_digit[0] = top - j;
            s_digit[1] = need - before;
            break;
          }
          before += (int)c[j];
        }
      }
      __syncthreads();
      prefix = round == 0 ? (uint32_t)s_digit[0] : (prefix << bits) | (uint32_t)s_digit[0];
      need = s_digit[1];   // of the tokens that share these digits, the heaviest `need`
      shift = down;
    }
  } else {
    __syncthreads();
  }
  // prefix is the key of the last token to be kept; `need` of its ties are, the first ones
  const bool any = p.keep - p.first - p.recent > 0;
  int sure = 0, ties = 0;
  for (int i = tid; i < n; i += kThreads) {
    const bool cand = i >= lo && i < hi;
    sure += !cand || (any && keys[i] > prefix);
    ties += cand && any && keys[i] == prefix;
  }
  int all_sure, all_ties;
  block_scan(sure, buf, &all_sure);
  block_scan(ties, buf, &all_ties);
  if (tid == 0) {
    s_counts[0] = (uint32_t)all_sure;
    s_counts[1] = (uint32_t)all_ties;
  }
  int at = 0, ties_before = 0;
  if (p.cluster > 1) {
    cluster_sync();
    for (int r = 0; r < rank; ++r) {
      at += (int)peer_word(&s_counts[0], r);
      ties_before += (int)peer_word(&s_counts[1], r);
    }
  }
  at += min(ties_before, need);
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + tid;
    const bool cand = i >= lo && i < hi, live = i < n;
    const bool tie = live && cand && any && keys[i] == prefix;
    int n_ties, n_kept;
    const int tie_rank = ties_before + block_scan(tie, buf, &n_ties);
    const bool keep = live && (!cand || (any && keys[i] > prefix) || (tie && tie_rank < need));
    const int pos = at + block_scan(keep, buf, &n_kept);
    if (keep) {
      kept[pos] = s0 + i;
      new_w[pos] = w[s0 + i];
    }
    at += n_kept;
    ties_before += n_ties;
  }
  if (p.cluster > 1) cluster_sync();   // peers may still read this CTA's counts
}

constexpr int kCopyTokens = 32, kCopyThreads = 256;

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ kvr_paged_evict_args a) {
  __shared__ int64_t src[kCopyTokens][2], dst[kCopyTokens][2];
  pdl_wait();
  const int b = blockIdx.y, i0 = blockIdx.x * kCopyTokens;
  if (threadIdx.x < kCopyTokens) {
    const int i = i0 + threadIdx.x;
    int64_t s = -1, sv = 0, d = 0, dv = 0;
    const int j = i < a.keep ? a.kept[(int64_t)b * a.keep + i] : -1;
    if (j >= 0) {
      const int from = a.block_table[(int64_t)b * a.table_stride + j / a.page_size];
      const int to = i / a.page_size < a.new_table_width
                         ? a.new_block_table[(int64_t)b * a.new_table_stride + i / a.page_size]
                         : -1;
      if (from >= 0 && from < a.num_pages && to >= 0 && to < a.num_pages) {
        const int rs = j % a.page_size, rd = i % a.page_size;
        s = (int64_t)from * a.key_page_stride + (int64_t)rs * a.key_row_stride;
        d = (int64_t)to * a.key_page_stride + (int64_t)rd * a.key_row_stride;
        sv = (int64_t)from * a.value_page_stride + (int64_t)rs * a.value_row_stride;
        dv = (int64_t)to * a.value_page_stride + (int64_t)rd * a.value_row_stride;
      }
    }
    src[threadIdx.x][0] = s;
    src[threadIdx.x][1] = sv;
    dst[threadIdx.x][0] = d;
    dst[threadIdx.x][1] = dv;
  }
  __syncthreads();
  const int pieces = a.head_dim / 8, per_head = kCopyTokens * pieces, n = a.kv_heads * per_head;
  uint16_t* kp = static_cast<uint16_t*>(a.key_pages);
  uint16_t* vp = static_cast<uint16_t*>(a.value_pages);
#pragma unroll 4
  for (int x = threadIdx.x; x < n; x += kCopyThreads) {
    const int h = x / per_head, y = x - h * per_head, t = y / pieces, c = y - t * pieces;
    if (src[t][0] < 0) continue;
    const int64_t ko = (int64_t)h * a.key_head_stride + c * 8, vo = (int64_t)h * a.value_head_stride + c * 8;
    const uint4 k = *reinterpret_cast<const uint4*>(kp + src[t][0] + ko);
    const uint4 v = *reinterpret_cast<const uint4*>(vp + src[t][1] + vo);
    *reinterpret_cast<uint4*>(kp + dst[t][0] + ko) = k;
    *reinterpret_cast<uint4*>(vp + dst[t][1] + vo) = v;
  }
}

// Slices of at most 40,000 weights (160 KB of shared memory), clusters of at most 8.
constexpr int kMaxSlice = 40000;

}  // namespace evict
}  // namespace kvr

using namespace kvr;

extern "C" int kvr_paged_evict(const kvr_paged_evict_args* a, kvr_stream_t stream) {
  if (!a || a->batch < 0 || a->kv_heads <= 0 || a->page_size <= 0 || a->table_width < 0 || a->num_pages < 0 ||
      a->new_table_width < 0 || a->head_dim <= 0 || a->keep <= 0 || a->recent < 0 || a->first < 0 ||
      (int64_t)a->first + a->recent > a->keep)
    return KVR_ERR_INVALID_ARGUMENT;
  if (a->head_dim % 8) return KVR_ERR_UNSUPPORTED;
  const int64_t cap = (int64_t)a->table_width * a->page_size;
  if (cap > 8ll * evict::kMaxSlice || a->batch > 65535) return KVR_ERR_UNSUPPORTED;
  if ((int64_t)a->new_table_width * a->page_size < std::min<int64_t>(a->keep, cap)) return KVR_ERR_CAPACITY;
  if (a->batch == 0) return KVR_OK;
  if (!a->lengths || !a->kept || !a->new_lengths || !a->new_weights ||
      (cap > 0 && (!a->block_table || !a->new_block_table || !a->token_weights)) ||
      (a->num_pages > 0 && (!a->key_pages || !a->value_pages)))
    return KVR_ERR_INVALID_ARGUMENT;
  const int64_t strides[] = {a->key_page_stride, a->key_head_stride, a->key_row_stride,
                             a->value_page_stride, a->value_head_stride, a->value_row_stride};
  for (int64_t x : strides)
    if (x & 7) return KVR_ERR_MISALIGNED;
  if (!aligned16(a->key_pages) || !aligned16(a->value_pages)) return KVR_ERR_MISALIGNED;
  cudaStream_t s = as_stream(stream);

  evict::Params p;
  p.weights = a->token_weights; p.weights_b = a->weights_b_stride;
  p.lengths = a->lengths; p.kept = a->kept; p.new_lengths = a->new_lengths; p.new_weights = a->new_weights;
  p.cap = (int)cap; p.keep = a->keep; p.recent = a->recent; p.first = a->first;
  // CTAs per sequence: as many as fit the GPU beside the batch, of 1024 weights or more
  p.cluster = 1;
  while (p.cluster < 8 && (cap > (int64_t)p.cluster * evict::kMaxSlice ||
                           (cap > 1024ll * p.cluster && (int64_t)a->batch * p.cluster * 2 <= 148)))
    p.cluster *= 2;
  p.slice = (int)std::max<int64_t>(1, (cap + p.cluster - 1) / p.cluster);
  const size_t smem = (size_t)p.slice * sizeof(uint32_t);
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (!ready[dev & 63]) {   // a benign race sets the same value
    const cudaError_t e = cudaFuncSetAttribute(evict::select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               evict::kMaxSlice * (int)sizeof(uint32_t));
    if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
    ready[dev & 63] = true;
  }
  cudaError_t e = pdl_launch(evict::select_kernel, dim3((unsigned)(a->batch * p.cluster)), dim3(evict::kThreads), smem,
                             s, p.cluster, p);
  const int64_t rows = std::min<int64_t>(a->keep, cap);
  if (e == cudaSuccess && rows > 0)
    e = pdl_launch(evict::copy_kernel,
                   dim3((unsigned)((rows + evict::kCopyTokens - 1) / evict::kCopyTokens), (unsigned)a->batch),
                   dim3(evict::kCopyThreads), 0, s, 1, *a);
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}
