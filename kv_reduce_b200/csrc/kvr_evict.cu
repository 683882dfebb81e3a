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
//    not matter and pages that sequences share stay as they are.  The last
//    `recent` tokens are kept whatever the weights say: their rows are copied
//    while the selection runs.
//
// Measured (bf16): 32 sequences of 4K to 16K to 4096, of them 1024 recent, 8
// heads of 64: 0.54 GB in 99 us, 5450 GB/s (107 us without the early copies;
// the copy alone runs at 94% of a plain copy's rate, the selection takes 15
// us); one of 5000 to 1024, 2 heads of 128: 11 us, the selection's latency.
#include "kvr_common.cuh"

#include <algorithm>

namespace kvr {
namespace evict {

constexpr int kThreads = 512;
constexpr int kBins = 2048;

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}
// A word of another CTA's shared memory.
__device__ __forceinline__ uint32_t peer_word(const void* p, int rank) {
  uint32_t a, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}
// 16 bytes at `p` from N CTAs, ranks r0 on.  One statement, so that the loads
// are all on their way before the first is used (left to itself the compiler
// adds each up as it arrives, a round trip apiece).
template <int N>
__device__ __forceinline__ void peer_vectors(const void* p, int r0, uint4 (&v)[N]) {
  static_assert(N == 2 || N == 4, "");
  const uint32_t a = smem_u32(p);
  if constexpr (N == 2) {
    asm volatile(
        "{\n.reg .u32 a0, a1;\n"
        "mapa.shared::cluster.u32 a0, %8, %9;\nmapa.shared::cluster.u32 a1, %8, %10;\n"
        "ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [a0];\nld.shared::cluster.v4.u32 {%4, %5, %6, %7}, [a1];\n}\n"
        : "=&r"(v[0].x), "=&r"(v[0].y), "=&r"(v[0].z), "=&r"(v[0].w), "=&r"(v[1].x), "=&r"(v[1].y), "=&r"(v[1].z),
          "=&r"(v[1].w)
        : "r"(a), "r"(r0), "r"(r0 + 1)
        : "memory");
  } else {
    asm volatile(
        "{\n.reg .u32 a0, a1, a2, a3;\n"
        "mapa.shared::cluster.u32 a0, %16, %17;\nmapa.shared::cluster.u32 a1, %16, %18;\n"
        "mapa.shared::cluster.u32 a2, %16, %19;\nmapa.shared::cluster.u32 a3, %16, %20;\n"
        "ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [a0];\nld.shared::cluster.v4.u32 {%4, %5, %6, %7}, [a1];\n"
        "ld.shared::cluster.v4.u32 {%8, %9, %10, %11}, [a2];\nld.shared::cluster.v4.u32 {%12, %13, %14, %15}, [a3];\n"
        "}\n"
        : "=&r"(v[0].x), "=&r"(v[0].y), "=&r"(v[0].z), "=&r"(v[0].w), "=&r"(v[1].x), "=&r"(v[1].y), "=&r"(v[1].z),
          "=&r"(v[1].w), "=&r"(v[2].x), "=&r"(v[2].y), "=&r"(v[2].z), "=&r"(v[2].w), "=&r"(v[3].x), "=&r"(v[3].y),
          "=&r"(v[3].z), "=&r"(v[3].w)
        : "r"(a), "r"(r0), "r"(r0 + 1), "r"(r0 + 2), "r"(r0 + 3)
        : "memory");
  }
}

// Weights as integers in the same order (-0 as 0; NaN above all others).
__device__ __forceinline__ uint32_t ordered(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  return w != w ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Exclusive sum over the block; *total the whole.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* buf, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(~0u, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = incl;
  __syncthreads();
  uint32_t before = 0, all = 0;
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
  int cap, keep, recent, first, slice;
};

// CL: CTAs of the cluster, one sequence.  Its slices are contiguous, and so
// are the threads' runs within a slice (of an odd number of words, so that 32
// runs are read without bank conflicts), so that one sum over the block gives
// every thread its place.
template <int CL>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ Params p) {
  extern __shared__ float slice[];     // [p.slice]
  __shared__ __align__(16) uint32_t hist[2][kBins];
  __shared__ uint32_t buf[kThreads / 32];
  __shared__ uint32_t s_counts;        // tokens kept for certain | ties << 16
  __shared__ int s_digit[2];
  const int tid = threadIdx.x, rank = CL == 1 ? 0 : blockIdx.x % CL, b = blockIdx.x / CL;
  for (int i = tid; i < 2 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
  // what came before is done: now the copies that need no selection may start
  pdl_wait();
  pdl_trigger();
  const int len = min(max(p.lengths[b], 0), p.cap);
  const float* w = p.weights + (int64_t)b * p.weights_b;
  int* kept = p.kept + (int64_t)b * p.keep;
  float* new_w = p.new_weights + (int64_t)b * p.keep;
  const int n_new = min(len, p.keep);
  if (rank == 0 && tid == 0) p.new_lengths[b] = n_new;
  // slots behind the last kept token
  for (int i = n_new + rank * kThreads + tid; i < p.keep; i += CL * kThreads) {
    kept[i] = -1;
    new_w[i] = 0.f;
  }
  if (len <= p.keep) {   // all of them (the whole cluster takes this way out)
    for (int i = rank * kThreads + tid; i < len; i += CL * kThreads) {
      kept[i] = i;
      new_w[i] = w[i];
    }
    return;
  }
  // candidates: [first, len - recent); this CTA's slice of the sequence
  const int part = (len + CL - 1) / CL;   // <= p.slice
  const int s0 = min(rank * part, len), n = min(part, len - s0);
#pragma unroll 4
  for (int i = tid; i < n; i += kThreads) slice[i] = __ldg(w + s0 + i);
  const int lo = max(p.first - s0, 0), hi = min(len - p.recent - s0, n);   // candidates of the slice
  int need = p.keep - p.first - p.recent;                                  // heaviest candidates to keep
  const bool any = need > 0;
  uint32_t prefix = 0;                                                     // digits of the need-th heaviest so far
  __syncthreads();
  if (any) {
#pragma unroll
    for (int round = 0; round < 3; ++round) {
      // bits 31-21, 20-10, 9-0 (the last round on 1024 bins)
      const int down = round == 0 ? 21 : round == 1 ? 10 : 0, up = round == 1 ? 21 : 10;
      const int bins = round == 2 ? 1024 : 2048;
      uint32_t* h = hist[round & 1];
      for (int i = lo + tid; i < hi; i += kThreads) {
        const uint32_t k = ordered(slice[i]);
        if (round == 0 || (k >> up) == prefix) atomicAdd(&h[(k >> down) & (bins - 1)], 1u);
      }
      if (CL > 1) cluster_sync();
      else __syncthreads();
      // thread t adds up 4 bins over the cluster, the highest first (in the last round half the threads do)
      const int at = bins - 4 - tid * 4;   // its lowest bin
      uint32_t c[4] = {0, 0, 0, 0};
      if (at >= 0) {
        auto add = [&](const uint4& x) {
          c[0] += x.x; c[1] += x.y; c[2] += x.z; c[3] += x.w;
        };
        if constexpr (CL == 1) {
          add(*reinterpret_cast<const uint4*>(&h[at]));
        } else {
          constexpr int N = CL < 4 ? CL : 4;
#pragma unroll
          for (int r = 0; r < CL; r += N) {
            uint4 v[N];
            peer_vectors<N>(&h[at], r, v);
#pragma unroll
            for (int y = 0; y < N; ++y) add(v[y]);
          }
        }
      }
      uint32_t total;
      int before = (int)block_scan(c[0] + c[1] + c[2] + c[3], buf, &total);
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        if (before < need && need <= before + (int)c[j]) {
          s_digit[0] = at + j;
          s_digit[1] = need - before;
        }
        before += (int)c[j];
      }
      // round 2 counts where round 0 did: every peer has read that by now (it is past round 1's cluster barrier)
      if (round == 1)
        for (int i = tid; i < kBins; i += kThreads) hist[0][i] = 0;
      __syncthreads();
      prefix = round == 0 ? (uint32_t)s_digit[0] : (prefix << (round == 1 ? 11 : 10)) | (uint32_t)s_digit[0];
      need = s_digit[1];   // of the tokens that share these digits, the heaviest `need`
    }
  }
  // prefix is the key of the last token to be kept; `need` of its ties are, the first ones
  const int run = ((n + kThreads - 1) / kThreads) | 1, r0 = min(tid * run, n), r1 = min(r0 + run, n);
  uint32_t mine = 0;   // (a slice may hold 40,000 ties: the upper half needs its sign bit)
  for (int i = r0; i < r1; ++i) {
    const uint32_t k = ordered(slice[i]);
    const bool cand = i >= lo && i < hi;
    mine += !cand || (any && k > prefix) ? 1u : any && k == prefix ? 1u << 16 : 0u;
  }
  uint32_t total;
  const uint32_t before = block_scan(mine, buf, &total);
  int sure = (int)(before & 0xffff), ties = (int)(before >> 16);
  if (CL > 1) {
    if (tid == 0) s_counts = total;
    cluster_sync();
    // lane r asks CTA r
    const int lane = tid & 31;
    const uint32_t x = lane < rank ? peer_word(&s_counts, lane) : 0u;
    sure += __reduce_add_sync(~0u, (int)(x & 0xffff));
    ties += __reduce_add_sync(~0u, (int)(x >> 16));
  }
  for (int i = r0; i < r1; ++i) {
    const uint32_t k = ordered(slice[i]);
    const bool cand = i >= lo && i < hi, in = !cand || (any && k > prefix), tie = !in && any && k == prefix;
    if (in || (tie && ties < need)) {
      const int pos = sure + min(ties, need);
      kept[pos] = s0 + i;
      new_w[pos] = slice[i];
    }
    sure += in;
    ties += tie;
  }
  if (CL > 1) cluster_sync();   // peers may still read this CTA's counts
}

constexpr int kCopyTokens = 32, kCopyThreads = 256;

// Blocks of kCopyTokens slots; first the `early` last ones of every sequence,
// which hold recent tokens only, then the others.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ kvr_paged_evict_args a, int blocks,
                                                            int early, int cap) {
  __shared__ int64_t src[kCopyTokens][2], dst[kCopyTokens][2];
  const int n_early = a.batch * early, late = blocks - early;
  const bool is_early = (int)blockIdx.x < n_early;
  const int u = is_early ? blockIdx.x : blockIdx.x - n_early;
  const int b = u / (is_early ? early : late), i0 = (is_early ? late + u % early : u % late) * kCopyTokens;
  // The selection passed its own wait before this kernel could start, so lengths, tables and pages are there;
  // `kept` is only behind this one's wait.  (No early trigger here: a selection that starts beside this kernel's
  // last CTAs slows them by a tenth.)
  if (!is_early) pdl_wait();
  if (threadIdx.x < kCopyTokens) {
    const int i = i0 + threadIdx.x;
    int64_t s = -1, sv = 0, d = 0, dv = 0;
    int j = -1;
    if (i < a.keep) {
      if (is_early) {
        const int len = min(max(a.lengths[b], 0), cap);
        j = len > a.keep ? len - a.keep + i : i < len ? i : -1;
      } else {
        j = a.kept[(int64_t)b * a.keep + i];
      }
    }
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
  if (is_early) pdl_wait();   // this kernel must not be done before the selection
}

// Slices of at most 40,000 weights: 160 KB of shared memory, counts of 16 bits.
constexpr int kMaxSlice = 40000;

template <int CL>
static cudaError_t launch_select(const Params& p, int batch, cudaStream_t s) {
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  if (!ready[dev & 63]) {   // a benign race sets the same value
    const cudaError_t e = cudaFuncSetAttribute(select_kernel<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kMaxSlice * (int)sizeof(float));
    if (e != cudaSuccess) return e;
    ready[dev & 63] = true;
  }
  return pdl_launch(select_kernel<CL>, dim3((unsigned)(batch * CL)), dim3(kThreads), (size_t)p.slice * sizeof(float), s,
                    CL, p);
}

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
  // (keep at most 2^30: slots and what a thread adds to them stay inside 32 bits)
  if (cap > 8ll * evict::kMaxSlice || a->batch > 65535 || a->keep > (1 << 30)) return KVR_ERR_UNSUPPORTED;
  if ((int64_t)a->new_table_width * a->page_size < std::min<int64_t>(a->keep, cap)) return KVR_ERR_CAPACITY;
  if (a->batch == 0) return KVR_OK;
  if (!a->lengths || !a->kept || !a->new_lengths || !a->new_weights ||
      (cap > 0 && (!a->block_table || !a->new_block_table || !a->token_weights)) ||
      (a->num_pages > 0 && (!a->key_pages || !a->value_pages)))
    return KVR_ERR_INVALID_ARGUMENT;
  // every CTA of a sequence reads what these would overwrite
  if (a->new_lengths == a->lengths || a->new_weights == a->token_weights) return KVR_ERR_INVALID_ARGUMENT;
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
  // CTAs per sequence, while they fit the GPU beside the batch: a CTA takes 4096 weights about as fast as a
  // cluster shares them (5K weights: 10.5, 10.9, 12.0, 15.1 us for the whole call with 1, 2, 4, 8 CTAs; 32 times
  // 4K to 16K: 114, 109, 107, 118 us), and a cluster of 8 takes 3 us longer than one of 4.
  int cluster = 1;
  while (cluster < 8 && (cap > (int64_t)cluster * evict::kMaxSlice ||
                         (cap > (cluster < 4 ? 4096ll : 8192ll) * cluster && (int64_t)a->batch * cluster * 2 <= 148)))
    cluster *= 2;
  p.slice = (int)std::max<int64_t>(1, (cap + cluster - 1) / cluster);
  cudaError_t e = cluster == 8   ? evict::launch_select<8>(p, a->batch, s)
                  : cluster == 4 ? evict::launch_select<4>(p, a->batch, s)
                  : cluster == 2 ? evict::launch_select<2>(p, a->batch, s)
                                 : evict::launch_select<1>(p, a->batch, s);
  const int64_t rows = std::min<int64_t>(a->keep, cap);
  if (e == cudaSuccess && rows > 0) {
    // slots [keep - recent, keep): whole blocks of them need no selection
    const int blocks = (int)((rows + evict::kCopyTokens - 1) / evict::kCopyTokens);
    const int first_early = (a->keep - a->recent + evict::kCopyTokens - 1) / evict::kCopyTokens;
    const int early = std::max(0, blocks - first_early);
    if ((int64_t)blocks * a->batch > (1ll << 31) - 1) return KVR_ERR_UNSUPPORTED;
    e = pdl_launch(evict::copy_kernel, dim3((unsigned)(blocks * a->batch)), dim3(evict::kCopyThreads), 0, s, 1, *a, blocks,
                   early, (int)cap);
  }
  if (e != cudaSuccess) { set_last_cuda_error(e); return KVR_ERR_CUDA; }
  return KVR_OK;
}
