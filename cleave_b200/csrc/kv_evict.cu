// Eviction from a paged KV cache by accumulated attention weight.
//
// Per (request, kv head) with n tokens, B = min(n, budget, room in the destination pages) of them stay: the first
// min(sinks, B), the last min(recent, B - those), and of the tokens between them the ones with the largest weight
// sums; equal sums go to the lower index, NaN counts as the largest value. The kept rows of K and V are copied, in
// their order, into the destination pages, and their sums with them.
//
// Two kernels. evict_select_kernel (one CTA per (request, kv head)) finds the smallest kept sum by a radix select over
// the sums' bits and writes the kept indices in order. evict_copy_kernel moves the rows: it has no dependence between
// its CTAs (source and destination pages are disjoint), so it is a plain gather of 2 D-byte rows that is bound by the
// memory's bandwidth, which is nearly all of the operator's time where the cache is large.

#include "common.cuh"

namespace cb200 {
namespace {

constexpr int kSelThreads = 512;
constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 128;  // (token, head) rows of K and of V per CTA

struct EvictParams {
  uint4* k;
  uint4* v;
  const float* sums;
  const int* kv_indptr;
  const int* kv_indices;
  const int* kv_last;
  const int* dst_indptr;
  const int* dst_indices;
  int* kept;
  float* kept_sums;
  int* dst_last;
  int hkv, row16, page_size, num_pages, n_idx, n_dst, max_len, budget, sinks, recent;  // row16: 16-byte chunks of a row
};

// the range of a request in a page table that is caller data: clipped to the entries that exist
__device__ __forceinline__ int2 table_range(const int* indptr, int b, int n_idx) {
  const int base = indptr[b];
  if (base < 0 || base >= n_idx) return make_int2(0, 0);
  return make_int2(base, max(min(indptr[b + 1] - base, n_idx - base), 0));
}

struct Request {
  int n, keep, src0, dst0;  // tokens, tokens that stay, first entries in the two page tables
};

__device__ __forceinline__ Request request_of(const EvictParams& p, int b) {
  const int2 src = table_range(p.kv_indptr, b, p.n_idx), dst = table_range(p.dst_indptr, b, p.n_dst);
  Request r;
  r.src0 = src.x;
  r.dst0 = dst.x;
  if (p.page_size == 1 || p.kv_last == nullptr) {
    r.n = src.y * p.page_size;
  } else {
    r.n = max(min(max(src.y - 1, 0) * p.page_size + max(p.kv_last[b], 0), src.y * p.page_size), 0);
  }
  const long long room = static_cast<long long>(dst.y) * p.page_size;
  r.keep = static_cast<int>(min(static_cast<long long>(min(r.n, p.budget)), room));
  return r;
}

// Bits whose unsigned order is the order of the sums: -0 counts as 0, NaN as the largest value.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int hist[256];
  __shared__ int found[2];  // digit, values above it
  __shared__ int warp_strict[kSelThreads / 32], warp_tie[kSelThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Request r = request_of(p, b);
  const size_t pair = static_cast<size_t>(b) * p.hkv + h;
  const float* sums = p.sums + pair * p.max_len;
  int* kept = p.kept + pair * p.budget;
  float* kept_sums = p.kept_sums + pair * p.max_len;
  const int first = min(p.sinks, r.keep), tail = min(p.recent, r.keep - first);
  const int lo = first, hi = r.n - tail;      // the tokens that are ranked: lo <= j < hi
  const int middle = r.keep - first - tail;   // of which this many stay
  auto sum_of = [&](int j) { return j < p.max_len ? __ldg(sums + j) : 0.f; };  // tokens without a record weigh nothing

  if (h == 0 && tid == 0) p.dst_last[b] = r.keep > 0 ? (r.keep - 1) % p.page_size + 1 : 0;
  auto put = [&](int i, int j) {
    kept[i] = j;
    if (i < p.max_len) kept_sums[i] = sum_of(j);
  };
  for (int i = tid; i < first; i += kSelThreads) put(i, i);
  for (int i = tid; i < tail; i += kSelThreads) put(r.keep - tail + i, r.n - tail + i);
  for (int i = r.keep + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
  for (int i = r.keep + tid; i < p.max_len; i += kSelThreads) kept_sums[i] = 0.f;
  if (middle <= 0) return;
  if (middle == hi - lo) {
    for (int i = tid; i < middle; i += kSelThreads) put(lo + i, lo + i);
    return;
  }

  // ---- the key of rank `middle`, eight bits at a time from the top
  uint32_t prefix = 0;
  int want = middle;  // its rank among the keys that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kSelThreads) {
      const uint32_t key = order_key(sum_of(j));
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds the digits 255 - 8 l .. 248 - 8 l, largest first
      int mine = 0, c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += c[i] = hist[255 - 8 * lane - i];
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int above = incl - mine;
      if (above < want && want <= incl) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < want && want <= above + c[i]) {
            found[0] = 255 - 8 * lane - i;
            found[1] = above;
          }
          above += c[i];
        }
      }
    }
    __syncthreads();
    prefix = (prefix << 8) | static_cast<uint32_t>(found[0]);
    want -= found[1];
  }
  // keys above `prefix` stay, and the first `want` of those equal to it
  int done_strict = 0, done_tie = 0;
  for (int j0 = lo; j0 < hi; j0 += kSelThreads) {
    const int j = j0 + tid;
    const uint32_t key = j < hi ? order_key(sum_of(j)) : 0u;
    const bool strict = j < hi && key > prefix, tie = j < hi && key == prefix;
    const uint32_t bs = __ballot_sync(0xffffffffu, strict), bt = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) {
      warp_strict[warp] = __popc(bs);
      warp_tie[warp] = __popc(bt);
    }
    __syncthreads();
    int s = done_strict, t = done_tie;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) {
        s += warp_strict[w];
        t += warp_tie[w];
      }
      done_strict += warp_strict[w];
      done_tie += warp_tie[w];
    }
    const uint32_t below = (1u << lane) - 1;
    s += __popc(bs & below);
    t += __popc(bt & below);
    if (strict || (tie && t < want)) put(lo + s + min(t, want), j);
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p) {
  __shared__ long long src_off[kCopyRows], dst_off[kCopyRows];  // in 16-byte chunks; dst < 0: no such page
  pdl_wait();
  const int b = blockIdx.y;
  const Request r = request_of(p, b);
  const long long rows = static_cast<long long>(r.keep) * p.hkv;  // (token, head), heads innermost
  const long long r0 = static_cast<long long>(blockIdx.x) * kCopyRows;
  if (r0 >= rows) return;
  const int here = static_cast<int>(min(static_cast<long long>(kCopyRows), rows - r0));
  for (int x = threadIdx.x; x < here; x += kCopyThreads) {
    const int i = static_cast<int>((r0 + x) / p.hkv), h = static_cast<int>((r0 + x) % p.hkv);
    const int j = __ldcg(p.kept + (static_cast<size_t>(b) * p.hkv + h) * p.budget + i);
    const int sp = min(max(__ldg(p.kv_indices + r.src0 + j / p.page_size), 0), p.num_pages - 1);
    const int dp = __ldg(p.dst_indices + r.dst0 + i / p.page_size);
    src_off[x] = ((static_cast<long long>(sp) * p.page_size + j % p.page_size) * p.hkv + h) * p.row16;
    dst_off[x] = dp < 0 || dp >= p.num_pages ? -1 : ((static_cast<long long>(dp) * p.page_size + i % p.page_size) * p.hkv + h) * p.row16;
  }
  __syncthreads();
  const int chunks = here * p.row16;
  constexpr int kAhead = 4;
  for (int c0 = threadIdx.x; c0 < chunks; c0 += kAhead * kCopyThreads) {
    uint4 kk[kAhead], vv[kAhead];
    long long to[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u * kCopyThreads;
      to[u] = -1;
      if (c < chunks) {
        const int x = c / p.row16, w = c - x * p.row16;
        kk[u] = __ldcs(p.k + src_off[x] + w);
        vv[u] = __ldcs(p.v + src_off[x] + w);
        if (dst_off[x] >= 0) to[u] = dst_off[x] + w;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (to[u] >= 0) {
        p.k[to[u]] = kk[u];
        p.v[to[u]] = vv[u];
      }
    }
  }
}

}  // namespace
}  // namespace cb200

extern "C" int cb200_kv_evict(const cb200_kv_evict_args* a, void* stream) {
  using namespace cb200;
  if (!a || a->batch <= 0 || a->num_kv_heads <= 0 || a->head_dim <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->max_len <= 0 ||
      a->budget <= 0 || a->sinks < 0 || a->recent < 0 || a->num_kv_indices < 0 || a->num_dst_indices < 0)
    return CB200_ERR_BAD_ARG;
  if (static_cast<long long>(a->sinks) + a->recent > a->budget) return CB200_ERR_BAD_ARG;
  if (a->head_dim % 8 || a->batch > 65535) return CB200_ERR_UNSUPPORTED;
  // token counts are held in 32 bits
  if (static_cast<long long>(a->num_kv_indices) * a->page_size >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  const long long copy_ctas = (static_cast<long long>(a->budget) * a->num_kv_heads + kCopyRows - 1) / kCopyRows;
  if (copy_ctas >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  if (!a->k_cache || !a->v_cache || !a->weight_sums || !a->kv_indptr || !a->dst_indptr || !a->kept || !a->kept_sums || !a->dst_last_page_len)
    return CB200_ERR_BAD_ARG;
  if ((!a->kv_indices && a->num_kv_indices > 0) || (!a->dst_indices && a->num_dst_indices > 0)) return CB200_ERR_BAD_ARG;
  if (a->page_size != 1 && !a->kv_last_page_len) return CB200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return CB200_ERR_ALIGNMENT;
  EvictParams p{};
  p.k = static_cast<uint4*>(a->k_cache);
  p.v = static_cast<uint4*>(a->v_cache);
  p.sums = a->weight_sums;
  p.kv_indptr = a->kv_indptr;
  p.kv_indices = a->kv_indices;
  p.kv_last = a->kv_last_page_len;
  p.dst_indptr = a->dst_indptr;
  p.dst_indices = a->dst_indices;
  p.kept = a->kept;
  p.kept_sums = a->kept_sums;
  p.dst_last = a->dst_last_page_len;
  p.hkv = a->num_kv_heads;
  p.row16 = a->head_dim / 8;
  p.page_size = a->page_size;
  p.num_pages = a->num_pages;
  p.n_idx = a->num_kv_indices;
  p.n_dst = a->num_dst_indices;
  p.max_len = a->max_len;
  p.budget = a->budget;
  p.sinks = a->sinks;
  p.recent = a->recent;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a->num_kv_heads), static_cast<unsigned>(a->batch), 1);
  cfg.blockDim = dim3(kSelThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
  cfg.gridDim = dim3(static_cast<unsigned>(copy_ctas), static_cast<unsigned>(a->batch), 1);
  cfg.blockDim = dim3(kCopyThreads, 1, 1);
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_copy_kernel, p));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}
