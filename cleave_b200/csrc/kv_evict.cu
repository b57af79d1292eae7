// Eviction from a paged KV cache by accumulated attention weight.
//
// Per (request, kv head) with n tokens, B = min(n, budget, room in the destination pages) of them stay: the first
// min(sinks, B), the last min(recent, B - those), and of the tokens between them the ones with the largest weight
// sums; equal sums go to the lower index, NaN counts as the largest value. The kept rows of K and V are copied, in
// their order, into the destination pages, and their sums with them.
//
// Two kernels. evict_select_kernel (one CTA per (request, kv head)) finds the smallest kept sum with two or three
// histograms over the sums, which it holds in registers, and writes the kept indices in order. evict_copy_kernel moves the
// rows: it has no dependence between its CTAs (source and destination pages are disjoint), so it is a plain gather of
// 2 D-byte rows that is bound by the memory's bandwidth, which is nearly all of the operator's time where the cache is large.
// Measured: 32 requests of 1000 .. 8192 tokens cut to 2048, 8 heads of 128: 92 us (the selection alone 16, the copy of 528
// MB alone 83); one request of 1500 cut to 512: 6.7 us.

#include "common.cuh"

namespace cb200 {
namespace {

constexpr int kSelThreads = 512;
constexpr int kBinBits = 11, kBins = 1 << kBinBits;  // four bins a thread
constexpr int kKeysMost = 64;   // sums a thread of the select kernel holds at most
constexpr int kCopyThreads = 256;

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
  int batch, hkv, row16, page_size, num_pages, n_idx, n_dst, max_len, budget, sinks, recent;  // row16: 16-byte chunks of a row
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
    r.n = min(max(src.y - 1, 0) * p.page_size + min(max(p.kv_last[b], 0), p.page_size), src.y * p.page_size);
  }
  const long long room = static_cast<long long>(dst.y) * p.page_size;
  r.keep = static_cast<int>(min(static_cast<long long>(min(r.n, p.budget)), room));
  return r;
}

// Bits whose unsigned order is the order of the sums: -0 counts as 0, NaN as the largest value.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : k;
}

// KEYS: sums a thread holds in registers (thread t of the CTA: tokens lo + t, lo + t + 512, ...). The sums of a longer
// range are read again in every step.
template <int KEYS>
__global__ void __launch_bounds__(kSelThreads, KEYS <= 16 ? 2 : 1) evict_select_kernel(const EvictParams p) {
  constexpr int kWarps = kSelThreads / 32;
  __shared__ __align__(16) int bins[kBins];
  __shared__ uint32_t range[2][kWarps];
  __shared__ int warp_sum[kWarps], found[3];  // found: bin, keys in bins above it, keys in it
  __shared__ uint32_t slab[KEYS * kWarps];  // tokens above the threshold, and those equal to it << 16
  __shared__ uint32_t slab_all;
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
  auto key_of = [&](int j) { return j < hi ? order_key(sum_of(j)) : 0u; };     // no sum has the key 0
  const bool rank = middle > 0 && middle < hi - lo;
  uint32_t key[KEYS];
  // all loads first, none of them behind a branch: they are in flight together
  auto load_keys = [&](int j0) {
    float x[KEYS];
    const int last = max(min(hi, p.max_len) - 1, 0);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) x[i] = __ldg(sums + min(j0 + i * kSelThreads + tid, last));
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = j0 + i * kSelThreads + tid;
      key[i] = j < hi ? order_key(j < p.max_len ? x[i] : 0.f) : 0u;
    }
  };
  if (rank) load_keys(lo);

  if (h == 0 && tid == 0) p.dst_last[b] = r.keep > 0 ? (r.keep - 1) % p.page_size + 1 : 0;
  for (int i = tid; i < first; i += kSelThreads) kept[i] = i;
  for (int i = tid; i < tail; i += kSelThreads) kept[r.keep - tail + i] = r.n - tail + i;
  for (int i = r.keep + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
  for (int i = r.keep + tid; i < p.max_len; i += kSelThreads) kept_sums[i] = 0.f;
  // The kept sums are copied at the end, through the indices: loads and stores of whole warps, several in flight.
  auto carry_sums = [&]() {
    __syncthreads();
    const int n = min(r.keep, p.max_len);
    for (int i0 = tid; i0 < n; i0 += 4 * kSelThreads) {
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = i0 + u * kSelThreads < n ? sum_of(__ldcg(kept + i0 + u * kSelThreads)) : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * kSelThreads < n) kept_sums[i0 + u * kSelThreads] = x[u];
    }
  };
  if (!rank) {
    for (int i = tid; i < middle; i += kSelThreads) kept[lo + i] = lo + i;
    carry_sums();
    return;
  }

  auto each_key = [&](auto&& f) {  // every ranked key of this thread, and 0 for places behind the range
#pragma unroll
    for (int i = 0; i < KEYS; ++i) f(key[i]);
    for (int j = lo + KEYS * kSelThreads + tid; j < hi; j += kSelThreads) f(key_of(j));
  };
  // ---- the key of rank `middle`, by histograms over ranges of keys that shrink by kBins a round. The first range
  // is that of the keys themselves, not of all 32-bit numbers: sums of attention weights span a few dozen exponents, and
  // a key is about the logarithm of its sum, so kBins equal steps spread them thinly where fixed digits would
  // pile them up in a few bins and their counting in a few words of shared memory.
  uint32_t base = 0xffffffffu, top = 0;
  each_key([&](uint32_t k) {
    base = min(base, k - 1);  // 0 is left out
    top = max(top, k);
  });
  base = __reduce_min_sync(0xffffffffu, base);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) {
    range[0][warp] = base;
    range[1][warp] = top;
  }
  for (int i = tid; i < kBins; i += kSelThreads) bins[i] = 0;
  __syncthreads();
  base = __reduce_min_sync(0xffffffffu, range[0][lane & (kWarps - 1)]) + 1;
  top = __reduce_max_sync(0xffffffffu, range[1][lane & (kWarps - 1)]);
  int want = middle, ties = 0;  // rank inside the range; in the end: how many of the keys equal to the threshold stay
  uint32_t threshold;           // keys above it stay
  while (true) {
    const int shift = max(32 - __clz(top - base) - kBinBits, 0);
    each_key([&](uint32_t k) {
      if (k - base <= top - base) atomicAdd(&bins[(k - base) >> shift], 1);
    });
    __syncthreads();
    // a thread's four bins, largest keys first, scanned over the CTA
    const int4 c = *reinterpret_cast<const int4*>(&bins[kBins - 4 * (tid + 1)]);
    const int mine = c.x + c.y + c.z + c.w;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    *reinterpret_cast<int4*>(&bins[kBins - 4 * (tid + 1)]) = make_int4(0, 0, 0, 0);  // for the next round
    int above = incl - mine + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
    if (above < want && want <= above + mine) {
      int bin = kBins - 1 - 4 * tid, n = c.w;
      if (above + n < want) { above += n; --bin; n = c.z; }
      if (above + n < want) { above += n; --bin; n = c.y; }
      if (above + n < want) { above += n; --bin; n = c.x; }
      found[0] = bin;
      found[1] = above;
      found[2] = n;
    }
    __syncthreads();
    const uint32_t low = base + (static_cast<uint32_t>(found[0]) << shift);
    want -= found[1];
    if (found[2] == want) {  // all of the bin stays
      threshold = low - 1;
      break;
    }
    if (shift == 0) {  // one value, more often than it is wanted
      threshold = low;
      ties = want;
      break;
    }
    base = low;
    top = low + min(top - low, (1u << shift) - 1);  // the bin's end may lie behind the last 32-bit number
  }

  // ---- keys above the threshold stay, and the first `ties` of those equal to it. Where a kept token goes follows from how
  // many stay before it: per slab of 512 tokens and warp the counts are taken from ballots, scanned once over all of
  // them by one warp, and added to the place inside the warp.
  int done_strict = 0, done_tie = 0;  // before this round of slabs
  const uint32_t below = (1u << lane) - 1;
  for (int j0 = lo; j0 < hi; j0 += KEYS * kSelThreads) {
    if (j0 > lo) load_keys(j0);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const uint32_t bs = __ballot_sync(0xffffffffu, key[i] > threshold), bt = ties ? __ballot_sync(0xffffffffu, key[i] == threshold) : 0u;
      if (lane == 0) slab[i * kWarps + warp] = __popc(bs) | __popc(bt) << 16;
    }
    __syncthreads();
    if (warp == 0) {
      constexpr int kPer = (KEYS * kWarps + 31) / 32;
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine += slab[lane * kPer + i];  // at most 512 KEYS <= 32768 per half: no carry
      uint32_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      uint32_t run = incl - mine;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t t = slab[lane * kPer + i];
        slab[lane * kPer + i] = run;
        run += t;
      }
      if (lane == 31) slab_all = run;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const bool strict = key[i] > threshold, tie = ties && key[i] == threshold;
      const uint32_t bs = __ballot_sync(0xffffffffu, strict), bt = ties ? __ballot_sync(0xffffffffu, tie) : 0u;
      const uint32_t before = slab[i * kWarps + warp];
      const int s = done_strict + static_cast<int>(before & 0xffffu) + __popc(bs & below);
      const int t = done_tie + static_cast<int>(before >> 16) + __popc(bt & below);
      const int j = j0 + i * kSelThreads + tid;
      if (strict || (tie && t < ties)) kept[lo + s + min(t, ties)] = j;
    }
    done_strict += slab_all & 0xffffu;
    done_tie += slab_all >> 16;
    __syncthreads();
  }
  carry_sums();
}

// ROWS: (token, head) rows of K and of V per CTA.
// The last and the first tokens of a request stay whatever their sums are: their rows come first in the grid, all requests'
// before any other row, and are copied while the selection runs (it is latency bound and leaves the memory idle; 500 of 2048 tokens: 99 -> 92 us). The
// selection lets this kernel start only once what precedes it is done, and writes nothing that is read before the wait.
template <int ROWS>
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p) {
  __shared__ long long src_off[ROWS], dst_off[ROWS];  // in 16-byte chunks; dst < 0: no such page
  const int b = static_cast<int>(blockIdx.x) % p.batch;
  const Request r = request_of(p, b);
  const int first = min(p.sinks, r.keep), tail = min(p.recent, r.keep - first);
  const long long rows = static_cast<long long>(r.keep) * p.hkv;  // (token, head), heads innermost; the last `tail` tokens in front
  const long long r0 = static_cast<long long>(blockIdx.x / p.batch) * ROWS;
  const int here = static_cast<int>(max(min(static_cast<long long>(ROWS), rows - r0), 0LL));
  // the grid's last CTA always waits: the kernel must not be done before the selection is
  if (r0 + here > static_cast<long long>(first + tail) * p.hkv || blockIdx.x == gridDim.x - 1) pdl_wait();
  if (here == 0) return;
  for (int x = threadIdx.x; x < here; x += kCopyThreads) {
    const int t = static_cast<int>((r0 + x) / p.hkv), h = static_cast<int>((r0 + x) % p.hkv);
    const int i = t < tail ? r.keep - tail + t : t - tail;
    const int j = t < tail ? r.n - tail + t : i < first ? i : __ldcg(p.kept + (static_cast<size_t>(b) * p.hkv + h) * p.budget + i);
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
  // token counts, and places up to a few blocks of threads behind them, are held in 32 bits
  constexpr long long kMost = 1LL << 30;
  if (static_cast<long long>(a->num_kv_indices) * a->page_size > kMost || a->max_len > kMost || a->budget > kMost || a->head_dim > 65536)
    return CB200_ERR_UNSUPPORTED;
  // Small CTAs where the rows would not give every SM several large ones (one request of 512 tokens and 8 heads).
  const long long rows = static_cast<long long>(a->budget) * a->num_kv_heads;
  const int copy_rows = rows * a->batch >= 128LL * 4 * 148 ? 128 : 32;
  const long long copy_ctas = (rows + copy_rows - 1) / copy_rows;
  if (copy_ctas * a->batch >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
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
  p.batch = a->batch;
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
  // enough registers for the longest request that the sums or the page table can hold
  const long long longest = static_cast<long long>(a->num_kv_indices) * a->page_size;
  const long long guess = longest < a->max_len ? longest : a->max_len;
  auto select = guess <= 4 * kSelThreads ? evict_select_kernel<4> : guess <= 16 * kSelThreads ? evict_select_kernel<16> : evict_select_kernel<kKeysMost>;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, select, p));
  cfg.gridDim = dim3(static_cast<unsigned>(copy_ctas * a->batch), 1, 1);
  cfg.blockDim = dim3(kCopyThreads, 1, 1);
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, copy_rows == 128 ? evict_copy_kernel<128> : evict_copy_kernel<32>, p));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}
