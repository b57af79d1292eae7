// Decode attention over a sliding window with sinks, and decode that accumulates attention weights: entry points
// over the modes of the kernel in decode_attn.cuh, and the kernel that turns kept scores into weights.
//
// Measured (32 query and 8 kv heads of 128, graph replays): windows of 1004 tokens, 64 requests, 16-token pages 52.8 us, 4.9 TB/s;
// windows of 4160, 128 requests, 64-token pages 333 us, 6.1 TB/s; weights of 64 requests of 512 .. 8192 tokens, 16-token pages
// 224 .. 229 us, of which the second kernel takes 15.

#include "decode_attn.cuh"

#include <algorithm>

namespace cb200 {
namespace {

// weight_sums[b, h, j] += sum over the kv head's query heads g of 2^(x_gj - lse_g), x the score of the decode kernel in
// log2 units: the softmax weight that key j had in this step. A thread takes four keys of a (request, kv head), a block
// apart, and a few heads at a time: every load is a warp's run of 128 bytes, and up to sixteen are in flight. A sum has
// one owner and its heads are added in their order, so the result does not depend on the launch. Bound by the stream of
// scores (written a moment ago, partly still in L2) and sums. A row whose scores are all -inf has no weights: it adds nothing.
constexpr int kSumThreads = 256, kSumKeys = 4;

__device__ __forceinline__ void sum_block(const DecodeParams& p, float* __restrict__ sums, int max_len, int pair, int block) {
  const int b = pair / p.hkv;
  const int n = min(item_valid_len(p, b), p.raw_len);
  const long long j0 = static_cast<long long>(block) * (kSumThreads * kSumKeys) + threadIdx.x;
  if (j0 >= n) return;
  const int j = static_cast<int>(j0), keys = min((n - j + kSumThreads - 1) / kSumThreads, kSumKeys);
  const size_t row = static_cast<size_t>(pair) * p.rows;
  const float* x = p.raw + row * p.raw_pitch + j;
  const float* lse = p.lse + row;
  float* dst = sums + static_cast<size_t>(pair) * max_len + j;
  float old[kSumKeys], w[kSumKeys];
#pragma unroll
  for (int i = 0; i < kSumKeys; ++i) {
    old[i] = i < keys ? dst[i * kSumThreads] : 0.f;
    w[i] = 0.f;
  }
#pragma unroll 4
  for (int g = 0; g < p.rows; ++g) {
    float l = __ldg(lse + g);
    if (l == -INFINITY) l = INFINITY;
    float v[kSumKeys];
#pragma unroll
    for (int i = 0; i < kSumKeys; ++i) v[i] = i < keys ? __ldcs(x + g * p.raw_pitch + i * kSumThreads) : -INFINITY;
#pragma unroll
    for (int i = 0; i < kSumKeys; ++i) w[i] += exp2f(v[i] - l);
  }
#pragma unroll
  for (int i = 0; i < kSumKeys; ++i)
    if (i < keys) dst[i * kSumThreads] = old[i] + w[i];
}

// `blocks` blocks of keys for each of `pairs` (request, kv head); the grid has a CTA for each of them, or fewer of either that
// WALK over them (the loops cost eight registers a thread: 1.2 us of 246 for 64 requests of up to 8192 tokens)
template <bool WALK>
__global__ void __launch_bounds__(kSumThreads) weight_sum_kernel(const DecodeParams p, float* __restrict__ sums, int max_len, int blocks, int pairs) {
  pdl_wait();
  if constexpr (WALK) {
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y)
      for (int block = blockIdx.x; block < blocks; block += gridDim.x) sum_block(p, sums, max_len, pair, block);
  } else {
    sum_block(p, sums, max_len, blockIdx.y, blockIdx.x);
  }
}

// Tokens whose scores are kept: no request is longer than the page table, however wide the accumulators are (a server
// that keeps room for its longest context would otherwise need scratch for that in every step).
long long raw_tokens(const cb200_attn_decode_args* a, int max_len) {
  const long long longest = static_cast<long long>(a->num_kv_indices) * a->page_size;
  return longest < max_len ? longest : max_len;
}
// floats between the score rows of two query heads: whole 32-byte runs
long long raw_pitch(long long tokens) { return (tokens + 7) / 8 * 8; }

}  // namespace
}  // namespace cb200

extern "C" int cb200_attn_decode_window(const cb200_attn_decode_args* a, int window, int sinks, void* stream) {
  using namespace cb200;
  if (!a || !a->kv_indptr || window <= 0 || sinks < 0) return CB200_ERR_BAD_ARG;
  if (a->q_rows > 1) return CB200_ERR_UNSUPPORTED;  // the window is that of one query, the request's last token
  DecodeSetup s;
  const int rc = plan_decode(a, &s, true, true);
  if (rc != CB200_OK) return rc;
  s.p.window = window;
  s.p.sinks = sinks;
  return launch_decode_mode<kWindow>(s, a, static_cast<cudaStream_t>(stream));
}

extern "C" size_t cb200_attn_decode_weights_scratch_bytes(const cb200_attn_decode_args* a, int max_len) {
  if (!a || a->batch <= 0 || a->num_qo_heads <= 0 || max_len <= 0 || a->num_kv_indices < 0 || a->page_size < 0) return 0;
  return static_cast<size_t>(a->batch) * a->num_qo_heads * cb200::raw_pitch(cb200::raw_tokens(a, max_len)) * sizeof(float);
}

extern "C" int cb200_attn_decode_weights(const cb200_attn_decode_args* a, float* weight_sums, int max_len, void* scratch,
                                         size_t scratch_bytes, void* stream) {
  using namespace cb200;
  if (!a || !a->kv_indptr || !a->lse || !weight_sums || max_len <= 0) return CB200_ERR_BAD_ARG;
  if (a->q_rows > 1) return CB200_ERR_UNSUPPORTED;
  DecodeSetup s;
  const int rc = plan_decode(a, &s, true, true);
  if (rc != CB200_OK) return rc;
  const long long pairs = static_cast<long long>(a->batch) * a->num_kv_heads;
  if (pairs > 65535) return CB200_ERR_UNSUPPORTED;
  const size_t need = cb200_attn_decode_weights_scratch_bytes(a, max_len);
  if (need > 0 && (!scratch || scratch_bytes < need)) return CB200_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(scratch) & 31) || (reinterpret_cast<uintptr_t>(weight_sums) & 3)) return CB200_ERR_ALIGNMENT;
  s.p.raw = static_cast<float*>(scratch);
  const long long tokens = raw_tokens(a, max_len);
  s.p.raw_len = static_cast<int>(tokens);
  s.p.raw_pitch = raw_pitch(tokens);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int done = launch_decode_mode<kWeights>(s, a, st);
  if (done != CB200_OK || tokens == 0) return done;
  cudaLaunchConfig_t cfg = {};
  const int blocks = static_cast<int>((tokens + kSumKeys * kSumThreads - 1) / (kSumKeys * kSumThreads));
  int grid_x = blocks, grid_y = static_cast<int>(pairs);
  if (bounded(a)) {
    grid_x = std::min(grid_x, a->max_ctas);
    grid_y = std::min(grid_y, a->max_ctas / grid_x);
  }
  cfg.gridDim = dim3(static_cast<unsigned>(grid_x), static_cast<unsigned>(grid_y), 1);
  cfg.blockDim = dim3(kSumThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = bounded(a) ? 0 : 1;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, bounded(a) ? weight_sum_kernel<true> : weight_sum_kernel<false>, s.p, weight_sums, max_len, blocks, static_cast<int>(pairs)));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}
