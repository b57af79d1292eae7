// Entry points of attention with many query rows (the kernel: attn_prefill_tc.cuh), and the row normalisation ahead of it.

#include "attn_prefill_tc.cuh"

namespace cb200 {
namespace fa {

// RMS-normalises rows of D elements, one warp per row: y = x * rsqrt(mean(x^2) + eps), fp32 statistics,
// result in the storage type. Used on K ahead of the attention kernel for demo/qknorm.py (K is the small
// operand: it is read by every query tile, so it is normalised once instead of per tile).
template <typename T, int D>
__global__ void __launch_bounds__(256) rms_rows_kernel(const T* __restrict__ x, T* __restrict__ y, long long rows, float eps) {
  constexpr int kPer = D / 32;  // 2 or 4 elements per lane
  const int lane = threadIdx.x & 31;
  const long long stride = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long r = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); r < rows; r += stride) {
    T e[kPer];
    if constexpr (kPer == 4) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(x + r * D + lane * 4);
    else *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(x + r * D + lane * 2);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float f = static_cast<float>(e[i]);
      ss = fmaf(f, f, ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float f = rsqrtf(ss * (1.f / D) + eps);
#pragma unroll
    for (int i = 0; i < kPer; ++i) e[i] = static_cast<T>(static_cast<float>(e[i]) * f);
    if constexpr (kPer == 4) *reinterpret_cast<uint2*>(y + r * D + lane * 4) = *reinterpret_cast<const uint2*>(e);
    else *reinterpret_cast<uint32_t*>(y + r * D + lane * 2) = *reinterpret_cast<const uint32_t*>(e);
  }
}

}  // namespace fa

namespace {

int plan_prefill(const cb200_attn_prefill_args* a) {
  if (!a) return CB200_ERR_BAD_ARG;
  if (a->num_qo_heads <= 0 || a->num_kv_heads <= 0 || a->q_len <= 0 || a->kv_len <= 0) return CB200_ERR_BAD_ARG;
  if (a->num_qo_heads % a->num_kv_heads) return CB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return CB200_ERR_UNSUPPORTED;
  if (a->dtype != CB200_F16 && a->dtype != CB200_BF16) return CB200_ERR_UNSUPPORTED;
  const long long ctas = static_cast<long long>(a->num_qo_heads) * ceil_div(a->q_len, fa::kBM);
  if (ctas >= (1LL << 31)) return CB200_ERR_UNSUPPORTED;
  if (a->score_mode != CB200_SCORE_SOFTMAX && a->score_mode != CB200_SCORE_LINEAR) return CB200_ERR_BAD_ARG;
  if (a->qk_norm && !(a->norm_eps >= 0.f)) return CB200_ERR_BAD_ARG;
  return CB200_OK;
}

// bytes of the normalised copy of K that follows the status header when qk_norm is set
size_t prefill_knorm_bytes(const cb200_attn_prefill_args* a) {
  if (!a->qk_norm) return 0;
  return static_cast<size_t>(a->num_kv_heads) * a->kv_len * a->head_dim * 2;
}

template <typename T, int D>
int launch_prefill(const cb200_attn_prefill_args* a, cudaStream_t stream) {
  using namespace fa;
  Params p{};
  p.out = a->out;
  p.lse = a->lse;
  p.status = reinterpret_cast<int*>(a->workspace);
  p.hq = a->num_qo_heads;
  p.hkv = a->num_kv_heads;
  p.sq = a->q_len;
  p.skv = a->kv_len;
  p.q_tiles = ceil_div(a->q_len, kBM);
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->sm_scale * kLog2e;
  p.linear = a->score_mode == CB200_SCORE_LINEAR ? 1 : 0;
  p.scale = a->sm_scale;
  p.q_norm = a->qk_norm ? 1 : 0;
  p.norm_eps = a->norm_eps;
  const void* k_src = a->k;
  if (a->qk_norm) {
    T* kn = reinterpret_cast<T*>(static_cast<uint8_t*>(a->workspace) + kWsHeaderBytes);
    const long long rows = static_cast<long long>(a->num_kv_heads) * a->kv_len;
    const int blocks = static_cast<int>(std::min<long long>((rows + 7) / 8, 148LL * 8));
    rms_rows_kernel<T, D><<<blocks, 256, 0, stream>>>(reinterpret_cast<const T*>(a->k), kn, rows, a->norm_eps);
    CB200_CUDA_TRY(cudaGetLastError());
    k_src = kn;
  }
  const CUtensorMapDataType dt = a->dtype == CB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tm_q, tm_k, tm_v;
  {
    uint32_t box[3] = {64u, 128u, 1u};
    uint64_t dq[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->q_len), static_cast<uint64_t>(a->num_qo_heads)};
    uint64_t sq[2] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(a->q_len) * D * 2};
    uint64_t dk[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a->kv_len), static_cast<uint64_t>(a->num_kv_heads)};
    uint64_t sk[2] = {static_cast<uint64_t>(D) * 2, static_cast<uint64_t>(a->kv_len) * D * 2};
    const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
    if (!encode_tensor_map(&tm_q, dt, 3, const_cast<void*>(a->q), dq, sq, box, sw) ||
        !encode_tensor_map(&tm_k, dt, 3, const_cast<void*>(k_src), dk, sk, box, sw) ||
        !encode_tensor_map(&tm_v, dt, 3, const_cast<void*>(a->v), dk, sk, box, sw))
      return CB200_ERR_CUDA;
  }
  // one CTA per SM at most, and then the CTAs deal the (head, query tile) items among themselves; with no more items
  // than SMs every item has its own CTA and the kernel's one-item form runs
  const long long n_items = static_cast<long long>(p.hq) * p.q_tiles;
  const bool persist = n_items > sm_count();
  auto kern = persist ? attn_prefill_kernel<T, D, 0, true> : attn_prefill_kernel<T, D, 0, false>;
  CB200_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmemBytes));
  const unsigned grid = static_cast<unsigned>(std::min<long long>(n_items, sm_count()));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<D>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  // scheduled while the preceding kernel of the stream drains; the kernel waits before its first global access
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  CB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm_q, tm_k, tm_v, p));
  CB200_CUDA_TRY(cudaGetLastError());
  return CB200_OK;
}

}  // namespace
}  // namespace cb200

extern "C" size_t cb200_attn_prefill_workspace_bytes(const cb200_attn_prefill_args* a) {
  return cb200::plan_prefill(a) == CB200_OK ? cb200::kWsHeaderBytes + cb200::prefill_knorm_bytes(a) : 0;
}

extern "C" int cb200_attn_prefill(const cb200_attn_prefill_args* a, void* stream) {
  using namespace cb200;
  const int rc = plan_prefill(a);
  if (rc != CB200_OK) return rc;
  if (!a->q || !a->k || !a->v || !a->out) return CB200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
       reinterpret_cast<uintptr_t>(a->out)) & 15)
    return CB200_ERR_ALIGNMENT;
  if (!a->workspace || a->workspace_bytes < kWsHeaderBytes + prefill_knorm_bytes(a)) return CB200_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = a->dtype == CB200_F16;
  if (a->head_dim == 64)
    return f16 ? launch_prefill<__half, 64>(a, st) : launch_prefill<__nv_bfloat16, 64>(a, st);
  return f16 ? launch_prefill<__half, 128>(a, st) : launch_prefill<__nv_bfloat16, 128>(a, st);
}

extern "C" size_t cb200_attn_prefill_ragged_workspace_bytes(const cb200_attn_prefill_ragged_args* a) {
  return cb200::plan_prefill_ragged(a) == CB200_OK ? cb200::kWsHeaderBytes : 0;
}

extern "C" int cb200_attn_prefill_ragged(const cb200_attn_prefill_ragged_args* a, void* stream) {
  using namespace cb200;
  const int rc = plan_prefill_ragged(a);
  if (rc != CB200_OK) return rc;
  const int prc = check_prefill_ragged_pointers(a);
  if (prc != CB200_OK) return prc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    // A key window far shorter than the run of query rows: only the last min(q_len, kv_len) rows of a request see a
    // key, the rest are written as 0 / -inf, and two light kernels do both faster than a CTA per tile of 128 rows.
    const int keys = a->kv_indices ? a->num_kv_indices : a->total_kv;
    if (a->causal && small_prefill_applies(keys, a->total_q))
      return launch_small_gqa(a->q, a->k, a->v, a->qo_indptr, a->kv_indptr, a->kv_indices, a->out, a->lse, a->batch, a->total_q,
                              a->num_qo_heads, a->num_kv_heads, a->head_dim, a->kv_indices ? a->total_kv : 0, keys, a->sm_scale,
                              a->dtype, st);
  }
  const bool f16 = a->dtype == CB200_F16;
  if (a->head_dim == 64)
    return f16 ? launch_prefill_ragged<__half, 64, false>(a, 0, 0, 0, st) : launch_prefill_ragged<__nv_bfloat16, 64, false>(a, 0, 0, 0, st);
  return f16 ? launch_prefill_ragged<__half, 128, false>(a, 0, 0, 0, st) : launch_prefill_ragged<__nv_bfloat16, 128, false>(a, 0, 0, 0, st);
}
