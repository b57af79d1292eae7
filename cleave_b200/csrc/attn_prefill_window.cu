// Causal prefill over a sliding window with sinks, ragged or paged (the kernel: attn_prefill_tc.cuh, WIN).

#include "attn_prefill_tc.cuh"

extern "C" int cb200_attn_prefill_ragged_window(const cb200_attn_prefill_ragged_args* a, int window, int sinks, int fill, void* stream) {
  using namespace cb200;
  const int rc = plan_prefill_ragged(a);
  if (rc != CB200_OK) return rc;
  if (window <= 0 || sinks < 0 || fill < 0 || fill > 3) return CB200_ERR_BAD_ARG;
  const int prc = check_prefill_ragged_pointers(a);
  if (prc != CB200_OK) return prc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = a->dtype == CB200_F16;
  if (a->head_dim == 64)
    return f16 ? launch_prefill_ragged<__half, 64, true>(a, window, sinks, fill, st) : launch_prefill_ragged<__nv_bfloat16, 64, true>(a, window, sinks, fill, st);
  return f16 ? launch_prefill_ragged<__half, 128, true>(a, window, sinks, fill, st) : launch_prefill_ragged<__nv_bfloat16, 128, true>(a, window, sinks, fill, st);
}
