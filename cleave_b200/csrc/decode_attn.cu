// Entry points of decode attention over contiguous or paged caches (the kernel: decode_attn.cuh).

#include "decode_attn.cuh"

#include <mutex>

namespace cb200 {
namespace {

// Scratch for cb200_attn_decode_static_scratch: lives in the library's device image, so every GPU
// that loads the library holds these 4 MiB until the process exits.
constexpr size_t kStaticScratchBytes = size_t(4) << 20;
static __device__ __align__(256) unsigned char g_decode_static_scratch[kStaticScratchBytes];

// In host code the array's name is only a handle for the runtime, not a device address. The
// address is looked up once per device, with that device current, and cached.
int static_scratch_address(unsigned char** out) {
  static unsigned char* cached[64] = {nullptr};
  static std::mutex mu;
  int dev = 0;
  CB200_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && cached[dev]) {
    *out = cached[dev];
    return CB200_OK;
  }
  unsigned char* ptr = nullptr;
  CB200_CUDA_TRY(cudaGetSymbolAddress(reinterpret_cast<void**>(&ptr), g_decode_static_scratch));
  if (!ptr) return CB200_ERR_CUDA;
  if (dev < 64) cached[dev] = ptr;
  *out = ptr;
  return CB200_OK;
}

}  // namespace
}  // namespace cb200

extern "C" size_t cb200_attn_decode_static_scratch_max_bytes(void) { return cb200::kStaticScratchBytes; }

extern "C" int cb200_attn_decode_static_scratch(const cb200_attn_decode_args* a, void* stream) {
  using namespace cb200;
  DecodeSetup s;
  int rc = plan_decode(a, &s, false);
  if (rc != CB200_OK) return rc;
  if (s.ws_needed > kStaticScratchBytes) return CB200_ERR_SCRATCH_LIMIT;
  unsigned char* scratch = nullptr;
  rc = static_scratch_address(&scratch);
  if (rc != CB200_OK) return rc;
  cb200_attn_decode_args b = *a;
  b.workspace = scratch;
  b.workspace_bytes = kStaticScratchBytes;
  rc = plan_decode(&b, &s, true);
  if (rc != CB200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The array keeps whatever the previous call left behind; the status word and this call's
  // arrival counters must start at zero.
  CB200_CUDA_TRY(cudaMemsetAsync(scratch, 0, kWsHeaderBytes, st));
  CB200_CUDA_TRY(cudaMemsetAsync(scratch + s.counters_off, 0, s.ws_needed - s.counters_off, st));
  return launch_decode_mode<kPlain>(s, &b, st);
}

extern "C" int cb200_attn_decode_static_scratch_status(void* stream) {
  unsigned char* scratch = nullptr;
  const int rc = cb200::static_scratch_address(&scratch);
  if (rc != CB200_OK) return rc;
  return cb200_workspace_status(scratch, stream);
}

extern "C" size_t cb200_attn_decode_workspace_bytes(const cb200_attn_decode_args* a) {
  cb200::DecodeSetup s;
  if (cb200::plan_decode(a, &s, false) != CB200_OK) return 0;
  return s.ws_needed;
}

extern "C" int cb200_attn_decode(const cb200_attn_decode_args* a, void* stream) {
  using namespace cb200;
  DecodeSetup s;
  const int rc = plan_decode(a, &s, true);
  if (rc != CB200_OK) return rc;
  return launch_decode_mode<kPlain>(s, a, static_cast<cudaStream_t>(stream));
}
