// C ABI entry points of the projections (include/kmoe.h): the argument check
// (linear_host.cpp, no HIP call), the device check, then the launches.
#include "linear_launch.h"

using namespace kmoe_host;

namespace {

kmoe_status launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return KMOE_OK;
  return fail(KMOE_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

}  // namespace

extern "C" {

kmoe_status kmoe_linear_pack_bytes(const kmoe_linear_weight* packed, size_t* values_bytes, size_t* scale_bytes) {
  return validate_linear_pack_bytes(packed, values_bytes, scale_bytes);
}

kmoe_status kmoe_linear_pack(const kmoe_weight* w, const kmoe_linear_weight* packed, void* stream) {
  KMOE_TRY(validate_linear_pack(w, packed));
  KMOE_TRY(kmoe_device_check());
  return launched(launch_linear_pack(*w, *packed, (hipStream_t)stream), "linear pack kernel");
}

kmoe_status kmoe_lora_pack_bytes(const kmoe_lora* lora, size_t* a_bytes, size_t* b_bytes) {
  return validate_lora_pack_bytes(lora, a_bytes, b_bytes);
}

kmoe_status kmoe_lora_pack(const kmoe_lora* lora, int64_t first, int64_t count, int64_t rank, const void* a,
                           const void* b, const float* factor, void* stream) {
  KMOE_TRY(validate_lora_pack(lora, first, count, rank, a, b, factor));
  KMOE_TRY(kmoe_device_check());
  if (count == 0) return KMOE_OK;
  return launched(launch_lora_pack(*lora, first, count, rank, a, b, factor, (hipStream_t)stream),
                  "adapter pack kernels");
}

kmoe_status kmoe_lora_sort_bytes(const kmoe_lora_batch* batch, size_t* bytes) {
  return validate_lora_sort_bytes(batch, bytes);
}

kmoe_status kmoe_lora_sort(const int32_t* adapter, const kmoe_lora_batch* batch, void* scratch, size_t scratch_bytes,
                           void* stream) {
  KMOE_TRY(validate_lora_sort(adapter, batch, scratch, scratch_bytes));
  KMOE_TRY(kmoe_device_check());
  if (batch->tokens == 0) return KMOE_OK;
  return launched(launch_lora_sort(adapter, *batch, scratch, (hipStream_t)stream), "adapter sort kernels");
}

kmoe_status kmoe_linear_workspace_bytes(const kmoe_linear_weight* w, int64_t tokens, kmoe_dtype x_dtype,
                                        const kmoe_lora* lora, size_t* bytes) {
  return validate_linear_workspace_bytes(w, tokens, x_dtype, lora, bytes);
}

kmoe_status kmoe_linear_call_bytes(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                                   int64_t x_stride, const kmoe_lora* lora, size_t* bytes) {
  return validate_linear_call_bytes(w, tokens, x, x_dtype, x_stride, lora, bytes);
}

kmoe_status kmoe_linear(const kmoe_linear_weight* w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                        int64_t x_stride, const float* x_scale, const kmoe_lora* lora, const kmoe_lora_batch* batch,
                        void* out, void* workspace, size_t workspace_bytes, void* stream) {
  LinearSpace space;
  KMOE_TRY(validate_linear(w, tokens, x, x_dtype, x_stride, x_scale, lora, batch, out, workspace, workspace_bytes,
                           &space));
  KMOE_TRY(kmoe_device_check());
  if (tokens == 0) return KMOE_OK;
  KMOE_TRY(validate_linear_apart(*w, tokens, x, x_dtype, x_stride, out, workspace, space));
  return launched(launch_linear(*w, tokens, x, x_dtype, x_stride, x_scale, lora, batch, out, workspace, space,
                                (hipStream_t)stream),
                  "linear kernels");
}

}  // extern "C"
