// Launch wrappers of the projections (linear.hip) for the entry points in linear_api.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "linear.h"

namespace kmoe_host {

hipError_t launch_linear_pack(const kmoe_weight& w, const kmoe_linear_weight& packed, hipStream_t st);
hipError_t launch_lora_pack(const kmoe_lora& l, int64_t first, int64_t count, int64_t rank, const void* a,
                            const void* b, const float* factor, hipStream_t st);
hipError_t launch_lora_sort(const int32_t* adapter, const kmoe_lora_batch& b, void* scratch, hipStream_t st);
// workspace: linear_space(...).total bytes
hipError_t launch_linear(const kmoe_linear_weight& w, int64_t tokens, const void* x, kmoe_dtype x_dtype,
                         int64_t x_stride, const float* x_scale, const kmoe_lora* lora, const kmoe_lora_batch* batch,
                         void* out, void* workspace, const LinearSpace& space, hipStream_t st);

}  // namespace kmoe_host
