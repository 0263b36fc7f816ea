// The norms' backward for callers within the library.
#pragma once

#include "capi.hpp"

namespace dabsn {
namespace norm {

// dabsn_hip_norm_bwd whose gradient has type gdtype: dtype's, or fp32 where there are rows to add.
int backward(int dtype, int wdtype, int gdtype, int layer, int64_t rows, int64_t H, const void* x, int64_t ldx,
             const void* weight, const float* stats, const void* grad, int64_t ldg, const void* add, void* dx,
             void* dweight, void* dbias, void* workspace, size_t workspace_bytes, hipStream_t stream);

}  // namespace norm
}  // namespace dabsn
