// gradients.h -- the norm and clipping of many tensors (gradients.hip).
#pragma once

#include "gs_internal.h"

namespace gs {

using ClipTensor = gsplat_clip_tensor;

size_t clip_workspace_bytes(const ClipTensor* x, int64_t count);
int launch_clip(const ClipTensor* x, int64_t count, double max_norm, float* norm,
                void* workspace, hipStream_t stream);

}  // namespace gs
