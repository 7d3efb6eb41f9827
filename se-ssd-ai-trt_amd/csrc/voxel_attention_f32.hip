// voxel_attention_f32.hip -- the kernel of voxel_attention.h for FP32 tensors.
#include "voxel_attention.h"

namespace sessd {

int launch_attention_float(const AttentionArgs& a, hipStream_t stream) {
    if (a.dim <= 16) launch_attention_dim<float, 16, 64>(a, stream);
    else if (a.dim <= 32) launch_attention_dim<float, 32, 64>(a, stream);
    else if (a.dim <= 64) launch_attention_dim<float, 64, 64>(a, stream);
    else launch_attention_dim<float, 128, 32>(a, stream);
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

}  // namespace sessd
