// The mixture-of-experts kernels (moe_kernels.cuh) for experts in LL_W_BF16.
#include <algorithm>

#include "moe_kernels.cuh"

namespace llk {

int launch_moe_bf16(MoeParams &p, int device, cudaStream_t st)
{
    return launch_moe<LL_W_BF16>(p, device, st);
}

}  // namespace llk
