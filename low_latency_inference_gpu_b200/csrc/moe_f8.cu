// The mixture-of-experts kernels (moe_kernels.cuh) for experts in LL_W_F8.
#include <algorithm>

#include "moe_kernels.cuh"

namespace llk {

int launch_moe_f8(MoeParams &p, int device, cudaStream_t st)
{
    return launch_moe<LL_W_F8>(p, device, st);
}

}  // namespace llk
