// What launches share.
#pragma once

#include <cuda_runtime.h>

#include <stddef.h>

namespace b200q {

// Lets a kernel have `smem` bytes of dynamic shared memory on the current device; asked for again only where it is more than before
inline cudaError_t configure_smem(const void *kern, size_t smem) {
    struct Done {
        const void *kern;
        int device;
        size_t smem;
    };
    static thread_local Done done[32];       // this thread's last ones
    static thread_local unsigned next = 0;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    Done *mine = nullptr;
    for (Done &d : done)
        if (d.kern == kern && d.device == device) mine = &d;
    if (mine && mine->smem >= smem) return cudaSuccess;
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return e;
    if (!mine) mine = &done[next++ % 32];
    *mine = Done{kern, device, smem};
    return cudaSuccess;
}

}  // namespace b200q
