// A wait of the tensor-core path that runs out: a phase that nothing completes. The waiting threads return, the block's other warps and the
// host are told, and the context serves the next launch.
#include <cstdio>

#include <cuda_runtime.h>

#include "../../oxidizr_b200/csrc/oxz_tcgen05.cuh"

__global__ void wait_for_nothing(int32_t* expired, int32_t* result, unsigned long long* ns) {
    __shared__ __align__(8) unsigned long long bars[2];
    __shared__ uint32_t dead;
    const uint32_t never = oxz::smem_u32(&bars[0]), done = oxz::smem_u32(&bars[1]);
    if (threadIdx.x == 0) {
        dead = 0;
        oxz::mbar_init(never, 1);
        oxz::mbar_init(done, 1);
    }
    __syncthreads();
    const oxz::WaitState w{&dead, expired};
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    // one thread of each of two warps waits, as in the products: the first to give up ends the other's wait
    const bool got = threadIdx.x % 32 ? true : oxz::mbar_wait(never, 0, w);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
    __syncthreads();
    if (threadIdx.x % 32 == 0) {
        result[threadIdx.x / 32] = got;
        ns[threadIdx.x / 32] = t1 - t0;
    }
    if (threadIdx.x == 0) result[2] = dead == 1;
    // a phase that is complete is found at once, also by a block that has given up before
    if (threadIdx.x == 0) {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(done) : "memory");
        result[3] = oxz::mbar_wait(done, 0, w);
    }
}

int main() {
    int32_t *expired, *result;
    unsigned long long* ns;
    if (cudaHostAlloc(&expired, 4, cudaHostAllocMapped) || cudaMallocManaged(&result, 16) || cudaMallocManaged(&ns, 16)) return 1;
    *expired = 0;
    int32_t* d_expired;
    if (cudaHostGetDevicePointer(&d_expired, expired, 0)) return 1;
    wait_for_nothing<<<1, 64>>>(d_expired, result, ns);
    const cudaError_t e = cudaDeviceSynchronize();
    if (e) {
        std::printf("error: %s\n", cudaGetErrorString(e));
        return 1;
    }
    std::printf("%d %d %d %d %d %.3f %.3f\n", result[0], result[1], result[2], result[3], *expired, ns[0] * 1e-9, ns[1] * 1e-9);
    return 0;
}
