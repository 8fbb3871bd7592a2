// A block whose waits run out, or end: what the kernels of the linear attention do around theirs (test_gpu_attention_waits.py).
#include "decay_attn.cuh"

using namespace bcm::decay_attn;

// `arrive`: whether anything arrives at the barriers.  told: threads that learn of a lost wait
__global__ void __launch_bounds__(256) wait_kernel(bool arrive, float* out, int64_t stride, int rows, int cols, int* told) {
    __shared__ Sync<3> sync;
    sync.init(32);
    if (arrive && threadIdx.x == 0)
        for (int i = 0; i < 3; ++i)
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bcm::t5::smem_u32(&sync.bars[i])) : "memory");
    sync.wait(threadIdx.x >> 5 & 1, 0);
    if (sync.lost()) {
        atomicAdd(told, 1);
        nan_rows(out, stride, rows, cols);
    }
    if (threadIdx.x == 0) out[-1] += sync.poison();           // (a float before the rows)
    sync.end(32);
}

extern "C" __attribute__((visibility("default"))) int run_wait(int arrive, float* out, int64_t stride, int rows, int cols, int* told, void* stream) {
    wait_kernel<<<1, 256, 0, (cudaStream_t)stream>>>(arrive != 0, out, stride, rows, cols, told);
    return (int)cudaGetLastError();
}
