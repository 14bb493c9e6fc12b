// Loads into LDS (turbofno_amd/csrc/direct_lds.h) whose place and scalar address are made right ahead of them: for a look at the assembly.
#include "../../turbofno_amd/csrc/direct_lds.h"

__global__ void direct_lds_check(const char* x, const int* from, float* y)
{
    extern __shared__ float lds[];
#pragma unroll
    for (int i = 0; i < 4; ++i) tfno::direct_to_lds(tfno::scalar(x, from[threadIdx.x + 64 * i]), threadIdx.x * 16, tfno::place_in_lds(lds) + from[i]);
    tfno::direct_word_to_lds(tfno::scalar(x, from[threadIdx.x]), threadIdx.x * 4, tfno::place_in_lds(lds) + 8192);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    y[threadIdx.x] = lds[threadIdx.x];
}
