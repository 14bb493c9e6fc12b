// Memory -> LDS past the registers, 16 bytes or one word per lane, of all lanes one after the other from `to` on, which is uniform. The compiler's form of it waits for all loads ahead of each
// transposing read of LDS (mix_blocks.hip: 149 us instead of 135); this one is waited for by its user, by the number of loads, ahead of the barrier behind which the values are read. What
// stands in M0 and in the scalar address has to have been there for a while: one wait state from a write of M0 to a load into LDS, and five from a vector instruction's write of a scalar
// register (v_readfirstlane) to a memory instruction that reads it. The compiler keeps them for its own instructions and does not look into these, so they keep both themselves.
#pragma once
#include "columns.h"

namespace tfno {

__device__ __forceinline__ unsigned place_in_lds(const void* p) { return (unsigned)(unsigned long)(__attribute__((address_space(3))) const char*)p; }
__device__ __forceinline__ void direct_to_lds(ScalarAddress base, unsigned offset, unsigned to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to)) : "m0", "memory");
}
__device__ __forceinline__ void direct_word_to_lds(ScalarAddress base, unsigned offset, unsigned to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dword %0, %1" : : "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to)) : "m0", "memory");
}

}  // namespace tfno
