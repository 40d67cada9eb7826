// 16-byte asynchronous copies global -> LDS: lane l writes LDS byte address
// lds + 16 l, lds the same in all lanes (the instruction takes it from m0). The
// compiler's wait counts do not know them: readers wait with an s_waitcnt vmcnt of
// their own. Nor does it pad inside an asm block: a copy takes m0 one wait state after
// it is written, hence the s_nop.
#pragma once
#include <hip/hip_runtime.h>

// From an address a lane.
__device__ __forceinline__ void kr_copy16(const void* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds), "v"(src) : "memory", "m0");
}

// From an address that all lanes share and a byte offset a lane. The address may come
// from a v_readfirstlane just before: five wait states until the copy reads it.
__device__ __forceinline__ void kr_copy16(const void* base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
