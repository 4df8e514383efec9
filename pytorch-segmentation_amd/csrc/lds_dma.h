// Global -> LDS copies without a register in between (buffer_load_dwordx4 ... offen lds), shared by the MFMA kernels.
// A wave-instruction deposits 64 lanes x 16 B = 1 KiB lane-linearly at the LDS address in M0; byte offsets beyond the descriptor's
// range write ZEROS to LDS.  Issued from inline asm: hipcc does not count asm memory operations, so it puts no s_waitcnt vmcnt(0)
// between the copies of stage t+1 and the ds_reads of stage t; the kernels wait themselves (one vmcnt(0) + barrier per stage).
// No register is written, so nothing the compiler could reuse is in flight.  M0 is written in the statement that consumes it.
#pragma once
#include <hip/hip_runtime.h>

typedef __attribute__((address_space(3))) void lds_void;
typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 make_rsrc(const void* base, unsigned bytes) {
    const unsigned long long a = (unsigned long long)base;
    i32x4 r;
    r.x = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
    r.y = __builtin_amdgcn_readfirstlane((int)((unsigned)(a >> 32) & 0xFFFFu));   // stride 0, no swizzle
    r.z = __builtin_amdgcn_readfirstlane((int)bytes);                              // num_records (bytes)
    r.w = 0x00020000;                                                              // raw buffer, 32-bit data format
    return r;
}
__device__ __forceinline__ unsigned lds_addr(const void* p) { return (unsigned)(unsigned long long)(lds_void*)p; }
// lane's bytes at rsrc.base + voffset + soffset (soffset is wave-uniform)
__device__ __forceinline__ void dma16s(const i32x4& rsrc, unsigned voffset, unsigned soffset, unsigned lds_dst) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :: "v"(voffset), "s"(rsrc), "s"(soffset), "s"(lds_dst) : "memory");
}
