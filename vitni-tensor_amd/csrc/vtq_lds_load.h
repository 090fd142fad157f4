// vtq_lds_load.h -- loads from memory straight into LDS, and the waits that order
// them (gfx950).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vtq {

typedef __attribute__((address_space(3))) uint8_t lds_u8;

// One buffer load straight into LDS: lane L's SIZE bytes (16 or 4) from
// buffer offset voff land at LDS byte lds_addr + SIZE * L.  Written as asm
// so that the compiler does not track it: it would otherwise wait for every
// such load (vmcnt(0)) before the first barrier or LDS read.  The kernel
// orders these loads itself with explicit vmcnt waits and barriers; the
// hardware completes loads in order, so the compiler's own waits on any
// later load stay correct.  m0 is a reserved register: the compiler keeps
// no value of its own in it in these kernels and does not honour it on a
// clobber list (it only warns), so it is not listed; tests/test_asm_checks.py and
// tests/test_serve_asm.py check the generated code of every kernel with such loads
// for any other use of m0.
template <int SIZE>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t lds_addr) {
    static_assert(SIZE == 16 || SIZE == 4, "dwordx4 or dword");
    if constexpr (SIZE == 16)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                     :
                     : "v"(voff), "s"(rs), "s"(lds_addr)
                     : "memory");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
                     :
                     : "v"(voff), "s"(rs), "s"(lds_addr)
                     : "memory");
}

// s_waitcnt vmcnt(N) alone (gfx9 encoding: vmcnt in bits 3:0 and 15:14, expcnt
// and lgkmcnt left at their maxima, so nothing else is waited for)
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

}  // namespace vtq
