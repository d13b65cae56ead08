// Loads from global memory straight into LDS, and the waits and barriers of
// kernels that keep several of them in flight (gemm.hip, gemm_fp8.hip).
#pragma once

#include "hip_util.hpp"

namespace aicf::hip {

// Buffer load straight into LDS (buffer_load_dwordx4 ... lds): lane i's 16
// bytes land at M0 + 16 i.  The LLVM intrinsic has no clang builtin; it is
// bound by name.  A buffer resource = 48-bit base, byte range (loads past it
// return zero), gfx9 format word.  Per-lane 32-bit offsets stay fixed for the
// whole K loop; the K advance is the scalar offset.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ void raw_buffer_load_lds(i32x4_t rsrc, __attribute__((address_space(3))) unsigned* lds,
                                    int size, int voffset, int soffset, int offset,
                                    int aux) __asm("llvm.amdgcn.raw.buffer.load.lds");
// The same load written as inline asm (M0 = LDS address, set by the
// compiler through the constraint).  The compiler's hazard recognizer does
// not see the vector-memory instruction inside the asm, so the asm covers the
// hazards of its scalar operands itself: a VMEM read of an SGPR that a VALU
// instruction wrote (v_readfirstlane / v_readlane into the resource words or
// the scalar offset) needs 5 wait states, and the M0 write one; s_nop 4
// provides 5.  (With s_nop 0 a build whose scheduler placed a
// v_readfirstlane of the resource base right before the asm ended in a GPU
// memory fault.)  PAD: the loads of a tile's first stages, which follow the
// resource set-up; the K loop's loads (scalar offsets from SALU adds) keep
// s_nop 0 for the M0 write, and codegen tests check every asm load's wait
// states against the VALU writes before it.
// The compiler does not know that it writes LDS, so it adds no vmcnt wait in
// front of the LDS reads that follow it: it cannot prove that a transposing
// ds_read_b64_tr_b16 does not alias an in-flight direct-to-LDS load, and
// with the intrinsic it waits for all loads before every such read.  The
// kernel orders every LDS read of a stage after that stage's loads itself
// (s_waitcnt 0 + barrier at the top of each K-step).  The memory clobber
// keeps the loads in program order with the LDS reads.
template <bool PAD>
__device__ __forceinline__ void asm_buffer_load_lds(i32x4_t rsrc, uint32_t lds_addr, int voffset,
                                                    int soffset) {
  if constexpr (PAD)
    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds_addr)
                 : "memory");
  else
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds_addr)
                 : "memory");
}
// The same for 4 bytes a lane: lane i's land at the LDS address + 4 i.
template <bool PAD>
__device__ __forceinline__ void asm_buffer_load_lds4(i32x4_t rsrc, uint32_t lds_addr, int voffset, int soffset) {
  if constexpr (PAD)
    asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds_addr)
                 : "memory");
  else
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(soffset), "{m0}"(lds_addr)
                 : "memory");
}
__device__ __forceinline__ i32x4_t buffer_rsrc(const void* base, uint32_t bytes) {
  struct __attribute__((packed)) Rsrc {
    const void* ptr;
    uint32_t range;
    uint32_t config;
  } r{base, bytes, 0x00020000u};
  i32x4_t v = __builtin_bit_cast(i32x4_t, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_readfirstlane(v[i]);
  return v;
}

// Waits until at most N of the wave's vector-memory operations, and none of
// its LDS operations, are in flight.  (s_waitcnt immediate, gfx9 layout: vmcnt bits
// 3:0 and 15:14, expcnt 6:4, left alone, lgkmcnt 11:8.)
template <int N>
__device__ __forceinline__ void wait_vm_lgkm0() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (((N >> 4) & 0x3) << 14));
}

// Workgroup barrier without the vmcnt(0) the compiler puts in front of
// __syncthreads (its release fence waits for every load in flight, which
// would drain a pipeline of more than two stages); the "memory" clobber
// keeps the compiler from moving memory accesses across it.  The caller
// waits right before for what the barrier publishes (its own loads of the
// next stage, its LDS reads of the stage about to be refilled).
__device__ __forceinline__ void barrier_keep_loads() { asm volatile("s_barrier" ::: "memory"); }

}  // namespace aicf::hip
