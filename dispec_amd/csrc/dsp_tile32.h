// What the kernels on 32-row tiles (v_mfma_f32_32x32x16) share: the MFMA, the LDS DMA and the
// transposing read of V.
#pragma once

#include "dsp_mfma.h"

namespace dsp_mfma {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename Tag>
__device__ __forceinline__ f32x16 mfma32x32(dsp_u32x4 a, dsp_u32x4 b, f32x16 c) {
  if constexpr (std::is_same<Tag, Bf16Tag>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void lds_void_t;

// One LDS DMA (global_load_lds_dwordx4): 16 bytes per lane from sbase + voff into LDS at
// m0 + 16 * lane.  It is issued from inline assembly so that the compiler does not make
// later LDS reads wait for it: its waitcnt pass cannot tell the DMA's target buffer from
// the one being read and would wait for the whole DMA.  The kernel waits for it itself
// (vmcnt) before the barrier that publishes the chunk.  M0 has no other user here.
// kNonTemporal marks the load nt: a shared-prefix launch reads most of its keys once (the
// prefix by one or a few packed tiles, each suffix by its sequence's tiles), so keeping them
// in the caches only evicts what other launches reuse (fork decode 23.5-23.8 -> 21.4 us
// per layer, verify unchanged).  An unshared prefill re-reads a sequence's keys from every
// 128-row tile of its queries and keeps the ordinary load (nt costs it 3-8 %).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <bool kNonTemporal>
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t m0) {
  if constexpr (kNonTemporal)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(voff), "s"(sbase), "s"(m0)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(voff), "s"(sbase), "s"(m0)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16_t;

// The V^T operand of 16-key step ps of a chunk in LDS: dim 32*dt + col, K index 8*hl + i <-> key
// 16*ps + 8*(i/4) + 4*hl + i%4 (the P^T order; col = lane % 32, hl = lane / 32).  In
// ds_read_b64_tr_b16, lane g + 4a + e of each 16-lane group g receives element e of the
// 4-element segments addressed by lanes g + a + 4j (j = 0..3); so lane s addresses key 16*ps +
// 8*inst + 4*hl + (s%16)/4, dims 32*dt + 16*((s/16)%2) + 4*(s%4) .. +3, for inst = 0, 1.
template <int D>
__device__ __forceinline__ dsp_u32x4 load_vt(const char* vs_lds, int ps, int dt) {
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  v4i16 vh[2];
#pragma unroll
  for (int inst = 0; inst < 2; ++inst) {
    const int kr = 16 * ps + 8 * inst + 4 * hl + ((lane & 15) >> 2);
    const int dim0 = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int swz = D >= 128 ? 4 * (kr & 3) : 4 * ((kr >> 1) & 1);
    vh[inst] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
        vs_lds + kr * 2 * D + 16 * ((dim0 >> 3) ^ swz) + 2 * (dim0 & 7)));
  }
  return __builtin_bit_cast(dsp_u32x4, vh);
}

}  // namespace dsp_mfma
