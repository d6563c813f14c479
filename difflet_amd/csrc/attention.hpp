// What the attention kernels share: matrix-core types, the V^T key order, direct-to-LDS loads and
// the exchanges between the two lanes that hold a query's statistics.
#pragma once

#include "common.hpp"

namespace dlt {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct MfmaT;
template <> struct MfmaT<bf16> {
  typedef bf16x8 frag;
  // lazy-rescale limit of the ping-pong softmax: every P below it is a finite 16-bit operand
  static constexpr float kLazyLimit = 0x1p20f;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    bf16x2 v = {(bf16)a, (bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <> struct MfmaT<f16> {
  typedef f16x8 frag;
  static constexpr float kLazyLimit = 0x1p15f;  // fp16's largest finite value is 65504
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
// Position of key quad q (keys 4q .. 4q + 3 of a tile) in a V^T row: inside each 16-key group the
// middle quads swap, so the 8 keys a lane group feeds one 16-key MFMA step, {4g .. 4g + 3,
// 8 + 4g .. 8 + 4g + 3}, sit side by side and load as one 16-byte read.
__device__ __forceinline__ int vt_quad_pos(int q) {
  const int r = q & 3;
  return (q & ~3) | (r == 1 ? 2 : r == 2 ? 1 : r);
}

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16_t;
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// One direct-to-LDS load: 16 bytes per lane at byte offset voff of buffer r into LDS bytes
// [lds_addr + 16 lane, + 16). Written as inline assembly so that the compiler does not track it:
// the builtin makes it wait for every such load before the next LDS read of any address (it
// cannot tell the tile being filled from the ones being read), which put each tile's whole
// load latency in front of the next phase's fragment reads. The kernel waits for these loads
// itself (vmcnt(0) before the barrier that publishes a tile); the compiler's own waits for the
// loads it does track only grow stricter with untracked loads in flight.
// r: the buffer resource's four words (rsrc_words).
__device__ __forceinline__ void dma16(i32x4_t r, const uint8_t* lds_ptr, uint32_t voff) {
  const uint32_t la = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds_ptr);
  // s_nop 4: five wait states for a resource word a VALU instruction (v_readlane) may have just
  // written; s_nop 0: one between the M0 write and the load that reads it
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(la), "v"(voff), "s"(r)
               : "memory", "m0");
}
// The same with a scalar offset beside the lanes' own.
__device__ __forceinline__ void dma16s(i32x4_t r, const uint8_t* lds_ptr, uint32_t voff, uint32_t soff) {
  const uint32_t la = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds_ptr);
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(la), "v"(voff), "s"(r), "s"(soff)
               : "memory", "m0");
}
// The words of make_rsrc's resource: base address, stride 0, `bytes` records, the same flags.
__device__ __forceinline__ i32x4_t rsrc_words(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i32x4_t{(int)(uint32_t)a, (int)(uint32_t)((a >> 32) & 0xffffu), (int)bytes, 0x00020000};
}

// max / sum of x over lanes l and l ^ 32 (the two lanes holding one query's statistics).
// v_permlane32_swap exchanges the upper half of its first operand with the lower half of its
// second: given x twice, the two results hold {x, x of lane l ^ 32} in every lane, so their max
// or sum is the pair's. A VALU instruction, unlike ds_bpermute, so it neither uses the LDS nor
// waits on it.
__device__ __forceinline__ float pair_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

}  // namespace dlt
