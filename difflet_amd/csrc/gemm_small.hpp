// The small-launch GEMM (gemm_small.hip) as gemm.hip's dispatch sees it, and the direct-to-LDS loads
// that it shares with adapters.hip.
#pragma once

#include "common.hpp"

namespace dlt {

// direct-to-LDS load of 16 bytes per lane (as attention.hip's dma16, with a scalar offset):
// untracked by the compiler, waited for by the K loop's own vmcnt
typedef __attribute__((address_space(3))) void lds_void_t;
__device__ __forceinline__ void dma16s(i32x4 r, const uint8_t* lds_ptr, uint32_t voff,
                                       uint32_t soff) {
  const uint32_t la = (uint32_t)reinterpret_cast<uintptr_t>((lds_void_t*)lds_ptr);
  asm volatile("s_nop 4\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(la), "v"(voff), "s"(r), "s"(soff)
               : "memory", "m0");
}
__device__ __forceinline__ i32x4 rsrc_of(const void* base, int64_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint32_t n = bytes > 0xffffffffLL ? 0xffffffffu : (uint32_t)bytes;
  return i32x4{(int)(uint32_t)a, (int)(uint32_t)((a >> 32) & 0xffffu), (int)n, 0x00020000};
}
template <int VM>
__device__ __forceinline__ void wait_vm() {
  static_assert(VM >= 0 && VM < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt(0x0070 | (VM & 15) | ((VM >> 4) << 14));  // and lgkmcnt(0)
}
__device__ __forceinline__ int swz8s(int row) { return (row & 7) ^ ((row >> 3) & 1); }

enum class SmallElem { BF16, FP8, MX, F32 };

// bm x bn tiles, K in `pieces` of piece_stages 128-byte stages; bm == 0: not worth it.
struct SmallPlan {
  int bm, bn, pieces, piece_stages;
};

// The fastest plan for one m x n x k problem on `cus` compute units with `scratch` bytes for the
// K pieces' sums (0: K stays whole), if it beats big_us, the 256 x 256 tiles' estimate.
SmallPlan small_plan(SmallElem e, int64_t m, int64_t n, int64_t k, int cus, int64_t scratch,
                     double big_us);

// Runs the plan: operands checked by the caller as for gemm.hip (F32: gemm_f32.hip, C, bias and
// residual fp32, residual + (acc + bias)). gate: EPI_GATE_RESIDUAL. lora: adapters of packed
// requests (not with gate or F32).
struct LoraDev;
void gemm_small(SmallElem e, const SmallPlan& plan, const difflet_gemm_problem& q, int64_t n,
                int64_t k, bool gate, int64_t rows_per_batch, void* scratch, hipStream_t s,
                const LoraDev* lora = nullptr);

// One problem without an epilogue, with adapters (gemm.hip); kind as difflet_rocm_gemm_single's,
// the workspace this launch's alone.
int gemm_lora(int kind, const difflet_gemm_problem& q, int64_t n, int64_t k, void* workspace,
              int64_t workspace_bytes, hipStream_t stream, const LoraDev& lora);

// Compute units of the current device (gemm.hip).
int gemm_device_cus();

}  // namespace dlt
