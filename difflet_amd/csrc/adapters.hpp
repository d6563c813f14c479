// Low-rank adapters of packed requests beside a shared GEMM: C[m] += s_a (x[m] A_a^T) B_a^T with a
// the adapter of row m's request.
//
// adapters.hip computes v = s_a x A_a^T (rank values a row, fp32, in `pieces` parts of K to be
// added). The GEMM kernels then go on with their accumulators over a few more K stages: the row's
// v, rounded to bf16, is the first operand's further columns and B_a the weight's. Nothing of C is
// read or written twice, and the sum is rounded once with the rest. A tile's rows may belong to
// several requests; its distinct adapters lie side by side along that K axis, every row zero
// outside its own. 0 times an infinity or NaN in a neighbour's B would not be 0, so those are staged
// as 0 and the columns noted, which then become NaN in the rows of that adapter alone.
#pragma once

#include "common.hpp"
#include "packed.hpp"

namespace dlt {

struct LoraDev {
  const float* v;         // [pieces][m][ldv] (fp32)
  const bf16* up;         // [adapters][n][rank]
  const int32_t* starts;  // requests + 1 row numbers
  const int32_t* ids;     // adapter of each request, others than [0, adapters): none
  int64_t v_piece;        // elements between the pieces
  int requests, adapters, rank;
  int ldv;                // rank rounded up to 8, the columns past it zero
  int pieces;
  int m, n;               // rows of x, rows of an adapter's B
};

// Row numbers and adapters of up to this many requests are looked up in LDS.
constexpr int LORA_LDS_REQUESTS = 2048;

// LDS of the bookkeeping below: row numbers and adapters, the slot of each row, the slots' adapters,
// two counts, a bit per slot and column.
constexpr int LORA_BOOK_BYTES = (2 * LORA_LDS_REQUESTS + 1 + 2 * 256 + 2 + 256 * 256 / 32) * 4;

// The adapter of row m (-1: none): the last request that starts at or before m, if m is in it.
template <typename Start, typename Id>
__device__ __forceinline__ int lora_row_adapter(const LoraDev& L, int m, Start start, Id id) {
  int lo = 0, hi = L.requests;  // first request that starts past m
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= m) lo = mid + 1;
    else hi = mid;
  }
  if (lo == 0 || m >= start(lo)) return -1;
  const int a = id(lo - 1);
  return (uint32_t)a < (uint32_t)L.adapters ? a : -1;
}

// Slots of the tile's rows m0 .. m0 + BM - 1: slot[r] (-1 for rows without an adapter or past m),
// list[s] the adapter of slot s; returns how many slots there are. bad: [slots][BN / 32] zeros and,
// ahead of them, a zero flag. `book`: LDS that is free, by all NT >= BM threads; ends with a barrier.
template <int BM, int BN, int NT>
__device__ __forceinline__ int lora_slots(const LoraDev& L, int m0, uint8_t* book, int*& slot,
                                          int*& list, uint32_t*& bad) {
  static_assert(BM <= 256 && BM <= NT, "a thread per row");
  int* ints = reinterpret_cast<int*>(book);
  int *starts = ints, *ids = ints + LORA_LDS_REQUESTS + 1;
  slot = ids + LORA_LDS_REQUESTS;
  list = slot + 256;
  int* count = list + 256;
  bad = reinterpret_cast<uint32_t*>(count + 2);
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const bool in_lds = L.requests <= LORA_LDS_REQUESTS;
  if (in_lds) {
    for (int i = tid; i <= L.requests; i += NT) starts[i] = packed_start(L.starts, i, L.m);
    for (int i = tid; i < L.requests; i += NT) ids[i] = L.ids[i];
  }
  __syncthreads();
  if (tid < BM) {
    const int m = m0 + tid;
    int a = -1;
    if (m < L.m) {
      if (in_lds)
        a = lora_row_adapter(L, m, [&](int i) { return starts[i]; }, [&](int i) { return ids[i]; });
      else
        a = lora_row_adapter(L, m, [&](int i) { return packed_start(L.starts, i, L.m); },
                             [&](int i) { return L.ids[i]; });
    }
    slot[tid] = a;
  }
  __syncthreads();
  // one wavefront numbers the distinct adapters in the order of their first rows: a round per
  // adapter and 64 rows, and most tiles have one or two
  if (tid < kWave) {
    int n = 0;
    for (int c = 0; c < BM; c += kWave) {
      const int a = slot[c + lane];
      int s = -1;
      uint64_t left = __ballot(a >= 0);
      while (left) {
        const int b = __builtin_amdgcn_readlane(a, __ffsll((unsigned long long)left) - 1);
        int at = -1;
        for (int i = 0; i < n && at < 0; i += kWave) {
          const uint64_t hit = __ballot(i + lane < n && list[i + lane] == b);
          if (hit) at = i + __ffsll((unsigned long long)hit) - 1;
        }
        if (at < 0) {
          at = n++;
          if (lane == 0) list[at] = b;
          __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        }
        if (a == b) s = at;
        left &= ~__ballot(a == b);
      }
      slot[c + lane] = s;
    }
    if (lane == 0) count[0] = n, count[1] = 0;
    for (int i = lane; i < n * (BN / 32); i += kWave) bad[i] = 0u;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(count[0]);
}

// Zero in place of the infinities and NaN among eight bf16 values; whether there were any.
__device__ __forceinline__ bool lora_finite8(u32x4& w) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
    any |= lo || hi;
    w[e] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
  }
  return any;
}

// The further K stages of a BM x BN tile at (m0, n0): `stage` is LDS for (BM + BN) rows of 128
// bytes in the GEMMs' layout (chunk c of row r at c ^ swz(r)), `book` as above, both free when this
// is called by all NT threads after a barrier. mma(ks) runs K step ks (16 values) of the staged
// operands into the accumulators; poison(slot, bad) makes those NaN whose row's slot s has bit n of
// bad[s * BN / 32 ..] set for their column n.
template <int BM, int BN, int NT, typename Swz, typename Mma, typename Poison>
__device__ __forceinline__ void lora_stages(const LoraDev& L, int m0, int n0, uint8_t* stage,
                                            uint8_t* book, Swz swz, Mma mma, Poison poison) {
  int *slot, *list;
  uint32_t* bad;
  const int slots = lora_slots<BM, BN, NT>(L, m0, book, slot, list, bad);
  const int per = L.ldv >> 3;  // chunks of 8 ranks of an adapter
  const int total = slots * per;
  const int tid = threadIdx.x, ch = tid & 7;
  constexpr int RP = NT / 8;  // rows a pass
  for (int c0 = 0; c0 < total; c0 += 8) {
    const int vc = c0 + ch, s = vc / per, r8 = (vc - s * per) * 8;
    const bool on = vc < total;
    const int a = on ? list[s] : 0;
    u32x4 w[BN / RP];
#pragma unroll
    for (int i = 0; i < BN / RP; ++i) {
      const int n = n0 + i * RP + (tid >> 3);
      w[i] = u32x4{0u, 0u, 0u, 0u};
      if (!on || n >= L.n || r8 >= L.rank) continue;
      const bf16* p = L.up + ((int64_t)a * L.n + n) * L.rank + r8;
      if ((L.rank & 7) == 0) {
        w[i] = *reinterpret_cast<const u32x4*>(p);
      } else {  // rows of B off 16 bytes
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (r8 + e < L.rank) w[i][e >> 1] |= (uint32_t)h[e] << (16 * (e & 1));
      }
      if (lora_finite8(w[i])) {
        const int c = n - n0;
        atomicOr(&bad[s * (BN / 32) + (c >> 5)], 1u << (c & 31));
        bad[-1] = 1u;
      }
    }
    u32x4 x[BM / RP];
#pragma unroll
    for (int i = 0; i < BM / RP; ++i) {
      const int r = i * RP + (tid >> 3);
      float v[8] = {};
      if (on && slot[r] == s) {
        const float* p = L.v + (int64_t)(m0 + r) * L.ldv + r8;
        for (int q = 0; q < L.pieces; ++q, p += L.v_piece) {
          const f32x4 lo = *reinterpret_cast<const f32x4*>(p);
          const f32x4 hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    }
#pragma unroll
    for (int i = 0; i < BM / RP; ++i) {
      const int r = i * RP + (tid >> 3);
      *reinterpret_cast<u32x4*>(stage + r * 128 + ((ch ^ swz(r)) << 4)) = x[i];
    }
#pragma unroll
    for (int i = 0; i < BN / RP; ++i) {
      const int r = i * RP + (tid >> 3);
      *reinterpret_cast<u32x4*>(stage + (BM + r) * 128 + ((ch ^ swz(r)) << 4)) = w[i];
    }
    __syncthreads();
    const int steps = (min(total - c0, 8) + 1) >> 1;
    for (int ks = 0; ks < steps; ++ks) mma(ks);
    __syncthreads();
  }
  if (total > 0 && bad[-1]) poison(slot, bad);
}

}  // namespace dlt
