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
//
// Most tiles of many rows lie in one request. Which ones do is found before the K loop from the row
// numbers (a lane each), and for those there are no slots: a tile waits for one round of loads and
// two barriers behind its K loop. 7141 x 3072 x 12288, bf16, rank 32: 504 us so, 580 with slots
// in every tile, 570 with the fragments straight from memory (32 rows a load, which the address unit
// takes one by one); the linear alone 467.
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

// Whether rows [m0, end) of a tile are all of one request, or of none: their adapter, -1 for none, -2
// for a tile that is not like that (or more requests than this looks at). load() reads what find()
// needs, which a kernel does before its K loop, so that nothing of it is waited for behind.
struct LoraOne {
  static constexpr int MOST = kWave - 1;
  int start = 0, id = -1;  // of request `lane`; lane `requests` the last row number
  __device__ __forceinline__ void load(const LoraDev& L) {
    const int lane = threadIdx.x & (kWave - 1);
    if (L.requests == 0 || L.requests > MOST) return;
    start = packed_start(L.starts, min(lane, L.requests), L.m);
    id = L.ids[min(lane, L.requests - 1)];
  }
  __device__ __forceinline__ int find(const LoraDev& L, int m0, int end) const {
    if (L.requests == 0) return -1;
    if (L.requests > MOST) return -2;
    const int lane = threadIdx.x & (kWave - 1);
    const int n = __popcll(__ballot(lane < L.requests && start <= m0));  // that start at or before m0
    const int next = __builtin_amdgcn_readlane(start, n);  // n == requests: where the last one ends
    if (n == L.requests && next <= m0) return -1;
    if (next < end) return -2;
    const int a = n ? __builtin_amdgcn_readlane(id, max(n - 1, 0)) : -1;
    return (uint32_t)a < (uint32_t)L.adapters ? a : -1;
  }
  // The adapter of row m (-1: none), of each lane's own, by all lanes; at most MOST requests.
  __device__ __forceinline__ int of_row(const LoraDev& L, int m) const {
    int n = 0;
    for (int i = 0; i < L.requests; ++i) n += __builtin_amdgcn_readlane(start, i) <= m;
    const int end = __shfl(start, n, kWave), a = __shfl(id, max(n - 1, 0), kWave);
    return n && m < end && (uint32_t)a < (uint32_t)L.adapters ? a : -1;
  }
};

// Eight rank values at p, their pieces added in order, the loads of FLY pieces at a time in flight.
template <int FLY>
__device__ __forceinline__ void lora_v8(const LoraDev& L, const float* p, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 1
  for (int q = 0; q < L.pieces; q += FLY, p += FLY * L.v_piece) {
    f32x4 t[FLY][2];
#pragma unroll
    for (int i = 0; i < FLY; ++i) {
      t[i][0] = t[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (q + i < L.pieces) {
        t[i][0] = *reinterpret_cast<const f32x4*>(p + i * L.v_piece);
        t[i][1] = *reinterpret_cast<const f32x4*>(p + i * L.v_piece + 4);
      }
    }
#pragma unroll
    for (int i = 0; i < FLY; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += t[i][e >> 2][e & 3];
  }
}

// Slots of the tile's rows m0 .. m0 + BM - 1: slot[r] (-1 for rows without an adapter or past m),
// list[s] the adapter of slot s; returns how many slots there are. bad: [slots][BN / 32] zeros and,
// ahead of them, a zero flag. `book`: LDS that is free, by all NT >= BM threads; ends with a barrier.
// Up to LoraOne::MOST requests are in the lanes' registers already (`rows`).
template <int BM, int BN, int NT>
__device__ __forceinline__ int lora_slots(const LoraDev& L, const LoraOne& rows, int m0, uint8_t* book,
                                          int*& slot, int*& list, uint32_t*& bad) {
  static_assert(BM <= 256 && BM <= NT, "a thread per row");
  int* ints = reinterpret_cast<int*>(book);
  int *starts = ints, *ids = ints + LORA_LDS_REQUESTS + 1;
  slot = ids + LORA_LDS_REQUESTS;
  list = slot + 256;
  int* count = list + 256;
  bad = reinterpret_cast<uint32_t*>(count + 2);
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const bool in_regs = L.requests <= LoraOne::MOST, in_lds = L.requests <= LORA_LDS_REQUESTS;
  if (in_lds && !in_regs) {
    for (int i = tid; i <= L.requests; i += NT) starts[i] = packed_start(L.starts, i, L.m);
    for (int i = tid; i < L.requests; i += NT) ids[i] = L.ids[i];
    __syncthreads();
  }
  if (tid < BM) {
    const int m = m0 + tid;
    int a = -1;
    if (in_regs) {
      a = rows.of_row(L, m);
    } else if (m < L.m) {
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
    int n = 0, mine = -1;  // mine: list[lane], the first 64 of the list
    for (int c = 0; c < BM; c += kWave) {
      const int a = slot[c + lane];
      int s = -1;
      uint64_t left = __ballot(a >= 0);
      while (left) {
        const int b = __builtin_amdgcn_readlane(a, __ffsll((unsigned long long)left) - 1);
        int at = __ffsll((unsigned long long)__ballot(mine == b)) - 1;
        for (int i = kWave; i < n && at < 0; i += kWave) {
          const uint64_t hit = __ballot(i + lane < n && list[i + lane] == b);
          if (hit) at = i + __ffsll((unsigned long long)hit) - 1;
        }
        if (at < 0) {
          at = n++;
          if (lane == at) mine = b;
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

// Ranks r8 .. r8 + 7 (r8 < rank) of column n of adapter a, those past the rank zero.
__device__ __forceinline__ u32x4 lora_up8(const LoraDev& L, int a, int n, int r8) {
  const bf16* p = L.up + ((int64_t)a * L.n + n) * L.rank + r8;
  if ((L.rank & 7) == 0) return *reinterpret_cast<const u32x4*>(p);
  u32x4 w = {0u, 0u, 0u, 0u};  // rows of B off 16 bytes
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (r8 + e < L.rank) w[e >> 1] |= (uint32_t)h[e] << (16 * (e & 1));
  return w;
}

// Chunks c0 .. c0 + 7 of adapter a's ranks into LDS (c0 a multiple of 8, `per` chunks in all), for rows
// that all have it: the rows' values and the columns' each lie in one piece of memory, which the
// threads read end to end. Ends with a barrier.
template <int BM, int BN, int NT, int FLY, typename Swz>
__device__ __forceinline__ void lora_stage_one(const LoraDev& L, int m0, int n0, int a, int c0, int per,
                                               uint8_t* stage, Swz swz) {
  const int tid = threadIdx.x;
  const int n8 = min(per - c0, 8), pairs = (n8 + 1) & ~1;  // K steps take two chunks
  const uint32_t inv = 65535u / (uint32_t)pairs + 1;       // i / pairs, exact below 2048
  constexpr int PX = BM * 8 / NT, PW = BN * 8 / NT;
  u32x4 x[PX], w[PW];
#pragma unroll
  for (int k = 0; k < PW; ++k) {
    const int i = k * NT + tid, r = (int)((uint32_t)i * inv >> 16), ch = i - r * pairs;
    w[k] = u32x4{0u, 0u, 0u, 0u};
    if (r < BN && n0 + r < L.n && ch < n8 && (c0 + ch) * 8 < L.rank)
      w[k] = lora_up8(L, a, n0 + r, (c0 + ch) * 8);
  }
#pragma unroll
  for (int k = 0; k < PX; ++k) {
    const int i = k * NT + tid, r = (int)((uint32_t)i * inv >> 16), ch = i - r * pairs;
    float v[8] = {};
    if (r < BM && m0 + r < L.m && ch < n8)
      lora_v8<FLY>(L, L.v + (int64_t)(m0 + r) * L.ldv + (c0 + ch) * 8, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[k][e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
  }
#pragma unroll
  for (int k = 0; k < PX; ++k) {
    const int i = k * NT + tid, r = (int)((uint32_t)i * inv >> 16), ch = i - r * pairs;
    if (r < BM) *reinterpret_cast<u32x4*>(stage + r * 128 + ((ch ^ swz(r)) << 4)) = x[k];
  }
#pragma unroll
  for (int k = 0; k < PW; ++k) {
    const int i = k * NT + tid, r = (int)((uint32_t)i * inv >> 16), ch = i - r * pairs;
    if (r < BN) *reinterpret_cast<u32x4*>(stage + (BM + r) * 128 + ((ch ^ swz(r)) << 4)) = w[k];
  }
  __syncthreads();
}

// Chunks c0 .. c0 + 7 of the slots' ranks into LDS (c0 a multiple of 8): the rows' rank values and the
// adapters' columns. Ends with a barrier.
template <int BM, int BN, int NT, int FLY, typename Swz>
__device__ __forceinline__ void lora_stage(const LoraDev& L, int m0, int n0, int c0, int total, int per,
                                           const int* slot, const int* list, uint32_t* bad,
                                           uint8_t* stage, Swz swz) {
  const int tid = threadIdx.x, ch = tid & 7;
  constexpr int RP = NT / 8;  // rows a pass
  const int vc = c0 + ch, s = vc / per, r8 = (vc - s * per) * 8;
  const bool on = vc < total;
  const int a = on ? list[s] : 0;
  u32x4 w[BN / RP];
#pragma unroll
  for (int i = 0; i < BN / RP; ++i) {
    const int n = n0 + i * RP + (tid >> 3);
    w[i] = u32x4{0u, 0u, 0u, 0u};
    if (on && n < L.n && r8 < L.rank) w[i] = lora_up8(L, a, n, r8);
  }
  u32x4 x[BM / RP];
#pragma unroll
  for (int i = 0; i < BM / RP; ++i) {
    const int r = i * RP + (tid >> 3);
    float v[8] = {};
    if (on && slot[r] == s) lora_v8<FLY>(L, L.v + (int64_t)(m0 + r) * L.ldv + r8, v);
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
    if (lora_finite8(w[i])) {  // looked at after both operands' loads went out
      atomicOr(&bad[s * (BN / 32) + (r >> 5)], 1u << (r & 31));
      bad[-1] = 1u;
    }
    *reinterpret_cast<u32x4*>(stage + (BM + r) * 128 + ((ch ^ swz(r)) << 4)) = w[i];
  }
  __syncthreads();
}

// The further K stages of a BM x BN tile at (m0, n0), whose rows all have adapter `one`, or, below 0,
// not. `stage` is LDS for (BM + BN) rows of 128 bytes in the GEMMs' layout (chunk c of row r at c ^
// swz(r)), `book` as above, both idle once every wavefront is here. mma(ks) runs K step ks (16
// values) of the staged operands into the accumulators; poison(slot, bad) makes those NaN whose row's
// slot s has bit n of bad[s * BN / 32 ..] set for their column n. Called by all NT threads.
template <int BM, int BN, int NT, int FLY, typename Swz, typename Mma, typename Poison>
__device__ __forceinline__ void lora_stages(const LoraDev& L, const LoraOne& rows, int m0, int n0,
                                            int one, uint8_t* stage, uint8_t* book, Swz swz, Mma mma,
                                            Poison poison) {
  int *slot = nullptr, *list = nullptr;
  uint32_t* bad = nullptr;
  const bool many = one < 0;
  int slots = 1;
  __syncthreads();  // every wavefront's reads of the ring are done
  if (many) slots = lora_slots<BM, BN, NT>(L, rows, m0, book, slot, list, bad);
  const int per = L.ldv >> 3;  // chunks of 8 ranks of an adapter
  const int total = slots * per;
#pragma unroll 1
  for (int c0 = 0; c0 < total; c0 += 8) {
    if (many) lora_stage<BM, BN, NT, FLY>(L, m0, n0, c0, total, per, slot, list, bad, stage, swz);
    else lora_stage_one<BM, BN, NT, FLY>(L, m0, n0, one, c0, per, stage, swz);
    const int steps = (min(total - c0, 8) + 1) >> 1;
#pragma unroll 1
    for (int ks = 0; ks < steps; ++ks) mma(ks);
    __syncthreads();
  }
  if (many && total > 0 && bad[-1]) poison(slot, bad);
}

}  // namespace dlt
