// Low-rank adapters of packed requests beside a shared linear:
//   y[m] = x[m] W^T + b + s_a (x[m] A_a^T) B_a^T,  a = the adapter of row m's request (none: x W^T + b)
// in two launches: the kernel here takes x to its rank values v = s_a x A_a^T, then the linear's own
// GEMM adds v B_a^T in its accumulators (adapters.hpp). What the adapters cannot do without is one
// more read of x, A and B; the GEMM's matrix work grows by rank / K.
//
// Few rows: a workgroup takes 32 rows of one request and a part of K, its four wavefronts each every
// fourth 64-wide step of it (MFMA 32x32x16, A first: a lane holds one row of x); x and A go from
// memory to the matrix cores without LDS, since each is used once there, and the wavefronts' sums
// meet in LDS. Many rows: a workgroup takes 128 rows, its wavefronts 32 each beside the same ranks,
// and both operands come through a ring of LDS stages, 128 bytes of a row at a time: read straight
// from memory, 32 rows at strides of the width share four sets of the L1, and each line is fetched
// for every 32 bytes of it (34125 x 5120, rank 64: 233 us; 110 through LDS, 3.2 TB/s,
// of about 4 that a read alone reaches).
// Where that leaves compute units idle, K is cut into `pieces` whose sums the GEMM adds in order.
#include <algorithm>

#include "adapters.hpp"
#include "gemm_small.hpp"

namespace dlt {

struct LoraDownArgs {
  const bf16* x;
  const bf16* down;  // [adapters][rank][k]
  const float* scale;
  const int32_t* starts;
  const int32_t* ids;
  float* v;
  int64_t ldx, v_piece;
  int m, k, rank, ldv, requests, adapters;
  int items, pieces, blocks;  // row tiles at most, K pieces, rank blocks of 32 NR
};

template <int NR>
__global__ __launch_bounds__(256) void lora_down_kernel(const LoraDownArgs a) {
  __shared__ float sums[4][32 * 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, g = lane >> 5;
  int id = blockIdx.x;
  const int item = id % a.items;
  id /= a.items;
  const int piece = id % a.pieces, rb = id / a.pieces;
  const PackedItem it = packed_item(a.starts, a.requests, a.m, 1, 32, false, item);
  if (it.req < 0) return;
  const int ad = a.ids[it.req];
  if ((uint32_t)ad >= (uint32_t)a.adapters) return;
  const int steps = (a.k + 63) / 64, per = (steps + a.pieces - 1) / a.pieces;
  const int sbeg = piece * per, send = min(sbeg + per, steps);
  // rows past the request and ranks past the adapter's read the last ones, whose results go nowhere
  const int row = min(it.tile * 32 + col, it.rows - 1);
  const bf16* xp = a.x + (int64_t)(it.row0 + row) * a.ldx + g * 8;
  const bf16* dp[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = min((rb * NR + i) * 32 + col, a.rank - 1);
    dp[i] = a.down + ((int64_t)ad * a.rank + r) * a.k + g * 8;
  }
  f32x16 acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) acc[i] = f32x16{};
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int s = sbeg + wave; s < send; s += 4) {
    u32x4 xv[4], dv[NR][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = s * 64 + c * 16;
      const bool in = k + g * 8 < a.k;  // k is a multiple of 8
      xv[c] = in ? *reinterpret_cast<const u32x4*>(xp + k) : zero;
#pragma unroll
      for (int i = 0; i < NR; ++i) dv[i][c] = in ? *reinterpret_cast<const u32x4*>(dp[i] + k) : zero;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < NR; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, dv[i][c]),
                                                         __builtin_bit_cast(bf16x8, xv[c]), acc[i],
                                                         0, 0, 0);
  }
  // lane: row col of x, ranks 8 q + 4 g + e of each block of 32
  const float scale = a.scale[ad];
  const int r4 = (tid & 7) * 4, xr = tid >> 3;  // this thread's ranks and row of the sum
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    if (i) __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(&sums[wave][col * 32 + (((2 * q + g) ^ (col & 7)) << 2)]) =
          f32x4{acc[i][4 * q], acc[i][4 * q + 1], acc[i][4 * q + 2], acc[i][4 * q + 3]};
    __syncthreads();
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 p = *reinterpret_cast<const f32x4*>(&sums[w][xr * 32 + (((r4 >> 2) ^ (xr & 7)) << 2)]);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += p[e];
    }
    const int r = (rb * NR + i) * 32 + r4, m = it.tile * 32 + xr;
    if (m < it.rows && r < a.ldv) {
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = r + e < a.rank ? t[e] * scale : 0.f;
      *reinterpret_cast<f32x4*>(a.v + piece * a.v_piece + (int64_t)(it.row0 + m) * a.ldv + r) = t;
    }
  }
}

constexpr int LORA_ROWS = 128;  // rows of a wide tile

// The same for 128 rows of a request: 32 NR ranks, stages of 64 K elements (128 bytes a row) in a
// ring of NS slots, NS - 1 of them in flight (NR = 2: 3 slots leave room for two workgroups on a
// compute unit, 110 us above; 4 slots 114, 6 slots 115). Rows of x past the request, ranks past the adapter's
// and K past the width read zero.
template <int NR, int NS>
__global__ __launch_bounds__(256, 1) void lora_down_wide_kernel(const LoraDownArgs a) {
  constexpr int ROWS = LORA_ROWS + 32 * NR, SLOT = ROWS * 128, LPW = ROWS / 8 / 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[NS * SLOT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  int id = blockIdx.x;
  const int item = id % a.items;
  id /= a.items;
  const int piece = id % a.pieces, rb = id / a.pieces;
  const PackedItem it = packed_item(a.starts, a.requests, a.m, 1, LORA_ROWS, false, item);
  if (it.req < 0) return;
  const int ad = a.ids[it.req];
  if ((uint32_t)ad >= (uint32_t)a.adapters) return;
  const int steps = (a.k + 63) / 64, per = (steps + a.pieces - 1) / a.pieces;
  const int sbeg = piece * per, n = min(sbeg + per, steps) - sbeg;
  const int rows = min(it.rows - it.tile * LORA_ROWS, LORA_ROWS);
  const int ranks = min(a.rank - rb * 32 * NR, 32 * NR);
  const int row0 = it.row0 + it.tile * LORA_ROWS;
  constexpr uint32_t kOut = 0xfffffff0u;
  const i32x4 rx = rsrc_of(a.x + (int64_t)row0 * a.ldx, (rows - 1) * a.ldx * 2 + (int64_t)a.k * 2);
  const i32x4 rd = rsrc_of(a.down + ((int64_t)ad * a.rank + rb * 32 * NR) * a.k, (int64_t)ranks * a.k * 2);
  // this wave's 1 KB loads of a stage: 8 rows of 8 chunks each, x's rows first
  uint32_t off[LPW];
  const int ch = lane & 7;
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int r = (wave * LPW + i) * 8 + (lane >> 3), kc = (ch ^ swz8s(r)) * 8;
    const bool is_x = r < LORA_ROWS;
    const int64_t o = is_x ? r * a.ldx * 2 : (int64_t)(r - LORA_ROWS) * a.k * 2;
    off[i] = (is_x ? r < rows : r - LORA_ROWS < ranks) ? (uint32_t)o + kc * 2 : kOut;
  }
  auto issue = [&](int s) {
    uint8_t* d = lds + (s % NS) * SLOT;
    const int k0 = (sbeg + s) * 64;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int r = (wave * LPW + i) * 8 + (lane >> 3);
      const bool in = s < n && k0 + (ch ^ swz8s(r)) * 8 < a.k && off[i] != kOut;
      const uint32_t o = in ? off[i] + (uint32_t)k0 * 2 : kOut;
      dma16s((wave * LPW + i) * 8 < LORA_ROWS ? rx : rd, d + (wave * LPW + i) * 1024, o, 0);
    }
  };
  f32x16 acc[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) acc[i] = f32x16{};
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(s);
  for (int s = 0; s < n; ++s) {
    // this wave's loads of stage s have landed (NS - 2 younger stages may be in flight), its reads of
    // stage s - 1 are done: the barrier publishes the one and frees the other's slot
    wait_vm<(NS - 2) * LPW>();
    asm volatile("s_barrier" ::: "memory");
    issue(s + NS - 1);
    const uint8_t* st = lds + (s % NS) * SLOT;
    auto frag = [&](int r, int c) {
      return *reinterpret_cast<const bf16x8*>(st + r * 128 + (((2 * c + g) ^ swz8s(r)) << 4));
    };
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bf16x8 xv = frag(wave * 32 + col, c);
#pragma unroll
      for (int i = 0; i < NR; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag(LORA_ROWS + i * 32 + col, c), xv,
                                                         acc[i], 0, 0, 0);
    }
  }
  wait_vm<0>();  // no load may outlive the workgroup's LDS
  const float scale = a.scale[ad];
  if (wave * 32 + col >= rows) return;
  float* v = a.v + piece * a.v_piece + (int64_t)(row0 + wave * 32 + col) * a.ldv;
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = (rb * NR + i) * 32 + 8 * q + 4 * g;
      if (r >= a.ldv) continue;
      f32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = r + e < a.rank ? acc[i][4 * q + e] * scale : 0.f;
      *reinterpret_cast<f32x4*>(v + r) = t;
    }
}

static int64_t lora_ldv(int64_t rank) { return (rank + 7) / 8 * 8; }
// Rows from which the wide tiles run: below, their workgroups are too few to draw x's bytes.
static bool lora_wide(int64_t m, int64_t requests) { return m >= 2048 && m >= 32 * requests; }
static int64_t lora_items(int64_t m, int64_t requests) {
  const int64_t rows = lora_wide(m, requests) ? LORA_ROWS : 32;
  return (m + rows - 1) / rows + requests;
}
// K pieces: a workgroup for every compute unit, twice over for the small tiles, and at least 4
// stages (a 64-wide step for each wavefront) a piece
static int64_t lora_pieces(int64_t m, int64_t k, int64_t requests) {
  const int64_t steps = (k + 63) / 64, want = lora_wide(m, requests) ? 256 : 512;
  return std::max<int64_t>(1, std::min<int64_t>({want / lora_items(m, requests), steps / 4, 16}));
}
static int64_t lora_v_bytes(int64_t m, int64_t k, int64_t rank, int64_t requests) {
  return (lora_pieces(m, k, requests) * m * lora_ldv(rank) * 4 + 255) / 256 * 256;
}

}  // namespace dlt

using namespace dlt;

extern "C" int64_t difflet_rocm_lora_workspace_bytes(int kind, int64_t m, int64_t n, int64_t k,
                                                     int64_t rank, int64_t requests) {
  if (kind < 0 || kind > 2 || m <= 0 || n <= 0 || k <= 0 || rank <= 0 || requests < 0 ||
      m >= (1LL << 30) || n >= (1LL << 30) || k >= (1LL << 30) || rank > 1024 ||
      requests >= (1LL << 24))
    return 0;
  return lora_v_bytes(m, k, rank, requests) + difflet_rocm_gemm_scratch_bytes(kind, m, n, k);
}

extern "C" int difflet_rocm_lora_linear(int kind, const void* a, int64_t lda, const void* a_scale,
                                        const void* w, int64_t ldw, const void* w_scale,
                                        const void* bias, void* c, int64_t ldc, int64_t m, int64_t n,
                                        int64_t k, const void* x, int64_t ldx, int64_t x_cols,
                                        const void* down, const void* up, int64_t up_rows,
                                        const float* scale, int64_t adapters, int64_t rank,
                                        const int32_t* starts, const int32_t* ids, int64_t requests,
                                        void* workspace, int64_t workspace_bytes,
                                        difflet_stream_t stream) {
  const char* name = "lora_linear";
  DLT_REQUIRE(kind >= 0 && kind <= 2, DIFFLET_EINVAL, "%s: unknown kind %d", name, kind);
  DLT_REQUIRE(m >= 0 && n > 0 && k > 0 && adapters >= 0 && requests >= 0, DIFFLET_EINVAL,
              "%s: bad shape", name);
  DLT_REQUIRE(rank >= 1, DIFFLET_EINVAL, "%s: rank must be positive", name);
  DLT_REQUIRE(rank <= 1024 && m < (1LL << 30) && requests < (1LL << 24) && adapters < (1LL << 24),
              DIFFLET_EUNSUPPORTED, "%s: rank over 1024 or too many rows, requests or adapters", name);
  DLT_REQUIRE(x_cols > 0 && x_cols <= k && x_cols % 8 == 0 && up_rows > 0 && up_rows <= n,
              DIFFLET_EINVAL, "%s: the adapters' widths (A's a multiple of 8) exceed the weight's",
              name);
  if (m == 0) return DIFFLET_OK;
  DLT_REQUIRE(x && starts && (requests == 0 || ids) && (adapters == 0 || (down && up && scale)),
              DIFFLET_EINVAL, "%s: null pointer", name);
  DLT_REQUIRE(ldx <= (1LL << 23) || m < 2, DIFFLET_EUNSUPPORTED, "%s: rows of x more than 16 MB apart",
              name);
  DLT_REQUIRE(ldx >= x_cols && ldx % 8 == 0 && (((uintptr_t)x | (uintptr_t)down | (uintptr_t)up) & 15) == 0,
              DIFFLET_EINVAL, "%s: rows of x and the adapters must start on 16 bytes", name);
  const int64_t vb = lora_v_bytes(m, x_cols, rank, requests);
  DLT_REQUIRE(workspace && workspace_bytes >= vb && ((uintptr_t)workspace & 255) == 0,
              DIFFLET_EINVAL, "%s: needs a 256-byte aligned workspace of at least %lld bytes", name,
              (long long)vb);
  const int64_t pieces = lora_pieces(m, x_cols, requests), ldv = lora_ldv(rank);
  hipStream_t s = (hipStream_t)stream;
  LoraDev lora = {(const float*)workspace, (const bf16*)up, starts, ids, m * ldv, (int)requests,
                  (int)adapters, (int)rank, (int)ldv, (int)pieces, (int)m, (int)up_rows};
  if (requests > 0 && adapters > 0) {
    LoraDownArgs d = {(const bf16*)x, (const bf16*)down, scale, starts, ids, (float*)workspace, ldx,
                      m * ldv, (int)m, (int)x_cols, (int)rank, (int)ldv, (int)requests,
                      (int)adapters, (int)lora_items(m, requests), (int)pieces, 1};
    const int nr = rank <= 32 ? 1 : rank <= 64 ? 2 : 4;
    d.blocks = (int)((rank + 32 * nr - 1) / (32 * nr));
    const int64_t grid = (int64_t)d.items * d.pieces * d.blocks;
    DLT_REQUIRE(grid < (1LL << 31), DIFFLET_EUNSUPPORTED, "%s: too many tiles", name);
    const dim3 g((unsigned)grid), b(256);
    if (lora_wide(m, requests)) {
      if (nr == 1) hipLaunchKernelGGL((lora_down_wide_kernel<1, 4>), g, b, 0, s, d);
      else if (nr == 2) hipLaunchKernelGGL((lora_down_wide_kernel<2, 3>), g, b, 0, s, d);
      else hipLaunchKernelGGL((lora_down_wide_kernel<4, 4>), g, b, 0, s, d);
    } else if (nr == 1) {
      hipLaunchKernelGGL((lora_down_kernel<1>), g, b, 0, s, d);
    } else if (nr == 2) {
      hipLaunchKernelGGL((lora_down_kernel<2>), g, b, 0, s, d);
    } else {
      hipLaunchKernelGGL((lora_down_kernel<4>), g, b, 0, s, d);
    }
    const int st = dlt_check_launch(name);
    if (st != DIFFLET_OK) return st;
  } else {
    lora.requests = 0;
  }
  difflet_gemm_problem q = {};
  q.a = a;
  q.lda = lda;
  q.w = w;
  q.ldw = ldw;
  q.c = c;
  q.ldc = ldc;
  q.bias = bias;
  q.a_scale = a_scale;
  q.w_scale = w_scale;
  q.m = m;
  q.rows_per_batch = m;
  const int64_t rest = workspace_bytes - vb;
  return gemm_lora(kind, q, n, k, rest > 0 ? (uint8_t*)workspace + vb : nullptr, rest > 0 ? rest : 0,
                   s, lora);
}
