// Cross attention over packed requests: the rows of request i attend to the states of its own
// encoder, out = softmax(q k^T scale) v over keys [k_starts[i], k_starts[i + 1]) for rows
// [q_starts[i], q_starts[i + 1]), head_dim 64 or 128, bf16 or fp16, fp32 statistics and sums, one
// pass over the keys. The query heads of a key head are extra rows: row r of a request's r-space
// is token r / group, head r % group, so a tile reads its keys once for all of them.
//
// A workgroup takes a tile of 128 such rows (four wavefronts of 32) of one request and key head
// and finds them itself from the row numbers on the device: the host knows only bounds, and a
// captured graph follows new lengths. Scores are computed transposed (S^T = K Q^T, 32x32x16), so
// the statistics of a row live in two lanes and P feeds the second product from registers, as in
// attention.hip. Keys come in tiles of 64 through two LDS buffers, K row-major, V transposed while
// it is written. Buffer ranges end with the request's last key: rows of the next request or past
// the tensor read as zero, whatever lies there.
//
// Few tiles (single tokens, short prompts): a request's keys are cut into `pieces`, each with
// statistics of its own, joined by a second kernel in the order of the pieces.
#include <float.h>

#include <algorithm>

#include "attention.hpp"
#include "packed.hpp"

namespace dlt {

struct PackedAttnArgs {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* o;
  int64_t qs[2], ks[2], vs[2], os[2];  // element strides: row, head
  const int32_t* q_starts;
  const int32_t* k_starts;
  int requests, rows_q, rows_k, kv_heads, group;
  int items;       // tiles per key head, at most
  int pieces;      // of a request's keys
  int zero_rest;   // rows of no request come out zero (else are not written)
  float scale_log2;  // |scale| log2(e)
  uint32_t q_sign;   // 0x80008000 for a negative scale
  float* part;       // [pieces][rows_q][heads][D] unnormalized sums (pieces > 1)
  f32x2* stats;      // [pieces][rows_q][heads]: running maximum (scaled), sum
};

constexpr int PA_ROWS = 128, PA_KEYS = 64;
constexpr int PA_VT = PA_KEYS * 2 + 16;  // bytes per V^T row

template <typename T, int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void packed_attn_kernel(const PackedAttnArgs a) {
  typedef typename MfmaT<T>::frag frag;
  constexpr int KP = D * 2 + 16, NC = D / 16, NDT = D / 32, KCH = D / 8;
  __shared__ __attribute__((aligned(16))) uint8_t sk[2][PA_KEYS * KP];
  __shared__ __attribute__((aligned(16))) uint8_t sv[2][D * PA_VT];
  auto kofs = [](int row, int chunk) { return row * KP + (chunk << 4); };
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, g = lane >> 5;

  // ids go round the 8 XCDs: each takes a run of (key head, tile), the tiles of a head side by
  // side, so a request's keys stay in one L2
  int id = blockIdx.x;
  if ((gridDim.x & 7) == 0) id = (id & 7) * (gridDim.x >> 3) + (id >> 3);
  const int item = id % a.items;
  const int hp = id / a.items;
  const int piece = SPLIT ? hp % a.pieces : 0;
  const int hk = SPLIT ? hp / a.pieces : hp;
  const PackedItem it = packed_item(a.q_starts, a.requests, a.rows_q, a.group, PA_ROWS,
                                    a.zero_rest != 0, item);
  if (it.req < 0) return;
  int kbeg = 0, keys = 0;
  if (it.req < a.requests) {
    kbeg = packed_start(a.k_starts, it.req, a.rows_k);
    keys = max(packed_start(a.k_starts, it.req + 1, a.rows_k) - kbeg, 0);
  }
  int j_beg = 0, j_end = keys;
  if (SPLIT) {
    const int tiles = (keys + PA_KEYS - 1) / PA_KEYS, per = (tiles + a.pieces - 1) / a.pieces;
    j_beg = min(piece * per * PA_KEYS, keys);
    j_end = min(j_beg + per * PA_KEYS, keys);
  }

  // this lane's row of the request
  const int r = it.tile * PA_ROWS + wave * 32 + col;
  const int tok = r / a.group, head = hk * a.group + (r - tok * a.group);
  const bool there = (uint32_t)tok < (uint32_t)it.rows;
  const int64_t row = it.row0 + tok;

  frag qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (there)
      raw = *reinterpret_cast<const u32x4*>(a.q + (row * a.qs[0] + head * a.qs[1] + c * 16 + g * 8) * 2);
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[e] ^= a.q_sign;
    qf[c] = __builtin_bit_cast(frag, raw);
  }

  const uint8_t* kp = a.k + ((int64_t)kbeg * a.ks[0] + hk * a.ks[1]) * 2;
  const uint8_t* vp = a.v + ((int64_t)kbeg * a.vs[0] + hk * a.vs[1]) * 2;
  const int64_t krow = a.ks[0] * 2, vrow = a.vs[0] * 2;
  constexpr int KRI = 256 / KCH, NKI = PA_KEYS / KRI;  // K rows per pass, passes
  const int kr = tid / KCH, kc = tid % KCH;
  const int vkg = tid & 15, vdg = tid >> 4;
  const bool v_on = vdg < D / 8;
  const int vt_pos = vt_quad_pos(vkg) * 8;
  u32x4 gk[NKI], gv[4];
  auto load_tile = [&](int j0) {  // the range ends with the last key's channels
    const int n = min(j_end - j0, PA_KEYS);
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kp + j0 * krow, (uint32_t)((n - 1) * krow + D * 2));
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(vp + j0 * vrow, (uint32_t)((n - 1) * vrow + D * 2));
#pragma unroll
    for (int i = 0; i < NKI; ++i) {
      const int key = kr + KRI * i;
      gk[i] = buf_load16(rk, key < n ? (uint32_t)(key * krow) + kc * 16 : 0xfffffff0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = vkg * 4 + i;
      gv[i] = v_on ? buf_load16(rv, key < n ? (uint32_t)(key * vrow) + vdg * 16 : 0xfffffff0u)
                   : u32x4{0u, 0u, 0u, 0u};
    }
  };
  auto store_tile = [&](int st) {
#pragma unroll
    for (int i = 0; i < NKI; ++i) *reinterpret_cast<u32x4*>(&sk[st][kofs(kr + KRI * i, kc)]) = gk[i];
    if (!v_on) return;
#pragma unroll
    for (int d = 0; d < 8; ++d) {  // the 4 keys' values of a channel side by side
      const int w = d >> 1, sh = (d & 1) * 16;
      const uint32_t k0 = (gv[0][w] >> sh) & 0xffffu, k1 = (gv[1][w] >> sh) & 0xffffu;
      const uint32_t k2 = (gv[2][w] >> sh) & 0xffffu, k3 = (gv[3][w] >> sh) & 0xffffu;
      *reinterpret_cast<u32x2*>(&sv[st][(vdg * 8 + d) * PA_VT + vt_pos]) =
          u32x2{k0 | (k1 << 16), k2 | (k3 << 16)};
    }
  };

  f32x16 acc[NDT];
#pragma unroll
  for (int i = 0; i < NDT; ++i) acc[i] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  if (j_beg < j_end) {
    load_tile(j_beg);
    store_tile(0);
  }
  __syncthreads();
  for (int j0 = j_beg, st = 0; j0 < j_end; j0 += PA_KEYS, st ^= 1) {
    const bool more = j0 + PA_KEYS < j_end;
    if (more) load_tile(j0 + PA_KEYS);
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c)
        s[t] = MfmaT<T>::mma(*reinterpret_cast<const frag*>(&sk[st][kofs(t * 32 + col, c * 2 + g)]),
                             qf[c], s[t]);
    }
    if (j0 + PA_KEYS > j_end) {  // keys past the request's last do not exist
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (j0 + t * 32 + (v >> 2) * 8 + g * 4 + (v & 3) >= j_end) s[t][v] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[t][v]);
    mx = pair_max(mx);
    const float m_new = fmaxf(m_run, mx * a.scale_log2);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    m_run = m_new;
    float ls = 0.f;
    uint32_t pp[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][v], a.scale_log2, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][v + 1], a.scale_log2, -m_use));
        ls += p0 + p1;
        pp[t][v >> 1] = MfmaT<T>::pack2(p0, p1);
      }
    l_run = l_run * alpha + ls;
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int i = 0; i < NDT; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][v] *= alpha;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        u32x4 pb;
#pragma unroll
        for (int u = 0; u < 4; ++u) pb[u] = pp[t][hh * 4 + u];
        const frag pf = __builtin_bit_cast(frag, pb);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
          acc[dt] = MfmaT<T>::mma(*reinterpret_cast<const frag*>(
                                      &sv[st][(dt * 32 + col) * PA_VT + (t * 32 + hh * 16 + g * 8) * 2]),
                                  pf, acc[dt]);
      }
    if (more) store_tile(st ^ 1);
    __syncthreads();
  }

  // lane: its row, channels dt * 32 + (v / 4) * 8 + 4 g + v % 4
  const float l = pair_sum(l_run);
  if (!there) return;
  if constexpr (SPLIT) {
    const int64_t at = ((int64_t)piece * a.rows_q + row) * ((int64_t)a.kv_heads * a.group) + head;
    if (g == 0) a.stats[at] = f32x2{m_run, j_beg < j_end ? l : -1.0f};
    if (j_beg >= j_end) return;  // no keys: the join reads no sums there
    float* p = a.part + at * D;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(p + dt * 32 + u * 8 + g * 4) =
            f32x4{acc[dt][4 * u], acc[dt][4 * u + 1], acc[dt][4 * u + 2], acc[dt][4 * u + 3]};
  } else {
    const float inv = keys == 0 ? 0.f : 1.0f / l;  // no keys: zeros
    T* op = reinterpret_cast<T*>(a.o) + row * a.os[0] + head * a.os[1];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<u32x2*>(op + dt * 32 + u * 8 + g * 4) =
            u32x2{MfmaT<T>::pack2(acc[dt][4 * u] * inv, acc[dt][4 * u + 1] * inv),
                  MfmaT<T>::pack2(acc[dt][4 * u + 2] * inv, acc[dt][4 * u + 3] * inv)};
  }
}

// The pieces of a row joined: a wavefront per (row, head). A piece without keys has sum -1 and no
// stored output; a row without any is zero. (A sum of 0, all scores -inf, gives NaN as it does
// in one piece.)
template <typename T, int D>
__global__ __launch_bounds__(256) void packed_attn_join(const PackedAttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t heads = (int64_t)a.kv_heads * a.group;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t all = a.rows_q * heads;
  if (at >= all) return;
  const int64_t row = at / heads, head = at - row * heads;
  if (!a.zero_rest && !packed_covers(a.q_starts, a.requests, a.rows_q, (int)row)) return;
  float m = -INFINITY;
  for (int p = 0; p < a.pieces; ++p) {
    const f32x2 s = a.stats[p * all + at];
    if (!(s[1] < 0.f)) m = fmaxf(m, s[0]);
  }
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[D / 64] = {};
  bool any = false;
  for (int p = 0; p < a.pieces; ++p) {
    const f32x2 s = a.stats[p * all + at];
    if (s[1] < 0.f) continue;
    any = true;
    const float w = __builtin_amdgcn_exp2f(s[0] - m_use);
    l += w * s[1];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] += w * a.part[(p * all + at) * D + i * 64 + lane];
  }
  const float inv = any ? 1.0f / l : 0.f;
  T* op = reinterpret_cast<T*>(a.o) + row * a.os[0] + head * a.os[1];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) Elt<T>::store(op + i * 64 + lane, o[i] * inv);
}

static int packed_items(int64_t rows_q, int64_t requests, int64_t group, int64_t rows) {
  return (int)((rows_q * group + rows - 1) / rows + requests + 2);
}

// Pieces per request: enough workgroups to give every compute unit a few, as long as a piece keeps
// two tiles of keys on average and the pieces' sums stay small beside the launch.
static int packed_pieces(int64_t rows_q, int64_t rows_k, int64_t requests, int64_t kv_heads,
                         int64_t group, int64_t head_dim) {
  const int64_t blocks = packed_items(rows_q, requests, group, PA_ROWS) * kv_heads;
  if (blocks >= 256) return 1;
  int64_t n = (1024 + blocks - 1) / blocks;
  n = std::min(n, (rows_k + 2 * PA_KEYS - 1) / (2 * PA_KEYS));
  n = std::min<int64_t>(n, (16 << 20) / std::max<int64_t>(1, rows_q * kv_heads * group * head_dim * 4));
  return (int)std::max<int64_t>(1, n);
}
static int64_t packed_stats_bytes(int64_t pieces, int64_t rows_q, int64_t heads) {
  return (pieces * rows_q * heads * 8 + 255) / 256 * 256;
}

}  // namespace dlt

using namespace dlt;

extern "C" int64_t difflet_rocm_packed_attention_workspace_bytes(int64_t rows_q, int64_t rows_k,
                                                                 int64_t requests,
                                                                 int64_t kv_heads, int64_t group,
                                                                 int64_t head_dim) {
  if (rows_q <= 0 || rows_k <= 0 || requests <= 0 || kv_heads <= 0 || group <= 0 ||
      rows_q * group >= (1LL << 30) || requests >= (1LL << 24) || kv_heads * group > 65536)
    return 0;
  const int64_t n = packed_pieces(rows_q, rows_k, requests, kv_heads, group, head_dim);
  if (n <= 1) return 0;
  return packed_stats_bytes(n, rows_q, kv_heads * group) + n * rows_q * kv_heads * group * head_dim * 4;
}

extern "C" int difflet_rocm_packed_attention(
    const void* q, const void* k, const void* v, void* o, int dtype, int64_t rows_q, int64_t rows_k,
    int64_t kv_heads, int64_t group, int64_t head_dim, const int64_t* q_strides,
    const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
    const int32_t* q_starts, const int32_t* k_starts, int64_t requests, float scale, int zero_rest,
    void* workspace, int64_t workspace_bytes, difflet_stream_t stream) {
  const char* name = "packed_attention";
  DLT_REQUIRE(rows_q >= 0 && rows_k >= 0 && requests >= 0 && kv_heads > 0 && group > 0,
              DIFFLET_EINVAL, "%s: bad shape", name);
  DLT_REQUIRE(dtype == DIFFLET_BF16 || dtype == DIFFLET_F16, DIFFLET_EUNSUPPORTED,
              "%s: bf16 or fp16, not dtype %d", name, dtype);
  DLT_REQUIRE(head_dim == 64 || head_dim == 128, DIFFLET_EUNSUPPORTED,
              "%s: head_dim %lld (64 or 128)", name, (long long)head_dim);
  DLT_REQUIRE(rows_q * group < (1LL << 30) && rows_k < (1LL << 30) && requests < (1LL << 24) &&
                  kv_heads * group <= 65536,
              DIFFLET_EUNSUPPORTED, "%s: too large", name);
  DLT_REQUIRE(scale - scale == 0.0f, DIFFLET_EINVAL, "%s: scale must be finite", name);
  if (rows_q == 0) return DIFFLET_OK;
  DLT_REQUIRE(q && o && q_strides && k_strides && v_strides && o_strides && q_starts && k_starts &&
                  (rows_k == 0 || (k && v)),
              DIFFLET_EINVAL, "%s: null pointer", name);
  for (int i = 0; i < 2; ++i)
    DLT_REQUIRE(q_strides[i] % 8 == 0 && k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0 &&
                    o_strides[i] % 4 == 0,
                DIFFLET_EINVAL, "%s: rows and heads must start on 16 bytes (the output's on 8)", name);
  DLT_REQUIRE(k_strides[0] >= 0 && v_strides[0] >= 0 && k_strides[0] < (1LL << 24) &&
                  v_strides[0] < (1LL << 24),
              DIFFLET_EUNSUPPORTED, "%s: key rows more than 32 MB apart", name);
  DLT_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((uintptr_t)o & 7) == 0,
              DIFFLET_EINVAL, "%s: misaligned pointers", name);
  PackedAttnArgs a = {};
  a.q = (const uint8_t*)q;
  a.k = (const uint8_t*)k;
  a.v = (const uint8_t*)v;
  a.o = (uint8_t*)o;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q_strides[i];
    a.ks[i] = k_strides[i];
    a.vs[i] = v_strides[i];
    a.os[i] = o_strides[i];
  }
  a.q_starts = q_starts;
  a.k_starts = k_starts;
  a.requests = (int)requests;
  a.rows_q = (int)rows_q;
  a.rows_k = (int)rows_k;
  a.kv_heads = (int)kv_heads;
  a.group = (int)group;
  a.zero_rest = zero_rest;
  // a scale of 0 would turn the -inf of keys that do not exist into NaN; the smallest normal float
  // weighs any real score as 0 does
  a.scale_log2 = std::max((scale < 0 ? -scale : scale) * LOG2E, FLT_MIN);
  a.q_sign = scale < 0 ? 0x80008000u : 0u;
  a.items = packed_items(rows_q, requests, group, PA_ROWS);
  a.pieces = rows_k > 0 && requests > 0
                 ? packed_pieces(rows_q, rows_k, requests, kv_heads, group, head_dim) : 1;
  if (a.pieces > 1) {
    const int64_t stats = packed_stats_bytes(a.pieces, rows_q, kv_heads * group);
    const int64_t need = stats + a.pieces * rows_q * kv_heads * group * head_dim * 4;
    if (!workspace || workspace_bytes < need) {
      a.pieces = 1;  // without room for the pieces' sums the keys stay whole
    } else {
      DLT_REQUIRE(((uintptr_t)workspace & 255) == 0, DIFFLET_EINVAL,
                  "%s: workspace must be 256-byte aligned", name);
      a.stats = (f32x2*)workspace;
      a.part = (float*)((uint8_t*)workspace + stats);
    }
  }
  const int64_t blocks = (int64_t)a.items * kv_heads * a.pieces;
  DLT_REQUIRE(blocks < (1LL << 31), DIFFLET_EUNSUPPORTED, "%s: too many tiles", name);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks), block(256);
  auto go = [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    if (a.pieces == 1) {
      hipLaunchKernelGGL((packed_attn_kernel<T, D, false>), grid, block, 0, s, a);
      return;
    }
    hipLaunchKernelGGL((packed_attn_kernel<T, D, true>), grid, block, 0, s, a);
    const int64_t all = rows_q * kv_heads * group;
    hipLaunchKernelGGL((packed_attn_join<T, D>), dim3((unsigned)((all + 3) / 4)), block, 0, s, a);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (dtype == DIFFLET_BF16) {
    if (head_dim == 64) go(bf16{}, D64{});
    else go(bf16{}, D128{});
  } else {
    if (head_dim == 64) go(f16{}, D64{});
    else go(f16{}, D128{});
  }
  return dlt_check_launch(name);
}
