// Cross attention over packed requests: the rows of request i attend to the states of its own
// encoder, out = softmax(q k^T scale) v over keys [k_starts[i], k_starts[i + 1]) for rows
// [q_starts[i], q_starts[i + 1]), head_dim 64 or 128, bf16 or fp16, fp32 statistics and sums, one
// pass over the keys. The query heads of a key head are extra rows: row r of a request's r-space
// is token r / group, head r % group, so a tile reads its keys once for all of them.
//
// A workgroup finds its tile of such rows (of one request and key head) itself, from the row numbers
// on the device: the host knows only bounds, and a captured graph follows new lengths. Scores are
// computed transposed (S^T = K Q^T, 32x32x16), so the statistics of a row live in two lanes and P
// feeds the second product from registers, as in attention.hip. Buffer ranges end with the
// request's last key: rows of the next request or past the tensor read as zero, whatever lies there.
//
// Which one runs is packed_plan's choice.
// packed_attn_wide_kernel: 256 rows, 64 a wavefront, where there are many (described beside it).
// packed_attn_kernel: 128 rows (four wavefronts of 32), tiles of 64 keys through two LDS buffers, K
// row-major, V transposed while it is written.
// packed_attn_few_kernel: few rows a request (single tokens): 32 rows, whose four wavefronts take 32
// keys each of tiles of 128 and join what they have in LDS.
//
// Few tiles: the launch has a fixed number of workgroups, which cut the requests' keys into chunks of
// about one length, one or two a workgroup (the length follows from the row numbers on the
// device). A row tile of several chunks leaves the unnormalized sums of each and their statistics in
// the workspace, joined by packed_attn_join in the order of the chunks. 16 single tokens over 0 to
// 8000 states (4 key heads): 28 + 6 us with every request's keys in 12 pieces, 24 + 5.7 so.
#include <float.h>

#include <algorithm>

#include "attention.hpp"
#include "packed.hpp"


namespace dlt {

int gemm_device_cus();  // compute units of the current device (gemm.hip)

struct PackedAttnArgs {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* o;
  int64_t qs[2], ks[2], vs[2], os[2];  // element strides: row, head
  const int32_t* q_starts;
  const int32_t* k_starts;
  int requests, rows_q, rows_k, kv_heads, group;
  int items;         // row tiles per key head, at most
  int zero_rest;     // rows of no request come out zero (else are not written)
  uint32_t group_m;  // conv_magic(group)
  float scale_log2;  // |scale| log2(e)
  uint32_t q_sign;   // 0x80008000 for a negative scale
  int groups;           // workgroups of a launch that cuts keys into chunks (0: whole keys)
  int slots;            // of the workspace: row numbers out of order could ask for more
  float* part;          // [slots][block][D] unnormalized sums, slot = item
  f32x2* stats;         // [slots][block]: running maximum (scaled), sum; sum -1: a chunk without keys
};

// ------------------------------------------------------------------ the schedule
// A row tile, its request's keys and the chunk of them that runs here. Items count chunks within
// row tiles within requests; an item of key head h is workgroup item `item * kv_heads + h`.
struct PackedWork {
  PackedItem it;
  int kbeg, keys;           // the request's keys
  int chunk, chunks, first; // of the row tile; item of its chunk 0
};

__device__ __forceinline__ void packed_keys(const PackedAttnArgs& a, int i, int& kbeg, int& keys) {
  kbeg = 0, keys = 0;
  if ((uint32_t)i < (uint32_t)a.requests) {
    kbeg = packed_start(a.k_starts, i, a.rows_k);
    keys = max(packed_start(a.k_starts, i + 1, a.rows_k) - kbeg, 0);
  }
}

// The chunks of a launch of at most PACKED_LANES requests, one request a lane: loaded once, every
// item of a workgroup is then found by a ballot.
constexpr int PACKED_LANES = kWave - 2;
template <int BLOCK, int KEYT> struct PackedChunks {
  int r0, len, kbeg, keys;  // the lane's request (or rows of none)
  int tiles, chunks, upto;  // row tiles, chunks of each; items up to and with the lane's
  // every request's keys in one chunk
  __device__ __forceinline__ void load(const PackedAttnArgs& a) {
    const int i = threadIdx.x & (kWave - 1);
    packed_rows(a.q_starts, a.requests, a.rows_q, a.zero_rest != 0, i, r0, len);
    packed_keys(a, i, kbeg, keys);
    tiles = (len * a.group + BLOCK - 1) / BLOCK;
    chunks = 1;
    upto = wave_prefix(tiles);
  }
  __device__ __forceinline__ void scan(const PackedAttnArgs& a) {
    load(a);
    const int kt = (keys + KEYT - 1) / KEYT;
    // key tiles per chunk, so that the chunks of all heads, a last short one for every row tile among
    // them, are one a workgroup (a schedule: every wavefront rounds alike, and that is all it takes)
    const float work = wave_sum((float)tiles * (float)kt) * (float)a.kv_heads;
    const float spare = (float)a.groups - wave_sum((float)tiles) * (float)a.kv_heads;
    const int per = max(1, (int)ceilf(work / fmaxf(spare, 0.25f * (float)a.groups)));
    chunks = max(1, (kt + per - 1) / per);
    upto = wave_prefix(tiles * chunks);
  }
  // the row tiles of lane l's request
  __device__ __forceinline__ PackedWork work_of(const PackedAttnArgs& a, int l) const {
    PackedWork w;
    w.it.req = min(l, a.requests);
    w.it.tile = w.chunk = 0;
    w.it.row0 = __builtin_amdgcn_readlane(r0, l);
    w.it.rows = __builtin_amdgcn_readlane(len, l);
    w.kbeg = __builtin_amdgcn_readlane(kbeg, l);
    w.keys = __builtin_amdgcn_readlane(keys, l);
    w.chunks = __builtin_amdgcn_readlane(chunks, l);
    w.first = __builtin_amdgcn_readlane(upto - tiles * chunks, l);
    return w;
  }
  __device__ __forceinline__ PackedWork item(const PackedAttnArgs& a, int n) const {
    const uint64_t past = __ballot(upto > n);
    if (!past) {
      PackedWork w = {};
      w.it.req = -1;
      return w;
    }
    PackedWork w = work_of(a, __ffsll((unsigned long long)past) - 1);
    w.it.tile = (n - w.first) / w.chunks;
    w.chunk = (n - w.first) % w.chunks;
    return w;
  }
};

// SPLIT: item `item` of the chunks, else of the row tiles, each with all of its keys.
template <bool SPLIT, typename Chunks>
__device__ __forceinline__ PackedWork packed_work(const PackedAttnArgs& a, const Chunks& chunks,
                                                  int block, int item) {
  if constexpr (SPLIT) return chunks.item(a, item);
  PackedWork w = {};
  w.it = packed_item(a.q_starts, a.requests, a.rows_q, a.group, block, a.zero_rest != 0, item);
  w.chunks = 1;
  if (w.it.req >= 0) packed_keys(a, w.it.req, w.kbeg, w.keys);
  return w;
}

// Keys [j_beg, j_end) of the request that chunk `chunk` of `chunks` covers.
__device__ __forceinline__ void packed_range(const PackedWork& w, int key_tile, int& j_beg,
                                             int& j_end) {
  const int cut = ((w.keys + key_tile - 1) / key_tile + w.chunks - 1) / w.chunks * key_tile;
  j_beg = min(w.chunk * cut, w.keys);
  j_end = min(j_beg + cut, w.keys);
}

// ------------------------------------------------------------------ pieces of a tile
// Q fragments of a lane: its row, channels 16 c + 8 g .. + 8.
template <typename T, int D>
__device__ __forceinline__ void packed_load_q(const PackedAttnArgs& a, bool there, int64_t row,
                                              int head, int g, typename MfmaT<T>::frag (&qf)[D / 16]) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (there)
      raw = *reinterpret_cast<const u32x4*>(a.q + (row * a.qs[0] + head * a.qs[1] + c * 16 + g * 8) * 2);
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[e] ^= a.q_sign;
    qf[c] = __builtin_bit_cast(typename MfmaT<T>::frag, raw);
  }
}

// Keys and values of a tile of KEYS keys by 256 threads: from memory into registers (zero past the
// n keys there are), from there into LDS, K rows of KP bytes, V^T rows of VT bytes with the key
// quads of each 16 in vt_quad_pos's order.
template <int D, int KEYS> struct PackedTile {
  static constexpr int KP = D * 2 + 16, VT = KEYS * 2 + 16, KCH = D / 8;
  static constexpr int KRI = 256 / KCH, NKI = KEYS / KRI;              // K rows per pass, passes
  static constexpr int VQ = KEYS / 4, VDP = 256 / VQ;                  // key quads, channel groups
  static constexpr int NVI = D / 8 > VDP ? D / 8 / VDP : 1;            // a pass; passes
  u32x4 k[NKI], v[NVI][4];
  __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int64_t krow,
                                       int64_t vrow, int n) {
    const int tid = threadIdx.x;
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(kp, (uint32_t)((n - 1) * krow + D * 2));
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(vp, (uint32_t)((n - 1) * vrow + D * 2));
    constexpr uint32_t kOut = 0xfffffff0u;  // past every range
#pragma unroll
    for (int i = 0; i < NKI; ++i) {
      const int key = tid / KCH + KRI * i;
      k[i] = buf_load16(rk, key < n ? (uint32_t)(key * krow) + (tid % KCH) * 16 : kOut);
    }
#pragma unroll
    for (int p = 0; p < NVI; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = (tid % VQ) * 4 + i, dg = p * VDP + tid / VQ;
        v[p][i] = buf_load16(rv, key < n && dg < D / 8 ? (uint32_t)(key * vrow) + dg * 16 : kOut);
      }
  }
  __device__ __forceinline__ void store(uint8_t* sk, uint8_t* sv) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < NKI; ++i)
      *reinterpret_cast<u32x4*>(sk + (tid / KCH + KRI * i) * KP + (tid % KCH) * 16) = k[i];
    const int pos = vt_quad_pos(tid % VQ) * 8;
#pragma unroll
    for (int p = 0; p < NVI; ++p) {
      const int dg = p * VDP + tid / VQ;
      if (dg >= D / 8) continue;
#pragma unroll
      for (int d = 0; d < 8; ++d) {  // the 4 keys' values of a channel side by side
        const int w = d >> 1, sh = (d & 1) * 16;
        const uint32_t k0 = (v[p][0][w] >> sh) & 0xffffu, k1 = (v[p][1][w] >> sh) & 0xffffu;
        const uint32_t k2 = (v[p][2][w] >> sh) & 0xffffu, k3 = (v[p][3][w] >> sh) & 0xffffu;
        *reinterpret_cast<u32x2*>(sv + (dg * 8 + d) * VT + pos) = u32x2{k0 | (k1 << 16), k2 | (k3 << 16)};
      }
    }
  }
};

// Online softmax of a lane's row and the second product, over NT x 32 keys from key0 of LDS on.
// Scores stay raw (p = exp2(s c - m), m in scaled units, c > 0); keys from `left` on do not exist.
template <typename T, int D> struct PackedRow {
  typedef typename MfmaT<T>::frag frag;
  f32x16 acc[D / 32];
  float m_run, l_run;
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
    m_run = -INFINITY, l_run = 0.f;
  }
  template <int NT>
  __device__ __forceinline__ void step(const frag (&qf)[D / 16], const uint8_t* sk, int kp,
                                       const uint8_t* sv, int vt, int key0, int left, float c) {
    const int lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
    f32x16 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] = f32x16{};
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        s[t] = MfmaT<T>::mma(
            *reinterpret_cast<const frag*>(sk + (key0 + t * 32 + col) * kp + (i * 2 + g) * 16), qf[i],
            s[t]);
    }
    if (left < NT * 32) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (t * 32 + (v >> 2) * 8 + g * 4 + (v & 3) >= left) s[t][v] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[t][v]);
    mx = pair_max(mx);
    const float m_new = fmaxf(m_run, mx * c);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    m_run = m_new;
    float ls = 0.f;
    uint32_t pp[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][v], c, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][v + 1], c, -m_use));
        ls += p0 + p1;
        pp[t][v >> 1] = MfmaT<T>::pack2(p0, p1);
      }
    l_run = l_run * alpha + ls;
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][v] *= alpha;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {  // 16 keys: {4g .. 4g + 3, 8 + 4g .. 8 + 4g + 3}
        u32x4 pb;
#pragma unroll
        for (int u = 0; u < 4; ++u) pb[u] = pp[t][hh * 4 + u];
        const frag pf = __builtin_bit_cast(frag, pb);
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          acc[dt] = MfmaT<T>::mma(*reinterpret_cast<const frag*>(
                                      sv + (dt * 32 + col) * vt + (key0 + t * 32 + hh * 16 + g * 8) * 2),
                                  pf, acc[dt]);
      }
  }
};

// Workgroup barrier after this wavefront's direct-to-LDS loads have landed but for the VM newest.
template <int VM = 0> __device__ __forceinline__ void wide_barrier() {
  static_assert(VM >= 0 && VM < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt(0x0070 | (VM & 15) | ((VM >> 4) << 14));  // vmcnt(VM) lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

// ------------------------------------------------------------------ kernels
constexpr int PA_ROWS = 128, PA_KEYS = 64;

template <typename T, int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void packed_attn_kernel(const PackedAttnArgs a) {
  typedef PackedTile<D, PA_KEYS> Tile;
  __shared__ __attribute__((aligned(16))) uint8_t sk[2][PA_KEYS * Tile::KP];
  __shared__ __attribute__((aligned(16))) uint8_t sv[2][D * Tile::VT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, g = lane >> 5;
  PackedChunks<PA_ROWS, PA_KEYS> chunks;
  if (SPLIT) chunks.scan(a);
  // whole keys: ids go round the 8 XCDs, and each takes a run of (key head, tile), the tiles of a head
  // side by side, so that a request's keys stay in one L2
  int id = blockIdx.x;
  if (!SPLIT && (gridDim.x & 7) == 0) id = (id & 7) * (gridDim.x >> 3) + (id >> 3);
  for (;; id += gridDim.x) {
    const int hk = SPLIT ? id % a.kv_heads : id / a.items;
    const PackedWork w = packed_work<SPLIT>(a, chunks, PA_ROWS, SPLIT ? id / a.kv_heads : id % a.items);
    if (w.it.req < 0 || (SPLIT && id >= a.slots)) return;
    int j_beg, j_end;
    packed_range(w, PA_KEYS, j_beg, j_end);
    const int r = w.it.tile * PA_ROWS + wave * 32 + col;  // this lane's row of the request
    const int tok = r / a.group, head = hk * a.group + (r - tok * a.group);
    const bool there = (uint32_t)tok < (uint32_t)w.it.rows;
    const int64_t row = w.it.row0 + tok;
    typename MfmaT<T>::frag qf[D / 16];
    packed_load_q<T, D>(a, there, row, head, g, qf);
    const uint8_t* kp = a.k + ((int64_t)w.kbeg * a.ks[0] + hk * a.ks[1]) * 2;
    const uint8_t* vp = a.v + ((int64_t)w.kbeg * a.vs[0] + hk * a.vs[1]) * 2;
    const int64_t krow = a.ks[0] * 2, vrow = a.vs[0] * 2;
    Tile tile;
    auto load = [&](int j0) {
      tile.load(kp + j0 * krow, vp + j0 * vrow, krow, vrow, min(j_end - j0, PA_KEYS));
    };
    PackedRow<T, D> st;
    st.reset();
    if (j_beg < j_end) {
      load(j_beg);
      tile.store(sk[0], sv[0]);
    }
    __syncthreads();
    for (int j0 = j_beg, b = 0; j0 < j_end; j0 += PA_KEYS, b ^= 1) {
      const bool more = j0 + PA_KEYS < j_end;
      if (more) load(j0 + PA_KEYS);
      st.template step<2>(qf, sk[b], Tile::KP, sv[b], Tile::VT, 0, j_end - j0, a.scale_log2);
      if (more) tile.store(sk[b ^ 1], sv[b ^ 1]);
      __syncthreads();
    }
    // lane: its row, channels dt * 32 + (v / 4) * 8 + 4 g + v % 4
    const float l = pair_sum(st.l_run);
    if (SPLIT && w.chunks > 1) {
      const int64_t at = (int64_t)id * PA_ROWS + wave * 32 + col;
      if (there && g == 0) a.stats[at] = f32x2{st.m_run, j_beg < j_end ? l : -1.0f};
      if (there && j_beg < j_end) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<f32x4*>(a.part + at * D + dt * 32 + u * 8 + g * 4) =
                f32x4{st.acc[dt][4 * u], st.acc[dt][4 * u + 1], st.acc[dt][4 * u + 2],
                      st.acc[dt][4 * u + 3]};
      }
    } else if (there) {
      const float inv = w.keys == 0 ? 0.f : 1.0f / l;  // no keys: zeros
      T* op = reinterpret_cast<T*>(a.o) + row * a.os[0] + head * a.os[1];
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *reinterpret_cast<u32x2*>(op + dt * 32 + u * 8 + g * 4) =
              u32x2{MfmaT<T>::pack2(st.acc[dt][4 * u] * inv, st.acc[dt][4 * u + 1] * inv),
                    MfmaT<T>::pack2(st.acc[dt][4 * u + 2] * inv, st.acc[dt][4 * u + 3] * inv)};
    }
    if (!SPLIT) return;
  }
}

// Many rows a request: 256 rows a workgroup, 64 a wavefront in two column groups, one workgroup a
// compute unit that walks tile after tile. Attention of many rows to a few hundred keys is bound by
// the matrix cores (at the power they draw, about 1.26 PFLOP/s of the 2.5), if the softmax, the LDS
// and the start and end of each tile stay beside them. On the 128-row kernel a fragment read feeds
// one MFMA (the LDS's 128 bytes a cycle, all of them) and each tile begins and ends by itself. Here a
// fragment feeds two MFMAs, the keys serve 256 rows, and one wavefront overlaps three halves (32
// keys) of its work by itself: while the matrix core runs the scores of half h + 1 and the second
// product of half h - 1, 32 MFMAs, the VALU takes the exponentials of half h. Four wavefronts with
// 512 registers each hold the 128 accumulators, two sets of scores and of P and the rows' Q.
//
// Keys and values come straight from memory into LDS, two tiles of 64 keys each, K rows of D / 8 +
// 1 slots of 16 bytes, V rows of 20 (12 for 64 channels), read through the transposing LDS read; slots
// past the channels are padding that keeps the reads of 16 rows in distinct banks. Tile j's keys are
// read in halves 2j - 1 and 2j, its values in 2j + 1 and 2j + 2, so one barrier a tile, before half
// 2j - 1, publishes K(j) and V(j - 1) and frees the slots of K(j - 1) and V(j - 2), to which K(j + 1)
// and V(j) go. Rows past the request's last key load that key again: their scores are masked to
// -inf and what their P of 0 meets is as finite as the key's own values are. The next row tile's Q
// comes the same way, a quarter of it with each tile of keys, and its first keys under the last half:
// nothing of a tile's start is waited for but what a request of few keys leaves no time for.
//
// Exponentials are relative to a reference that moves to the running maximum when a lane's sum of
// a half reaches the type's limit (the first half always): the statistics cost no maximum on the way.
//
// Rows of Q are fetched whole, 256 bytes a row: read as fragments, 32 rows at the stride of all
// heads share a few sets of the L1, and each line comes four times. For the same reason the result goes
// out through LDS (stored from the accumulators, 32 bytes of 32 rows an instruction, it took
// 5,400 cycles a tile, so 4,000).
//
// Loads issued one by one between the MFMAs instead of in one go before them cost 6 % (their branches
// cut the groups of MFMAs).
//
// 32,768 rows of 40 heads to 64, 128, 256, 512, 1024, 2048 keys: 165, 212, 285, 474, 831, 1474 us
// (0.93 PFLOP/s); tiles of 128 rows: 246, 271, 356, 538, 873, 1575. Of the 49,000 cycles of a tile of 512
// keys its loop takes 37,500; without the exponentials 2048 keys took 1331 us of then 1599, which is
// what the matrix cores and the LDS draw the card's power for.
template <int D> struct WideLds {
  static constexpr int KS = D / 8 + 1, VS = D == 128 ? 20 : 12;  // slots of 16 bytes per row
  static constexpr int KB = 64 * KS * 16, VB = 64 * VS * 16;     // bytes per tile: KS, VS loads of 1 KB
  static constexpr int QB = 64 * D * 2;                          // a wavefront's rows of Q
  static constexpr int QL = QB / 1024, QQ = QL / 4;              // loads of it, a quarter
  static constexpr int STORES = D / 8;                           // of a wavefront's output
  static constexpr int BYTES = 2 * (KB + VB) + 4 * QB + 4 * 4096;
};
constexpr int PW_ROWS = 256;

template <typename T, int D>
__global__ __launch_bounds__(256, 1) void packed_attn_wide_kernel(const PackedAttnArgs a) {
  typedef typename MfmaT<T>::frag frag;
  typedef WideLds<D> L;
  constexpr int NC = D / 16, NDT = D / 32, RPL = D / 8;  // RPL: 16-byte chunks a row
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  uint8_t* qlds = lds + 2 * (L::KB + L::VB) + wave * L::QB;
  auto kbuf = [&](int b) { return lds + b * L::KB; };
  auto vbuf = [&](int b) { return lds + 2 * L::KB + b * L::VB; };

  // the requests, one a lane, and how many row tiles there are up to and with the lane's when those
  // of most keys come first: the launch's last round, which its workgroups share unevenly, is then
  // of short ones, and no tile costs another load to find
  PackedChunks<PW_ROWS, 64> reqs;
  reqs.load(a);
  int upto = 0, tiles = 0;
  for (int l = 0; l < a.requests + 2; ++l) {
    const int k = __builtin_amdgcn_readlane(reqs.keys, l), n = __builtin_amdgcn_readlane(reqs.tiles, l);
    if (k > reqs.keys || (k == reqs.keys && l <= lane)) upto += n;
    tiles += n;
  }
  struct Tile {
    PackedWork w;
    int hk, nt;
  };
  auto find = [&](int64_t n) {
    Tile t = {};
    t.w.it.req = -1;
    if (n >= (int64_t)tiles * a.kv_heads) return t;
    const int64_t end = (int64_t)upto * a.kv_heads, begin = end - (int64_t)reqs.tiles * a.kv_heads;
    const int l = __ffsll((unsigned long long)__ballot(begin <= n && n < end)) - 1;
    t.w = reqs.work_of(a, l);
    const int of = __builtin_amdgcn_readlane(reqs.tiles, l);
    const int in = (int)(n - (int64_t)(__builtin_amdgcn_readlane(upto, l) - of) * a.kv_heads);
    t.hk = in / of;
    t.w.it.tile = in - t.hk * of;
    t.nt = (t.w.keys + 63) / 64;
    return t;
  };
  // load i of a wavefront's rows of Q: RPI rows, the lane's chunk lane % RPL of LDS row r holds chunk
  // (lane % RPL) ^ (r % RPL) of it; rows past the request are its last. A load's offsets cost more
  // than the load, so whole tiles of single heads step from the first one's
  constexpr int RPI = 64 / RPL;
  const bool single = a.group == 1;
  const uint32_t qrow = (uint32_t)(a.qs[0] * 2);
  auto q_offset = [&](const Tile& t, int i, uint32_t tok0) {
    const int r = i * RPI + lane / RPL, last = t.w.it.rows * a.group - 1;
    uint32_t h;
    const uint32_t tok = conv_udiv((uint32_t)min(t.w.it.tile * PW_ROWS + wave * 64 + r, last),
                                   (uint32_t)a.group, a.group_m, h);
    return (tok - tok0) * qrow + h * (uint32_t)(a.qs[1] * 2) + (uint32_t)((lane % RPL) ^ (r & (RPL - 1))) * 16;
  };
  // loads [i0, i1) of it
  auto load_q = [&](const Tile& t, int i0, int i1) {
    const uint32_t tok0 = single ? (uint32_t)(t.w.it.tile * PW_ROWS)
                                 : (uint32_t)(t.w.it.tile * PW_ROWS) / (uint32_t)a.group;
    const uint8_t* p = a.q + (((int64_t)t.w.it.row0 + tok0) * a.qs[0] + (int64_t)t.hk * a.group * a.qs[1]) * 2;
    const i32x4_t r = rsrc_words(p, 0xffffffffu);
    if (single && (t.w.it.tile + 1) * PW_ROWS <= t.w.it.rows) {
      // chunk (lane % RPL) ^ (row % RPL): the row's part of it below RPI is the lane's, above i's
      const uint32_t off = (uint32_t)(wave * 64 + lane / RPL) * qrow;
#pragma unroll 4
      for (int i = i0; i < i1; ++i)
        dma16s(r, qlds + i * 1024,
               off + (uint32_t)((lane % RPL) ^ ((i * RPI + lane / RPL) & (RPL - 1))) * 16,
               (uint32_t)(i * RPI) * qrow);
    } else {
#pragma unroll 1
      for (int i = i0; i < i1; ++i)
        dma16(r, lds + __builtin_amdgcn_readfirstlane((int)(qlds - lds) + i * 1024), q_offset(t, i, tok0));
    }
  };
  // this wavefront's loads of a tile of K or V: slot (wave + 4 i) * 64 + lane of SLOTS a row is a row
  // and a chunk of it, at the same offsets for every whole tile. Rows past the last key read that
  // key again
  auto key_offset = [&](int i, int slots, uint32_t row, int n) {
    const int sl = (wave + 4 * i) * 64 + lane;
    return (uint32_t)min(sl / slots, n - 1) * row + (uint32_t)min(sl % slots, RPL - 1) * 16;
  };
  uint32_t ko[(L::KS + 3) / 4], vo[(L::VS + 3) / 4];
#pragma unroll
  for (int i = 0; i < (L::KS + 3) / 4; ++i) ko[i] = key_offset(i, L::KS, (uint32_t)(a.ks[0] * 2), 64);
#pragma unroll
  for (int i = 0; i < (L::VS + 3) / 4; ++i) vo[i] = key_offset(i, L::VS, (uint32_t)(a.vs[0] * 2), 64);
  auto load_keys = [&](const Tile& t, const uint8_t* base, const int64_t (&st)[2], int j, uint8_t* dst,
                       const auto& off, auto slots) {
    constexpr int S = decltype(slots)::value;
    if (j >= t.nt) return;
    const int n = min(t.w.keys - j * 64, 64);
    const uint32_t row = (uint32_t)(st[0] * 2);
    const uint8_t* p = base + (((int64_t)t.w.kbeg + j * 64) * st[0] + t.hk * st[1]) * 2;
    const i32x4_t r = rsrc_words(p, (uint32_t)(n - 1) * row + D * 2);
    if (n == 64) {
#pragma unroll
      for (int i = 0; i < (S + 3) / 4; ++i)
        if (wave + 4 * i < S) dma16(r, dst + (wave + 4 * i) * 1024, off[i]);
    } else {
#pragma unroll 1
      for (int i = 0; i < (S + 3) / 4; ++i)
        if (wave + 4 * i < S)
          dma16(r, lds + __builtin_amdgcn_readfirstlane((int)(dst - lds) + (wave + 4 * i) * 1024),
                key_offset(i, S, row, n));
    }
  };
  auto load_k = [&](const Tile& t, int j, int b) {
    load_keys(t, a.k, a.ks, j, kbuf(b), ko, std::integral_constant<int, L::KS>{});
  };
  auto load_v = [&](const Tile& t, int j, int b) {
    load_keys(t, a.v, a.vs, j, vbuf(b), vo, std::integral_constant<int, L::VS>{});
  };

  // a round of the launch's workgroups takes consecutive (key head, tile) pairs, those of an XCD
  // consecutive ones among them: neighbours read the same keys through one L2
  const int per = gridDim.x >> 3;
  int64_t id = (gridDim.x & 7) == 0 ? (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3) : blockIdx.x;
  Tile t = find(id);
  bool first = true;
  if (t.w.it.req < 0) return;
  int kb = 0;  // K(j) and V(j) of this row tile are in slots (kb + j) % 2
  load_k(t, 0, 0);
  load_q(t, 0, L::QL);
  load_k(t, 1, 1), load_v(t, 0, 0);
  for (;;) {
    id += gridDim.x;
    const Tile next = find(id);
    const int nt = t.nt, keys = t.w.keys;
    frag qf[2][NC];
    f32x16 acc[2][NDT];
    float m_run[2], l_run[2];
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      m_run[gr] = 0.f, l_run[gr] = 0.f;
#pragma unroll
      for (int i = 0; i < NDT; ++i) acc[gr][i] = f32x16{};
    }
    // V^T fragments: lane l of a 16-lane group supplies key row 4 g + (l / 4) % 4 of 8 keys and 4
    // channels; it receives channel l % 32 of keys {4g .. 4g + 3} and {8 + 4g .. 8 + 4g + 3}
    const uint32_t vl = (uint32_t)((4 * g + ((lane >> 2) & 3)) * (L::VS * 16) +
                                   32 * ((lane >> 4) & 1) + 8 * (lane & 3));
    auto v_frag = [&](const uint8_t* sv, int half, int f) {
      const int hh = f / NDT, dt = f % NDT;
      const uint8_t* p = sv + vl + (half * 32 + hh * 16) * (L::VS * 16) + dt * 64;
      const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)p);
      const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(p + 8 * (L::VS * 16)));
      const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
      return __builtin_bit_cast(frag, u32x4{l2[0], l2[1], h2[0], h2[1]});
    };
    auto k_frag = [&](const uint8_t* sk, int half, int c) {
      return *reinterpret_cast<const frag*>(sk + (half * 32 + col) * (L::KS * 16) + (2 * c + g) * 16);
    };
    auto p_frag = [](const uint32_t (&pp)[8], int hh) {
      return __builtin_bit_cast(frag, u32x4{pp[hh * 4], pp[hh * 4 + 1], pp[hh * 4 + 2], pp[hh * 4 + 3]});
    };
    const float cmul = a.scale_log2;
    // One half h: exponentials of its scores `sc` into `pc` beside, with QK, the scores of half h + 1
    // (half kh of the keys in sk) into `sn` and, with PV, the second product of half h - 1 (`pl`, half
    // vh of the values in sv).
    auto half_step = [&](auto qk, auto pv, f32x16 (&sc)[2], f32x16 (&sn)[2], uint32_t (&pl)[2][8],
                         uint32_t (&pc)[2][8], const uint8_t* sk, int kh, const uint8_t* sv, int vh,
                         int left) {
      constexpr bool QK = decltype(qk)::value, PV = decltype(pv)::value;
      if (left < 32) {  // keys past the request's last do not exist
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if ((v >> 2) * 8 + g * 4 + (v & 3) >= left) sc[gr][v] = -INFINITY;
      }
      if constexpr (!PV) {  // the first half: the reference is its maximum
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          float mx = sc[gr][0];
#pragma unroll
          for (int v = 1; v < 16; ++v) mx = fmaxf(mx, sc[gr][v]);
          m_run[gr] = fmaxf(pair_max(mx) * cmul, -FLT_MAX);
        }
      }
      frag kf[3], vf[3];
      auto read = [&](int c) {
        if constexpr (QK) kf[c % 3] = k_frag(sk, kh, c);
        if constexpr (PV) vf[c % 3] = v_frag(sv, vh, c);
      };
      float ls[2] = {0.f, 0.f};
      auto exps = [&](int gr, int e) {  // pair e of group gr
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[gr][2 * e], cmul, -m_run[gr]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[gr][2 * e + 1], cmul, -m_run[gr]));
        ls[gr] += p0 + p1;
        pc[gr][e] = MfmaT<T>::pack2(p0, p1);
        asm volatile("" : "+v"(pc[gr][e]));  // here, not where it is first read
      };
      constexpr int PER = 8 / NC;  // pairs a group of MFMAs: NC groups of two or four
      read(0);
      read(1);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c + 2 < NC) read(c + 2);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (QK)
          sn[0] = MfmaT<T>::mma(kf[c % 3], qf[0][c], c == 0 ? f32x16{} : sn[0]);
#pragma unroll
        for (int e = 0; e < PER; ++e) exps(0, c * PER + e);
        if constexpr (QK) sn[1] = MfmaT<T>::mma(kf[c % 3], qf[1][c], c == 0 ? f32x16{} : sn[1]);
        if constexpr (PV)
          acc[0][c % NDT] = MfmaT<T>::mma(vf[c % 3], p_frag(pl[0], c / NDT), acc[0][c % NDT]);
#pragma unroll
        for (int e = 0; e < PER; ++e) exps(1, c * PER + e);
        if constexpr (PV)
          acc[1][c % NDT] = MfmaT<T>::mma(vf[c % 3], p_frag(pl[1], c / NDT), acc[1][c % NDT]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (PV && __any(!(ls[0] < MfmaT<T>::kLazyLimit) || !(ls[1] < MfmaT<T>::kLazyLimit))) {
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          float mx = -INFINITY;
#pragma unroll
          for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[gr][v]);
          const float m_use = fmaxf(m_run[gr], pair_max(mx) * cmul);
          const float alpha = __builtin_amdgcn_exp2f(m_run[gr] - m_use);
          m_run[gr] = m_use;
          l_run[gr] *= alpha;
#pragma unroll
          for (int i = 0; i < NDT; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[gr][i][v] *= alpha;
          ls[gr] = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[gr][2 * e], cmul, -m_use));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[gr][2 * e + 1], cmul, -m_use));
            ls[gr] += p0 + p1;
            pc[gr][e] = MfmaT<T>::pack2(p0, p1);
          }
        }
      }
      l_run[0] += ls[0];
      l_run[1] += ls[1];
      // the accumulators stay where the matrix core has them: left free, they move out and back
      // beside every half for the sake of the rescaling above, which hardly ever runs
      if constexpr (PV)
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
#pragma unroll
          for (int i = 0; i < NDT; ++i) asm volatile("" : "+a"(acc[gr][i]));
    };
    auto last_pv = [&](uint32_t (&pl)[2][8], const uint8_t* sv, int vh) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const frag vf = v_frag(sv, vh, c);
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
          acc[gr][c % NDT] = MfmaT<T>::mma(vf, p_frag(pl[gr], c / NDT), acc[gr][c % NDT]);
      }
    };
    using Yes = std::true_type;
    using No = std::false_type;
    // K(0) and Q, loaded under the row tile before, have landed for every wavefront. Its output's
    // stores, as many on every path, are younger and may be on their way, and between the two the
    // loads of K(1) and V(0), where there are both
    if (first) wide_barrier();
    else if (nt > 1) wide_barrier<L::STORES + L::KS / 4 + L::VS / 4>();
    else wide_barrier<L::STORES>();
#pragma unroll
    for (int gr = 0; gr < 2; ++gr)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int r = gr * 32 + col;
        u32x4 v = *reinterpret_cast<const u32x4*>(qlds + r * D * 2 + (((2 * c + g) ^ (r & (RPL - 1))) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] ^= a.q_sign;
        qf[gr][c] = __builtin_bit_cast(frag, v);
      }
    int quarters = 0;  // of the next tile's Q on the way
    auto load_quarter = [&]() {
      if (next.w.it.req >= 0 && quarters < 4) {
        load_q(next, quarters * L::QQ, (quarters + 1) * L::QQ);
        ++quarters;
        return true;
      }
      return false;
    };
    if (nt > 0) {
      f32x16 sa[2], sb[2];
      uint32_t pa[2][8], pb[2][8];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const frag kf = k_frag(kbuf(kb), 0, c);
#pragma unroll
        for (int gr = 0; gr < 2; ++gr)
          sa[gr] = MfmaT<T>::mma(kf, qf[gr][c], c == 0 ? f32x16{} : sa[gr]);
      }
      half_step(Yes{}, No{}, sa, sb, pb, pa, kbuf(kb), 1, nullptr, 0, keys);
      // before half 2j - 1: K(j) and V(j - 1) have landed. For j = 1 only the stores are younger, after
      // that a quarter of Q, if one was left to load
      bool q_last = false;
      auto landed = [&](int j) {
        if (j == 1 && !first) wide_barrier<L::STORES>();
        else if (q_last) wide_barrier<L::QQ>();
        else wide_barrier();
      };
      for (int j = 1; j < nt; ++j) {
        landed(j);
        if (j + 1 < nt) load_k(t, j + 1, (kb + j + 1) & 1);
        else if (next.w.it.req >= 0) load_k(next, 0, (kb + nt) & 1);
        load_v(t, j, (kb + j) & 1);
        q_last = load_quarter();
        half_step(Yes{}, Yes{}, sb, sa, pa, pb, kbuf((kb + j) & 1), 0, vbuf((kb + j - 1) & 1), 0,
                  keys - j * 64 + 32);
        half_step(Yes{}, Yes{}, sa, sb, pb, pa, kbuf((kb + j) & 1), 1, vbuf((kb + j - 1) & 1), 1,
                  keys - j * 64);
      }
      landed(nt);
      if (next.w.it.req >= 0) {
        if (nt == 1) load_k(next, 0, (kb + 1) & 1);
        while (load_quarter()) {
        }
        load_k(next, 1, (kb + nt + 1) & 1), load_v(next, 0, (kb + nt) & 1);
      }
      const uint8_t* sv = vbuf((kb + nt - 1) & 1);
      half_step(No{}, Yes{}, sb, sa, pa, pb, nullptr, 0, sv, 0, keys - nt * 64 + 32);
      last_pv(pb, sv, 1);
    } else if (next.w.it.req >= 0) {
      __syncthreads();  // every wavefront has its rows of Q
      load_k(next, 0, kb);
      while (load_quarter()) {
      }
      load_k(next, 1, (kb + 1) & 1), load_v(next, 0, kb);
    }
    first = false;
    // ---- normalize; lane: rows col of each group, channels dt * 32 + (v / 4) * 8 + 4 g + v % 4. 32 rows
    // of 64 channels at a time go through 4 KB of the wavefront's own (chunk c of row r at c ^ (r % 8))
    // and out as 128 bytes of a row by 8 lanes; a row that is not there is stored past the buffer's end
    const uint32_t tok0 = single ? (uint32_t)(t.w.it.tile * PW_ROWS)
                                 : (uint32_t)(t.w.it.tile * PW_ROWS) / (uint32_t)a.group;
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(
        a.o + (((int64_t)t.w.it.row0 + tok0) * a.os[0] + (int64_t)t.hk * a.group * a.os[1]) * 2, 0x80000000u);
    uint8_t* olds = lds + 2 * (L::KB + L::VB) + 4 * L::QB + wave * 4096;
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      const float l = pair_sum(l_run[gr]);
      const float inv = keys == 0 ? 0.f : 1.0f / l;  // no keys: zeros
      uint32_t off[4];  // of rows lane / 8 + 8 i
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t h;
        const uint32_t tok = conv_udiv((uint32_t)(t.w.it.tile * PW_ROWS + wave * 64 + gr * 32 + i * 8 + lane / 8),
                                       (uint32_t)a.group, a.group_m, h);
        off[i] = tok < (uint32_t)t.w.it.rows ? (tok - tok0) * (uint32_t)(a.os[0] * 2) +
                                                   h * (uint32_t)(a.os[1] * 2) + (lane & 7) * 16
                                             : 0x80000000u;
      }
#pragma unroll
      for (int d2 = 0; d2 < NDT; d2 += 2) {
#pragma unroll
        for (int dt = d2; dt < d2 + 2; ++dt)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<u32x2*>(olds + col * 128 + ((((dt - d2) * 4 + u) ^ (col & 7)) << 4) + g * 8) =
                u32x2{MfmaT<T>::pack2(acc[gr][dt][4 * u] * inv, acc[gr][dt][4 * u + 1] * inv),
                      MfmaT<T>::pack2(acc[gr][dt][4 * u + 2] * inv, acc[gr][dt][4 * u + 3] * inv)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + lane / 8;
          const u32x4 w = *reinterpret_cast<const u32x4*>(olds + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          __builtin_amdgcn_raw_buffer_store_b128(w, ro, off[i] + d2 * 64, 0, 0);
        }
      }
    }
    if (next.w.it.req < 0) return;
    kb = (kb + nt) & 1;
    t = next;
  }
}

// Tiles of 32 rows against tiles of 128 keys, 32 of them each wavefront's: with the few rows of
// single tokens every wavefront's matrix work and softmax is on keys of its own, where
// packed_attn_kernel's second to fourth would work on rows that are not there. The keys of the next
// tile wait in registers while this one's are in LDS, so two workgroups fit a compute unit and keep
// 128 KB of keys in flight on it.
constexpr int PF_ROWS = 32, PF_KEYS = 128;

template <typename T, int D, bool SPLIT>
__global__ __launch_bounds__(256, 2) void packed_attn_few_kernel(const PackedAttnArgs a) {
  typedef PackedTile<D, PF_KEYS> Tile;
  constexpr int JOIN = 4 * PF_ROWS * D * 4, TILES = PF_KEYS * Tile::KP + D * Tile::VT;
  __shared__ __attribute__((aligned(16))) uint8_t lds[TILES > JOIN ? TILES : JOIN];
  __shared__ f32x2 ml[4][PF_ROWS];
  uint8_t *sk = lds, *sv = lds + PF_KEYS * Tile::KP;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, g = lane >> 5;
  PackedChunks<PF_ROWS, PF_KEYS> chunks;
  if (SPLIT) chunks.scan(a);
  int id = blockIdx.x;
  if (!SPLIT && (gridDim.x & 7) == 0) id = (id & 7) * (gridDim.x >> 3) + (id >> 3);
  for (;; id += gridDim.x) {
    const int hk = SPLIT ? id % a.kv_heads : id / a.items;
    const PackedWork w = packed_work<SPLIT>(a, chunks, PF_ROWS, SPLIT ? id / a.kv_heads : id % a.items);
    if (w.it.req < 0 || (SPLIT && id >= a.slots)) return;
    int j_beg, j_end;
    packed_range(w, PF_KEYS, j_beg, j_end);
    const uint8_t* kp = a.k + ((int64_t)w.kbeg * a.ks[0] + hk * a.ks[1]) * 2;
    const uint8_t* vp = a.v + ((int64_t)w.kbeg * a.vs[0] + hk * a.vs[1]) * 2;
    const int64_t krow = a.ks[0] * 2, vrow = a.vs[0] * 2;
    Tile tile;
    auto load = [&](int j0) {
      tile.load(kp + j0 * krow, vp + j0 * vrow, krow, vrow, min(j_end - j0, PF_KEYS));
    };
    if (j_beg < j_end) load(j_beg);
    const int r = w.it.tile * PF_ROWS + col;
    const int tok = r / a.group, head = hk * a.group + (r - tok * a.group);
    typename MfmaT<T>::frag qf[D / 16];
    packed_load_q<T, D>(a, (uint32_t)tok < (uint32_t)w.it.rows, (int64_t)w.it.row0 + tok, head, g, qf);
    PackedRow<T, D> st;
    st.reset();
    for (int j0 = j_beg; j0 < j_end; j0 += PF_KEYS) {
      tile.store(sk, sv);
      __syncthreads();
      if (j0 + PF_KEYS < j_end) load(j0 + PF_KEYS);
      st.template step<1>(qf, sk, Tile::KP, sv, Tile::VT, wave * 32, j_end - j0 - wave * 32,
                          a.scale_log2);
      __syncthreads();
    }
    // ---- the four wavefronts' parts of each row, in their order
    const float l_w = pair_sum(st.l_run);
    if (g == 0) ml[wave][col] = f32x2{st.m_run, l_w};
    __syncthreads();
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, ml[i][col][0]);
    const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 4; ++i) l += ml[i][col][1] * __builtin_amdgcn_exp2f(ml[i][col][0] - m_use);
    const float mine = __builtin_amdgcn_exp2f(st.m_run - m_use);
    constexpr int CH = D / 4, CM = CH < 32 ? CH - 1 : 31;  // 16-byte chunk c of row r at c ^ (r & CM)
    float* parts = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<f32x4*>(parts + (wave * PF_ROWS + col) * D +
                                  (((dt * 8 + u * 2 + g) ^ (col & CM)) << 2)) =
            f32x4{st.acc[dt][4 * u] * mine, st.acc[dt][4 * u + 1] * mine,
                  st.acc[dt][4 * u + 2] * mine, st.acc[dt][4 * u + 3] * mine};
    __syncthreads();
    if (wave == 0 && g == 0) ml[0][col] = f32x2{m, l};  // to the threads that write the row
    __syncthreads();
    for (int i = tid; i < PF_ROWS * CH; i += 256) {
      const int rr = i / CH, c = i % CH;
      const int rq = w.it.tile * PF_ROWS + rr;
      const int t = rq / a.group, h = hk * a.group + (rq - t * a.group);
      if ((uint32_t)t >= (uint32_t)w.it.rows) continue;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(parts + (p * PF_ROWS + rr) * D +
                                                        ((c ^ (rr & CM)) << 2));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += v[e];
      }
      const f32x2 x = ml[0][rr];
      if (SPLIT && w.chunks > 1) {
        const int64_t at = (int64_t)id * PF_ROWS + rr;
        if (c == 0) a.stats[at] = f32x2{x[0], j_beg < j_end ? x[1] : -1.0f};
        if (j_beg < j_end) *reinterpret_cast<f32x4*>(a.part + at * D + c * 4) = o;
      } else {
        const float inv = w.keys == 0 ? 0.f : 1.0f / x[1];
        *reinterpret_cast<u32x2*>(reinterpret_cast<T*>(a.o) + (int64_t)(w.it.row0 + t) * a.os[0] +
                                  h * a.os[1] + c * 4) =
            u32x2{MfmaT<T>::pack2(o[0] * inv, o[1] * inv), MfmaT<T>::pack2(o[2] * inv, o[3] * inv)};
      }
    }
    if (!SPLIT) return;
    __syncthreads();  // the next item's keys overwrite the parts
  }
}

// The chunks of a row joined in their order: a workgroup per (row, head), each wavefront every fourth
// chunk, a lane per chunk for the statistics, 64 at a time. (A sum of 0, all scores -inf, gives NaN
// as it does whole.)
template <typename T, int D, int BLOCK, int KEYT>
__global__ __launch_bounds__(256) void packed_attn_join(const PackedAttnArgs a) {
  constexpr int PL = D / 64;  // channels per lane
  __shared__ float parts[4][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int heads = a.kv_heads * a.group;
  const int row = blockIdx.x / heads, head = blockIdx.x - row * heads;
  PackedChunks<BLOCK, KEYT> chunks;
  chunks.scan(a);
  const uint64_t in = __ballot(chunks.r0 <= row && row < chunks.r0 + chunks.len);
  if (!in) return;
  const PackedWork w = chunks.work_of(a, __ffsll((unsigned long long)in) - 1);
  if (w.chunks <= 1) return;  // written where it was computed
  const int hk = head / a.group, r = (row - w.it.row0) * a.group + head - hk * a.group;
  const int tile = r / BLOCK;
  // chunk p's slot and this row in it
  const int64_t s0 = ((int64_t)(w.first + tile * w.chunks) * a.kv_heads + hk) * BLOCK + r - tile * BLOCK;
  const int64_t step = (int64_t)a.kv_heads * BLOCK;
  if (s0 + (w.chunks - 1) * step >= (int64_t)a.slots * BLOCK) return;
  auto stats = [&](int c) {
    return c + lane < w.chunks ? a.stats[s0 + (c + lane) * step] : f32x2{-INFINITY, -1.0f};
  };
  float m = -INFINITY;
  for (int c = 0; c < w.chunks; c += kWave) {
    const f32x2 s = stats(c);
    m = fmaxf(m, wave_max(s[1] < 0.f ? -INFINITY : s[0]));
  }
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[PL] = {};
  for (int c = 0; c < w.chunks; c += kWave) {
    const f32x2 s = stats(c);
    const bool on = !(s[1] < 0.f);
    const float wt = on ? __builtin_amdgcn_exp2f(s[0] - m_use) : 0.f;
    l += wave_sum(on ? wt * s[1] : 0.f);
    const uint64_t there = __ballot(on);
    const int n = min(w.chunks - c, kWave);
#pragma unroll 8
    for (int p = wave; p < n; p += 4) {  // what a chunk without keys holds is not looked at
      const float wp = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wt), p));
      const float* q = a.part + (s0 + (c + p) * step) * D + lane * PL;
      const bool use = (there >> p) & 1;
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const float x = q[i];
        o[i] += use ? wp * x : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PL; ++i) parts[wave][lane * PL + i] = o[i];
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int d = threadIdx.x;
  const float sum = parts[0][d] + parts[1][d] + parts[2][d] + parts[3][d];
  Elt<T>::store(reinterpret_cast<T*>(a.o) + row * a.os[0] + head * a.os[1] + d, sum * (1.0f / l));
}

// ------------------------------------------------------------------ host
// What the host decides from the sizes it knows (never from the row numbers on the device).
struct PackedPlan {
  int block, key_tile;  // rows and keys of a tile
  int items;            // row tiles per key head, at most
  int groups;           // workgroups that cut keys into chunks; 0: keys stay whole
  int64_t slots;        // chunks, at most
};
static PackedPlan packed_plan(int64_t rows_q, int64_t rows_k, int64_t requests, int64_t kv_heads,
                              int64_t group, bool wide_strides) {
  PackedPlan p = {};
  // tiles of 32 rows where requests have fewer than 48 on average
  const bool few = rows_q * group <= 48 * std::max<int64_t>(requests, 1);
  // tiles of 256 where requests fill them and every compute unit has two (us, tiles of 256 against
  // 128; 24 heads of 128 channels unless said): 264 tiles to 512 keys 54 to 48, 528 tiles 72 to 71
  // (64 keys: 27.6 to 33.7), 792 tiles to 256 keys 61 to 66, 40 heads 2560 tiles to 512 keys 232 to
  // 280; 60 requests of 83 rows 103 to 66, of 200 rows 71 to 74
  const bool wide = !few && wide_strides && requests <= PACKED_LANES &&
                    rows_q * group >= PW_ROWS * requests &&
                    (rows_q * group / PW_ROWS) * kv_heads >= 512;
  p.block = few ? PF_ROWS : wide ? PW_ROWS : PA_ROWS;
  p.key_tile = few ? PF_KEYS : PA_KEYS;
  p.items = (int)((rows_q * group + p.block - 1) / p.block + requests + 2);
  // two workgroups for each compute unit; launches of as many row tiles keep their keys whole
  constexpr int kGroups = 512;
  if (!wide && requests > 0 && requests <= PACKED_LANES && rows_k > p.key_tile &&
      p.items * kv_heads < kGroups) {
    p.groups = kGroups;
    // PackedChunks::scan's count: at most `groups` and one for every row tile (and a few, for the
    // rounding of its quotient)
    p.slots = kGroups + p.items * kv_heads + 16;
  }
  return p;
}
static int64_t packed_stats_bytes(const PackedPlan& p) {
  return (p.slots * p.block * 8 + 255) / 256 * 256;
}
static int64_t packed_workspace(const PackedPlan& p, int64_t head_dim) {
  return p.groups ? packed_stats_bytes(p) + p.slots * p.block * head_dim * 4 : 0;
}

}  // namespace dlt

using namespace dlt;

extern "C" int64_t difflet_rocm_packed_attention_workspace_bytes(int64_t rows_q, int64_t rows_k,
                                                                 int64_t requests,
                                                                 int64_t kv_heads, int64_t group,
                                                                 int64_t head_dim) {
  if (rows_q <= 0 || rows_k <= 0 || requests <= 0 || kv_heads <= 0 || group <= 0 ||
      kv_heads * group > 65536 || rows_q * group >= (1LL << 30) || requests >= (1LL << 24))
    return 0;
  return packed_workspace(packed_plan(rows_q, rows_k, requests, kv_heads, group, true), head_dim);
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
  DLT_REQUIRE(kv_heads <= 65536 && group <= 65536 && kv_heads * group <= 65536 &&
                  rows_q < (1LL << 30) && rows_q * group < (1LL << 30) && rows_k < (1LL << 30) &&
                  requests < (1LL << 24),
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
  DLT_REQUIRE(k_strides[0] >= 0 && v_strides[0] >= 0 && k_strides[0] <= (1LL << 23) &&
                  v_strides[0] <= (1LL << 23),
              DIFFLET_EUNSUPPORTED, "%s: key rows more than 16 MB apart", name);
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
  // the wide kernel addresses a tile's rows of q and o in 31 bits and stores 16 bytes of o
  auto near = [&](const int64_t* st) {
    return st[0] >= 0 && st[1] >= 0 && st[0] < (1LL << 29) && st[1] < (1LL << 29) &&
           (PW_ROWS / group + 2) * st[0] + group * st[1] + head_dim < (1LL << 29);
  };
  const bool wide_strides = near(q_strides) && near(o_strides) && ((uintptr_t)o & 15) == 0 &&
                            o_strides[0] % 8 == 0 && o_strides[1] % 8 == 0;
  const PackedPlan plan = packed_plan(rows_q, rows_k, requests, kv_heads, group, wide_strides);
  a.items = plan.items;
  if (plan.groups && workspace && workspace_bytes >= packed_workspace(plan, head_dim)) {
    DLT_REQUIRE(((uintptr_t)workspace & 255) == 0, DIFFLET_EINVAL,
                "%s: workspace must be 256-byte aligned", name);
    a.groups = plan.groups;
    a.slots = (int)plan.slots;
    a.stats = (f32x2*)workspace;
    a.part = (float*)((uint8_t*)workspace + packed_stats_bytes(plan));
  }
  a.group_m = conv_magic((uint32_t)group);
  const int64_t blocks = a.groups ? a.groups : (int64_t)a.items * kv_heads;
  DLT_REQUIRE(blocks < (1LL << 31), DIFFLET_EUNSUPPORTED, "%s: too many tiles", name);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)blocks), block(256);
  auto go = [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    const bool few = plan.block == PF_ROWS;
    if (plan.block == PW_ROWS) {
      // one workgroup a compute unit
      const dim3 cus((unsigned)std::min<int64_t>(blocks, std::max(gemm_device_cus(), 1)));
      hipLaunchKernelGGL((packed_attn_wide_kernel<T, D>), cus, block, 0, s, a);
      return;
    }
    if (!a.groups) {
      if (few) hipLaunchKernelGGL((packed_attn_few_kernel<T, D, false>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((packed_attn_kernel<T, D, false>), grid, block, 0, s, a);
      return;
    }
    const dim3 rows((unsigned)(rows_q * kv_heads * group));
    if (few) {
      hipLaunchKernelGGL((packed_attn_few_kernel<T, D, true>), grid, block, 0, s, a);
      hipLaunchKernelGGL((packed_attn_join<T, D, PF_ROWS, PF_KEYS>), rows, block, 0, s, a);
    } else {
      hipLaunchKernelGGL((packed_attn_kernel<T, D, true>), grid, block, 0, s, a);
      hipLaunchKernelGGL((packed_attn_join<T, D, PA_ROWS, PA_KEYS>), rows, block, 0, s, a);
    }
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
