// Row-wise operators over packed rows of several requests: RMSNorm with the residual's addition
// and an 8-bit output, and rotary embedding from positions on several axes. Both are bound by
// HBM: one read and one write of every element, the statistics and the angles in between.
#include <math.h>

#include <algorithm>

#include "common.hpp"

namespace dlt {

// Eight consecutive elements, to and from fp32 (16-byte accesses: the hosts check alignment).
template <typename T> struct Vec8;
template <> struct Vec8<bf16> {
  static __device__ __forceinline__ void load(const bf16* p, float* v) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16bits_to_f32(r[i] & 0xffffu);
      v[2 * i + 1] = bf16bits_to_f32(r[i] >> 16);
    }
  }
  static __device__ __forceinline__ void store(bf16* p, const float* v) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<u32x4*>(p) = r;
  }
};
template <> struct Vec8<f16> {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void load(const f16* p, float* v) {
    const h8 r = *reinterpret_cast<const h8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
  }
  static __device__ __forceinline__ void store(f16* p, const float* v) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)v[i];
    *reinterpret_cast<h8*>(p) = r;
  }
};
template <> struct Vec8<float> {
  static __device__ __forceinline__ void load(const float* p, float* v) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  }
  static __device__ __forceinline__ void store(float* p, const float* v) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
};

// ------------------------------------------------------------------ RMSNorm to 8 bits
// h = x + residual in fp32, y = h / sqrt(mean(h^2) + eps) * weight, and y as e4m3 codes with one
// fp32 scale per row (max|y| / 448) or E8M0 scales per block of 32 in swizzle order. y is rounded
// once, to e4m3: layernorm_modulate's 8-bit forms round to bf16 before that because they stand
// for two calls, this one stands for its formula. h is written out rounded to x's type (the next
// residual stream); the norm takes the sum before that rounding.
//
// A row is held in registers, so x and the residual are read once. MX: a thread owns a whole block
// of 32, whose elements are the four runs k0 + j tile / 4 + 8 b + [0, 8) of a 512-wide tile (or the
// remainder): four 16-byte loads, 16 threads covering 256 consecutive bytes with each, and two
// 16-byte stores of codes in swizzle order; nothing crosses lanes but the row's sum (and maximum).
// A workgroup takes a row with as many wavefronts as SLOTS units a thread leave (WG), or, where one
// wavefront holds a row, four rows.
struct RmsArgs {
  const void* x;
  const void* res;     // NULL: none
  const void* weight;  // NULL: ones
  void* hidden;        // NULL: not written
  uint8_t* codes;
  void* scales;
  int64_t ldx, ldr, ldh, ldq, lds;
  int64_t rows;
  int dim, weight_dtype;
  float eps;
};

__device__ __forceinline__ void load_weight8(const void* w, int dtype, int i, float* v) {
  if (dtype == DIFFLET_BF16) Vec8<bf16>::load(reinterpret_cast<const bf16*>(w) + i, v);
  else if (dtype == DIFFLET_F16) Vec8<f16>::load(reinterpret_cast<const f16*>(w) + i, v);
  else Vec8<float>::load(reinterpret_cast<const float*>(w) + i, v);
}

// The offset of run j (of RUNS) of unit u: MX units are blocks of 32 in swizzle order, others
// eight consecutive elements.
template <bool MX>
__device__ __forceinline__ int rms_run(int u, int j, int dim) {
  if constexpr (!MX) return u * 8;
  const int k0 = u >> 4 << 9, sub = min(512, dim - k0) >> 2;
  return k0 + j * sub + 8 * (u & 15);
}

template <typename T, bool MX, bool WG, int SLOTS>
__global__ __launch_bounds__(WG ? 1024 : 256) void rms_norm_quant_kernel(const RmsArgs a) {
  constexpr int RUNS = MX ? 4 : 1;  // runs of 8 per unit
  __shared__ float red[2][16];
  const int tpr = WG ? blockDim.x : kWave;  // threads per row
  const int t = WG ? threadIdx.x : threadIdx.x & (kWave - 1);
  const int64_t row = WG ? blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (!WG && row >= a.rows) return;
  auto over_row = [&](float v, float* slots, auto join) {  // v already joined over the wavefront
    if constexpr (!WG) return v;
    if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slots[0];
    for (int i = 1; i < (int)blockDim.x / kWave; ++i) v = join(v, slots[i]);
    return v;
  };
  const int units = a.dim / (8 * RUNS);
  const T* xr = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* rr = a.res ? reinterpret_cast<const T*>(a.res) + row * a.ldr : nullptr;
  float v[SLOTS][RUNS][8];
  float ss = 0.f;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int u = s * tpr + t;
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
      if (u < units) Vec8<T>::load(xr + rms_run<MX>(u, j, a.dim), v[s][j]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][j][e] = 0.f;
    }
  }
  if (rr) {
    T* hr = a.hidden ? reinterpret_cast<T*>(a.hidden) + row * a.ldh : nullptr;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int u = s * tpr + t;
      if (u >= units) continue;
#pragma unroll
      for (int j = 0; j < RUNS; ++j) {
        float r[8];
        Vec8<T>::load(rr + rms_run<MX>(u, j, a.dim), r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[s][j][e] += r[e];
        if (hr) Vec8<T>::store(hr + rms_run<MX>(u, j, a.dim), v[s][j]);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s)
#pragma unroll
    for (int j = 0; j < RUNS; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[s][j][e], v[s][j][e], ss);
  ss = over_row(wave_sum(ss), red[0], [](float p, float q) { return p + q; });
  const float rs = 1.0f / __fsqrt_rn(ss / (float)a.dim + a.eps);
  float amax = 0.f;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int u = s * tpr + t;
#pragma unroll
    for (int j = 0; j < RUNS; ++j) {
      float w[8];
      if (a.weight && u < units) load_weight8(a.weight, a.weight_dtype, rms_run<MX>(u, j, a.dim), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[s][j][e] *= rs;
        if (a.weight && u < units) v[s][j][e] *= w[e];
        amax = fmaxf(amax, fabsf(v[s][j][e]));
      }
    }
  }
  // NaN anywhere in the row: ss, and so every y, is NaN, as is an infinity's own y (inf * 0).
  // A maximum passes over NaN, so the scales say it: NaN for the row, E8M0's NaN for a block.
  uint8_t* qr = a.codes + row * a.ldq;
  if constexpr (!MX) {
    bool bad = false;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) bad |= v[s][0][e] != v[s][0][e];
    amax = bad ? INFINITY : amax;
    amax = over_row(wave_max(amax), red[1], [](float p, float q) { return fmaxf(p, q); });
    const bool nan = amax == INFINITY;  // a finite row never reaches it: |y| <= sqrt(dim) |w|
    const float inv = nan ? __builtin_nanf("") : rowwise_inv(amax);
    if (t == 0) reinterpret_cast<float*>(a.scales)[row] = nan ? inv : rowwise_scale(amax);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int u = s * tpr + t;
      if (u >= units) continue;
      *reinterpret_cast<u32x2*>(qr + u * 8) =
          nan ? u32x2{0x7f7f7f7fu, 0x7f7f7f7fu} : encode8_rowwise(v[s][0], inv);
    }
  } else {
    uint8_t* sr = reinterpret_cast<uint8_t*>(a.scales) + row * a.lds;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int u = s * tpr + t;
      if (u >= units) continue;
      uint32_t emax = 0;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t x = (__builtin_bit_cast(uint32_t, v[s][j][e]) >> 23) & 0xffu;
          emax = max(emax, x);
        }
      bad = emax == 255;
      const int su = max((int)emax - 7, 0);
      const float mul = __builtin_bit_cast(float, (uint32_t)(254 - su) << 23);  // 2^(127 - su)
      float c[4][8];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) c[j][e] = clamp448(__fmul_rn(v[s][j][e], mul));
      u32x4 o0, o1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o0[e] = bad ? 0x7f7f7f7fu : e4m3x4(c[0][e], c[1][e], c[2][e], c[3][e]);
        o1[e] = bad ? 0x7f7f7f7fu : e4m3x4(c[0][4 + e], c[1][4 + e], c[2][4 + e], c[3][4 + e]);
      }
      *reinterpret_cast<u32x4*>(qr + u * 32) = o0;
      *reinterpret_cast<u32x4*>(qr + u * 32 + 16) = o1;
      sr[u] = bad ? 255 : (uint8_t)su;
    }
  }
}

template <typename T, bool MX>
static void launch_rms(const RmsArgs& a, hipStream_t s) {
  // one unit (MX) or two (rows) a thread keep registers few and the loads of many rows in flight:
  // 32760 x 5120 MXFP8 in 224 us (5.2 TB/s), 388 with a wavefront per row and three units a thread
  constexpr int SLOTS = MX ? 1 : 2;
  const int units = a.dim / (MX ? 32 : 8), waves = (units + SLOTS * kWave - 1) / (SLOTS * kWave);
  if (waves > 1)
    hipLaunchKernelGGL((rms_norm_quant_kernel<T, MX, true, SLOTS>), dim3((unsigned)a.rows),
                       dim3((unsigned)(waves * kWave)), 0, s, a);
  else
    hipLaunchKernelGGL((rms_norm_quant_kernel<T, MX, false, SLOTS>),
                       dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
}

// ------------------------------------------------------------------ rotary positions
// Pair p of a head turns by positions[axis(p)] * f(p): f is given in turns (frequency / 2 pi) and
// the product taken in fp64, whose fraction of a turn is exact to 2^-52 of the whole turns before
// it is rounded to fp32 for sine and cosine. In fp32 a position of 2^20 would lose the angle's
// last 0.06 rad. A workgroup computes the angles of its tokens once into LDS and rotates all
// heads of q and k with them.
constexpr int ROPE_MAX_PAIRS = 128, ROPE_MAX_AXES = 8;
constexpr int ROPE_LDS_PAIRS = 2048;  // (token, pair) angles of a workgroup
constexpr int ROPE_TOKENS = 64;       // its tokens, at most
struct RopeAxesArgs {
  const void* x[2];
  void* y[2];
  int64_t xs[2][3], ys[2][3];  // batch, token, head strides
  int heads[2];
  const void* pos;
  int64_t pos_batch;  // elements between batch elements (0: one for all)
  int pos_dtype;      // DIFFLET_F32, DIFFLET_I32 or -1 for int64
  int axes, pairs, dim;
  int64_t tokens, seq;  // batch * seq tokens
  int tok;              // tokens per workgroup
  int units;            // units per head: rotated ones, then copied ones
  int rot_units;
  uint32_t per_tok, per_tok_m, units_m, pairs_m;
  double turns[ROPE_MAX_PAIRS];
  uint8_t axis[ROPE_MAX_PAIRS];
};

// V: pairs per unit. HALVES: pair p is (p, pairs + p), else (2 p, 2 p + 1).
template <typename T, bool HALVES, int V>
__device__ __forceinline__ void rope_unit(const T* x, T* y, int p0, int pairs, const float2* cs) {
  if constexpr (V == 1) {
    const int i = HALVES ? p0 : 2 * p0, j = HALVES ? pairs + p0 : 2 * p0 + 1;
    const float a = Elt<T>::load(x + i), b = Elt<T>::load(x + j);
    const float2 c = cs[0];
    Elt<T>::store(y + i, __builtin_fmaf(a, c.x, -(b * c.y)));
    Elt<T>::store(y + j, __builtin_fmaf(b, c.x, a * c.y));
  } else if constexpr (HALVES) {
    static_assert(V == 8, "eight pairs of two 8-element runs");
    float a[8], b[8];
    Vec8<T>::load(x + p0, a);
    Vec8<T>::load(x + pairs + p0, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 c = cs[e];
      const float u = __builtin_fmaf(a[e], c.x, -(b[e] * c.y));
      b[e] = __builtin_fmaf(b[e], c.x, a[e] * c.y);
      a[e] = u;
    }
    Vec8<T>::store(y + p0, a);
    Vec8<T>::store(y + pairs + p0, b);
  } else {
    static_assert(V == 4, "four pairs of one 8-element run");
    float a[8];
    Vec8<T>::load(x + 2 * p0, a);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 c = cs[e];
      const float u = __builtin_fmaf(a[2 * e], c.x, -(a[2 * e + 1] * c.y));
      a[2 * e + 1] = __builtin_fmaf(a[2 * e + 1], c.x, a[2 * e] * c.y);
      a[2 * e] = u;
    }
    Vec8<T>::store(y + 2 * p0, a);
  }
}

template <typename T, bool HALVES, bool WIDE>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeAxesArgs a) {
  constexpr int V = !WIDE ? 1 : HALVES ? 8 : 4;
  __shared__ float2 cs[ROPE_LDS_PAIRS];
  // where a token's rows lie: a 64-bit division for every unit of 16 bytes would bound the kernel
  // (32760 tokens of 80 heads of 128 bf16: 312 us with it, 260 so, 5.2 TB/s)
  __shared__ const T* xrow[2][ROPE_TOKENS];
  __shared__ T* yrow[2][ROPE_TOKENS];
  const int64_t t0 = (int64_t)blockIdx.x * a.tok;
  const int nt = (int)min((int64_t)a.tok, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
    uint32_t p;
    const uint32_t dt = conv_udiv((uint32_t)i, (uint32_t)a.pairs, a.pairs_m, p);
    const int64_t tk = t0 + dt, b = tk / a.seq;
    const int64_t at = b * a.pos_batch + (tk - b * a.seq) * a.axes + a.axis[p];
    double pos;
    if (a.pos_dtype == DIFFLET_F32) pos = (double)reinterpret_cast<const float*>(a.pos)[at];
    else if (a.pos_dtype == DIFFLET_I32) pos = (double)reinterpret_cast<const int32_t*>(a.pos)[at];
    else pos = (double)reinterpret_cast<const int64_t*>(a.pos)[at];
    double turn = pos * a.turns[p];
    turn -= __builtin_rint(turn);
    float s, c;
    sincospif((float)(2.0 * turn), &s, &c);
    cs[i] = float2{c, s};
  }
  for (int i = threadIdx.x; i < 2 * nt; i += 256) {
    const int w = i & 1, dt = i >> 1;
    const int64_t tk = t0 + dt, b = tk / a.seq, s = tk - b * a.seq;
    xrow[w][dt] = reinterpret_cast<const T*>(a.x[w]) + b * a.xs[w][0] + s * a.xs[w][1];
    yrow[w][dt] = reinterpret_cast<T*>(a.y[w]) + b * a.ys[w][0] + s * a.ys[w][1];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < (uint32_t)nt * a.per_tok; i += 256) {
    uint32_t r, u;
    const uint32_t dt = conv_udiv(i, a.per_tok, a.per_tok_m, r);
    uint32_t h = conv_udiv(r, (uint32_t)a.units, a.units_m, u);
    const int w = h >= (uint32_t)a.heads[0];
    if (w) h -= a.heads[0];
    const T* x = xrow[w][dt] + h * (w ? a.xs[1][2] : a.xs[0][2]);
    T* y = yrow[w][dt] + h * (w ? a.ys[1][2] : a.ys[0][2]);
    if ((int)u < a.rot_units) {
      rope_unit<T, HALVES, V>(x, y, (int)u * V, a.pairs, cs + dt * a.pairs + u * V);
    } else {  // channels past the rotated ones
      const int c = 2 * a.pairs + ((int)u - a.rot_units) * (WIDE ? 8 : 1);
      if constexpr (WIDE) {
        float v[8];
        Vec8<T>::load(x + c, v);
        Vec8<T>::store(y + c, v);
      } else {
        y[c] = x[c];
      }
    }
  }
}

template <typename T>
static void launch_rope_axes(const RopeAxesArgs& a, bool halves, bool wide, hipStream_t s) {
  const dim3 grid((unsigned)((a.tokens + a.tok - 1) / a.tok)), block(256);
  if (halves) {
    if (wide) hipLaunchKernelGGL((rope_axes_kernel<T, true, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_axes_kernel<T, true, false>), grid, block, 0, s, a);
  } else {
    if (wide) hipLaunchKernelGGL((rope_axes_kernel<T, false, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rope_axes_kernel<T, false, false>), grid, block, 0, s, a);
  }
}

}  // namespace dlt

using namespace dlt;

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" int difflet_rocm_rms_norm_quant(const void* x, int64_t ldx, const void* residual,
                                           int64_t ldr, void* hidden, int64_t ldh, uint8_t* codes,
                                           int64_t ldq, void* scales, int64_t lds, int dtype,
                                           int64_t rows, int64_t dim, const void* weight,
                                           int weight_dtype, float eps, int mx,
                                           difflet_stream_t stream) {
  DLT_REQUIRE(rows >= 0 && dim > 0, DIFFLET_EINVAL, "rms_norm_quant: bad shape");
  DLT_REQUIRE(rows < (1LL << 31), DIFFLET_EUNSUPPORTED, "rms_norm_quant: too many rows");
  DLT_REQUIRE(dim % (mx ? 128 : 8) == 0, DIFFLET_EINVAL,
              "rms_norm_quant: dim = %lld must be a multiple of %d", (long long)dim, mx ? 128 : 8);
  DLT_REQUIRE(dim <= 16384, DIFFLET_EUNSUPPORTED, "rms_norm_quant: dim = %lld exceeds 16384",
              (long long)dim);
  DLT_REQUIRE(dtype == DIFFLET_F32 || dtype == DIFFLET_BF16 || dtype == DIFFLET_F16,
              DIFFLET_EINVAL, "rms_norm_quant: unsupported dtype %d", dtype);
  DLT_REQUIRE(!weight || weight_dtype == DIFFLET_F32 || weight_dtype == DIFFLET_BF16 ||
                  weight_dtype == DIFFLET_F16,
              DIFFLET_EINVAL, "rms_norm_quant: unsupported weight dtype %d", weight_dtype);
  if (rows == 0) return DIFFLET_OK;
  DLT_REQUIRE(x && codes && scales, DIFFLET_EINVAL, "rms_norm_quant: null pointer");
  DLT_REQUIRE(!hidden || residual, DIFFLET_EINVAL,
              "rms_norm_quant: the sum is written where a residual is added");
  DLT_REQUIRE(ldx % 8 == 0 && (!residual || ldr % 8 == 0) && (!hidden || (ldh % 8 == 0 && ldh >= dim)) &&
                  ldq % (mx ? 16 : 8) == 0 && ldq >= dim && (!mx || lds >= dim / 32),
              DIFFLET_EINVAL, "rms_norm_quant: bad row strides");
  DLT_REQUIRE(aligned16(x) && aligned16(residual) && aligned16(hidden) && aligned16(weight) &&
                  ((uintptr_t)codes & (mx ? 15 : 7)) == 0 && (mx || ((uintptr_t)scales & 3) == 0),
              DIFFLET_EINVAL, "rms_norm_quant: misaligned pointers");
  RmsArgs a = {x, residual, weight, hidden, codes, scales, ldx, ldr, ldh, ldq, lds, rows,
               (int)dim, weight_dtype, eps};
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (mx) launch_rms<T, true>(a, s);
    else launch_rms<T, false>(a, s);
  };
  if (dtype == DIFFLET_BF16) go(bf16{});
  else if (dtype == DIFFLET_F16) go(f16{});
  else go(float{});
  return dlt_check_launch("rms_norm_quant");
}

extern "C" int difflet_rocm_rope_axes(const void* q, void* q_out, const int64_t* q_strides,
                                      const int64_t* q_out_strides, int64_t q_heads, const void* k,
                                      void* k_out, const int64_t* k_strides,
                                      const int64_t* k_out_strides, int64_t k_heads, int dtype,
                                      int64_t batch, int64_t seq, int64_t head_dim,
                                      const void* positions, int positions_dtype,
                                      int64_t positions_batch_stride, int64_t axes, int64_t pairs,
                                      const double* turns, const uint8_t* pair_axis, int halves,
                                      difflet_stream_t stream) {
  DLT_REQUIRE(batch >= 0 && seq >= 0 && head_dim > 0 && q_heads >= 0 && k_heads >= 0,
              DIFFLET_EINVAL, "rope_axes: bad shape");
  DLT_REQUIRE(dtype == DIFFLET_F32 || dtype == DIFFLET_BF16 || dtype == DIFFLET_F16,
              DIFFLET_EINVAL, "rope_axes: unsupported dtype %d", dtype);
  DLT_REQUIRE(positions_dtype == DIFFLET_F32 || positions_dtype == DIFFLET_I32 ||
                  positions_dtype == -1,
              DIFFLET_EINVAL, "rope_axes: unsupported positions dtype %d", positions_dtype);
  DLT_REQUIRE(axes >= 1 && axes <= ROPE_MAX_AXES && pairs >= 1 && pairs <= ROPE_MAX_PAIRS &&
                  2 * pairs <= head_dim && turns && pair_axis,
              DIFFLET_EINVAL, "rope_axes: 1 to %d axes over 1 to %d pairs of channels within the head",
              ROPE_MAX_AXES, ROPE_MAX_PAIRS);
  DLT_REQUIRE(head_dim <= 4096 && q_heads + k_heads <= 65536 && batch < (1LL << 31) &&
                  seq < (1LL << 31) && batch * seq < (1LL << 40),
              DIFFLET_EUNSUPPORTED, "rope_axes: too large");
  for (int64_t p = 0; p < pairs; ++p)
    DLT_REQUIRE(pair_axis[p] < axes, DIFFLET_EINVAL, "rope_axes: pair %d has axis %d of %d", (int)p,
                (int)pair_axis[p], (int)axes);
  if (batch * seq == 0 || q_heads + k_heads == 0) return DIFFLET_OK;
  DLT_REQUIRE(positions && (q_heads == 0 || (q && q_out && q_strides && q_out_strides)) &&
                  (k_heads == 0 || (k && k_out && k_strides && k_out_strides)),
              DIFFLET_EINVAL, "rope_axes: null pointer");
  RopeAxesArgs a = {};
  const void* xs[2] = {q, k};
  void* ys[2] = {q_out, k_out};
  const int64_t* sx[2] = {q_strides, k_strides};
  const int64_t* sy[2] = {q_out_strides, k_out_strides};
  const int64_t hs[2] = {q_heads, k_heads};
  // 16-byte accesses where every head starts on 16 bytes and the pairs fill them
  bool wide = head_dim % 8 == 0 && (halves ? pairs % 8 == 0 : pairs % 4 == 0);
  for (int w = 0; w < 2; ++w) {
    a.heads[w] = (int)hs[w];
    if (hs[w] == 0) continue;
    a.x[w] = xs[w];
    a.y[w] = ys[w];
    const int es = dtype == DIFFLET_F32 ? 4 : 2;
    wide = wide && aligned16(xs[w]) && aligned16(ys[w]);
    for (int i = 0; i < 3; ++i) {
      a.xs[w][i] = sx[w][i];
      a.ys[w][i] = sy[w][i];
      wide = wide && sx[w][i] * es % 16 == 0 && sy[w][i] * es % 16 == 0;
    }
  }
  a.pos = positions;
  a.pos_dtype = positions_dtype;
  a.pos_batch = positions_batch_stride;
  a.axes = (int)axes;
  a.pairs = (int)pairs;
  a.dim = (int)head_dim;
  a.tokens = batch * seq;
  a.seq = seq;
  const int v = !wide ? 1 : halves ? 8 : 4;
  a.rot_units = (int)pairs / v;
  a.units = a.rot_units + (int)(head_dim - 2 * pairs) / (wide ? 8 : 1);
  a.per_tok = (uint32_t)((q_heads + k_heads) * a.units);
  a.per_tok_m = conv_magic(a.per_tok);
  a.units_m = conv_magic((uint32_t)a.units);
  a.pairs_m = conv_magic((uint32_t)pairs);
  for (int64_t p = 0; p < pairs; ++p) {
    a.turns[p] = turns[p];
    a.axis[p] = pair_axis[p];
  }
  // tokens per workgroup: about four units per thread, as long as the chip stays full of workgroups
  int64_t tok = std::max<int64_t>(1, 1024 / a.per_tok);
  tok = std::min<int64_t>(tok, std::max<int64_t>(1, a.tokens / 2048));
  tok = std::min<int64_t>({tok, ROPE_LDS_PAIRS / pairs, ROPE_TOKENS});
  a.tok = (int)std::max<int64_t>(1, tok);
  DLT_REQUIRE((a.tokens + a.tok - 1) / a.tok < (1LL << 31), DIFFLET_EUNSUPPORTED,
              "rope_axes: too many tokens");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DIFFLET_BF16) launch_rope_axes<bf16>(a, halves != 0, wide, s);
  else if (dtype == DIFFLET_F16) launch_rope_axes<f16>(a, halves != 0, wide, s);
  else launch_rope_axes<float>(a, halves != 0, wide, s);
  return dlt_check_launch("rope_axes");
}
