// Residual add + RMSNorm that keeps the sum in 8 bits for its backward pass (the form: packed.cuh).
//
//   h = x + a, r = (mean h^2 + eps)^(-1/2), y = h r w, h kept packed with r; backward, with x^ = h^ r:
//   dx = r (dy w - x^ mean(dy w x^)) + dh,  dw = sum_rows dy x^,  y again = x^ w
//
// Products, sums and statistics are in 32 bits; an output is rounded once, to its type.  h is rounded to its type
// before the norm, since the residual stream that the backward pass differentiates is what the tensor holds.
//
// Bound by the bytes that it moves: a row is held in registers, so every tensor is read once and written once.  A thread
// holds 16 neighbouring values (half a group: 32-byte accesses, one shuffle for the scale), through 16-byte pieces where
// rows are not whole multiples of that or not aligned (kRagged: packed.cuh).  A CTA takes a row, or a
// warp one of up to 512 values (several, where rows are shorter still).  The backward pass keeps its CTAs for all rows:
// each sums dw beside dx over its rows in order, and a last kernel adds the CTAs' sums in order.  32768 x 4096 bf16, forward and
// backward: 0.383 ms, 6.3 TB/s (a copy runs at 6.55); x 4090, ragged and bound by instructions and, in the backward pass, by the 16
// warps an SM that its registers leave: 0.66 ms, 3.7 TB/s.  Whole fp32 rows of 513 to 8192 values spill 100 bytes a thread in the
// backward pass, ragged fp32 ones over 8192 spill 56 (16384 x 4096 fp32: 0.19 ms against 0.17 of bytes).
#include <algorithm>
#include <type_traits>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWarpRow = 512;   // values of a row that a warp holds
constexpr int kHalfRow = 8192;  // values of a row that a CTA holds at 16 a thread
constexpr int kMaxRow = 16384;  // the same at 32

struct NormFwd {
  int64_t rows, d;
  const void *x, *a, *w;
  int64_t x_ld, a_ld;
  float eps;
  void *h, *y;
  int64_t h_ld, y_ld;
  uint8_t *codes, *scales;
  int64_t c_ld, s_ld;
  float* rstd;
  int lanes;  // of a row, where a warp holds several
};

struct NormBwd {
  int64_t rows, d;
  const void *dy, *dh, *w;
  int64_t dy_ld, dh_ld;
  const uint8_t *codes, *scales;
  int64_t c_ld, s_ld;
  const float* rstd;
  void *dx, *y, *dw;
  int64_t dx_ld, y_ld;
  float* part;  // [parts, d] partial sums of dw
  int parts;
  int lanes;
};

template <typename T>
__device__ __forceinline__ float residual(const NormFwd& a, int64_t r, int64_t i) {
  float v = to_float(static_cast<const T*>(a.x)[r * a.x_ld + i]);
  if (a.a) v = to_float(from_float<T>(v + to_float(static_cast<const T*>(a.a)[r * a.a_ld + i])));
  return v;
}

// Sum over a CTA's threads, the same value in each of them.  ws may be written again after the CTA's next barrier.
__device__ __forceinline__ float cta_sum(float v, float* ws) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? ws[lane] : 0.f);
}
// Sum over a row's threads: the CTA, or `lanes` neighbouring lanes (a power of two).
template <bool kWarpRows>
__device__ __forceinline__ float row_sum(float v, int lanes, float* ws) {
  if (!kWarpRows) return cta_sum(v, ws);
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float rstd_of(float ss, const NormFwd& a) { return 1.0f / sqrtf(ss / (float)a.d + a.eps); }

// ---------------------------------------------------------------------------------------------
// 16 neighbouring values a thread, kHalves times.
// ---------------------------------------------------------------------------------------------
template <typename T, bool kRagged, bool kWarpRows, int kHalves, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) add_rmsnorm_pack16_kernel(const NormFwd a) {
  __shared__ float ws[32];
  const int lane = threadIdx.x & 31, per = kWarpRows ? 32 / a.lanes : 1;
  const int64_t r = kWarpRows ? ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * per + lane / a.lanes : blockIdx.x;
  const int64_t i0 = (kWarpRows ? lane & (a.lanes - 1) : threadIdx.x) * 16;
  const int64_t step = (int64_t)blockDim.x * 16;  // between a thread's halves
  const T *x = static_cast<const T*>(a.x), *add = static_cast<const T*>(a.a), *w = static_cast<const T*>(a.w);
  float v[kHalves][16], ss = 0.f;
#pragma unroll
  for (int j = 0; j < kHalves; ++j) {
    const int64_t i = i0 + j * step;
    const Spot at = spot_of<kRagged>(i, a.d, r < a.rows);
    HalfIn<T, kRagged> hx, ha;
    hx.zero();
    ha.zero();
    if (kRagged || at.live) {
      hx.load(x + r * a.x_ld + i, at, extent_of(x, a.rows, a.x_ld, a.d));
      if (a.a) ha.load(add + r * a.a_ld + i, at, extent_of(add, a.rows, a.a_ld, a.d));
    }
    hx.get(v[j], at);
    if (a.a) {
      float t[16];
      ha.get(t, at);
#pragma unroll
      for (int k = 0; k < 16; ++k) v[j][k] += t[k];
      Half<T> sum;
      sum.set(v[j]);
      sum.get(v[j]);
      if (a.h) put_values<kRagged>(static_cast<T*>(a.h) + r * a.h_ld + i, v[j], at);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) ss = fmaf(v[j][k], v[j][k], ss);
  }
  const float rstd = rstd_of(row_sum<kWarpRows>(ss, a.lanes, ws), a);
  if (i0 == 0 && r < a.rows) a.rstd[r] = rstd;
#pragma unroll
  for (int j = 0; j < kHalves; ++j) {
    const int64_t i = i0 + j * step;
    const Spot at = spot_of<kRagged>(i, a.d, r < a.rows);
    if (kRagged || at.live) {
      HalfIn<T, kRagged> hw;
      hw.zero();
      if (kRagged || at.live) hw.template load<true>(w + i, at, extent_of(w, 1, 0, a.d));
      float t[16];
      hw.get(t, at);
#pragma unroll
      for (int k = 0; k < 16; ++k) t[k] = v[j][k] * rstd * t[k];
      put_values<kRagged>(static_cast<T*>(a.y) + r * a.y_ld + i, t, at);
    }
    uint4 q;
    const int s = pack_half(v[j], &q);
    if (!at.live) continue;
    store_codes(a.codes + r * a.c_ld + i, q);
    if ((threadIdx.x & 1) == 0) a.scales[r * a.s_ld + i / kGroup] = (uint8_t)s;
  }
}

// What the backward pass reads of 16 values of a row.
template <typename T, bool kRagged>
struct RowIn {
  HalfIn<T, kRagged> dy, dh;
  uint4 codes;
  float scale, rstd;
  __device__ __forceinline__ void load(const NormBwd& a, int64_t r, int64_t i) {
    dy.zero();
    dh.zero();
    codes = make_uint4(0, 0, 0, 0);
    scale = rstd = 0.f;
    const Spot at = spot_of<kRagged>(i, a.d, r < a.rows);
    if (!kRagged && !at.live) return;
    const T *py = static_cast<const T*>(a.dy), *ph = static_cast<const T*>(a.dh);
    dy.load(py + r * a.dy_ld + i, at, extent_of(py, a.rows, a.dy_ld, a.d));
    codes = load_codes<kRagged>(a.codes + r * a.c_ld + i, at);
    if (a.dh) dh.load(ph + r * a.dh_ld + i, at, extent_of(ph, a.rows, a.dh_ld, a.d));
    if (!at.live) return;
    scale = pow2_of(a.scales[r * a.s_ld + i / kGroup]);
    rstd = a.rstd[r];
  }
};

// The columns' sums of a CTA whose warps held rows: acc[k] of column first + k, added over the warps in order.
__device__ __forceinline__ void warp_rows_part(const NormBwd& a, const float* acc, float* part, float (*col)[kWarpRow],
                                               int first, bool writes) {
  if (writes)
#pragma unroll
    for (int k = 0; k < 16; ++k) col[threadIdx.x >> 5][first + k] = acc[k];
  __syncthreads();
  for (int c = threadIdx.x; c < a.d; c += kThreads) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += col[w][c];
    part[c] = t;
  }
}

// A thread's 16 sums of a CTA's share of dw.
template <bool kRagged>
__device__ __forceinline__ void put_part(float* part, const float* acc, int live) {
  if (kRagged) {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (k < live) part[k] = acc[k];
  } else if (live) {
#pragma unroll
    for (int k = 0; k < 16; k += 4)
      *reinterpret_cast<float4*>(part + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
  }
}

// Rows blockIdx.x, blockIdx.x + gridDim.x, ... (or as many for each warp); part[blockIdx.x] = the CTA's sum of dy x^ over
// its rows, in that order.  The next row is loaded before this row's sum is waited for; not so a
// ragged one, for want of registers.
template <typename T, bool kRagged, bool kWarpRows>
__global__ void __launch_bounds__(kWarpRows ? kThreads : 512) rmsnorm_bwd16_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  __shared__ float col[kWarpRows ? kWarps : 1][kWarpRow];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = kWarpRows ? 32 / a.lanes : 1;
  const int64_t i = (kWarpRows ? lane & (a.lanes - 1) : threadIdx.x) * 16;
  const Spot col_at = spot_of<kRagged>(i, a.d, true);
  HalfIn<T, kRagged> hw;
  hw.zero();
  if (kRagged || col_at.live)
    hw.template load<true>(static_cast<const T*>(a.w) + i, col_at, extent_of(static_cast<const T*>(a.w), 1, 0, a.d));
  float acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
  const int64_t step = (int64_t)gridDim.x * (kWarpRows ? kWarps : 1) * per;
  int64_t base = (kWarpRows ? (int64_t)blockIdx.x * kWarps + warp : blockIdx.x) * per;
  const int slot = kWarpRows ? lane / a.lanes : 0;
  RowIn<T, kRagged> in;
  if (!kRagged) in.load(a, base + slot, i);
  const float inv_d = 1.0f / (float)a.d;
  for (int turn = 0; base < a.rows; ++turn, base += step) {
    const int64_t r = base + slot;
    if (kRagged) in.load(a, r, i);
    const RowIn<T, kRagged> cur = in;
    const Spot at = spot_of<kRagged>(i, a.d, r < a.rows);
    if (!kRagged) in.load(a, r + step, i);
    float dy[16], xh[16], w[16];
    cur.dy.get(dy, at);
    hw.get(w, col_at);
    unpack_half(cur.codes, cur.scale, xh);
    float along = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      xh[k] *= cur.rstd;
      along = fmaf(dy[k] * w[k], xh[k], along);
      acc[k] = fmaf(dy[k], xh[k], acc[k]);
    }
    along = row_sum<kWarpRows>(along, a.lanes, ws[turn & 1]) * inv_d;
    if (kRagged || at.live) {
      float dh[16];
      cur.dh.get(dh, at);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        dh[k] += cur.rstd * (dy[k] * w[k] - xh[k] * along);
        xh[k] *= w[k];
      }
      put_values<kRagged>(static_cast<T*>(a.dx) + r * a.dx_ld + i, dh, at);
      if (a.y) put_values<kRagged>(static_cast<T*>(a.y) + r * a.y_ld + i, xh, at);
    }
  }
  if (!a.dw) return;
  float* part = a.part + (int64_t)blockIdx.x * a.d;
  if (kWarpRows) {
    for (int o = a.lanes; o < 32; o <<= 1)  // the warp's rows side by side
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    warp_rows_part(a, acc, part, col, (int)i, lane < a.lanes);
  } else {
    put_part<kRagged>(part + i, acc, col_at.live);
  }
}

// Rows of more than 8192 values: 32 a thread.  Their sums of dw leave no registers to load ahead, or for the weights.
template <typename T, bool kRagged>
__global__ void __launch_bounds__(512) rmsnorm_bwd32_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  const int64_t step = (int64_t)blockDim.x * 16;
  const T *py = static_cast<const T*>(a.dy), *ph = static_cast<const T*>(a.dh), *pw = static_cast<const T*>(a.w);
  const Extent in_w = extent_of(pw, 1, 0, a.d);
  Spot at[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) at[j] = spot_of<kRagged>(threadIdx.x * 16 + j * step, a.d, true);
  float acc[2][16];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[j][k] = 0.f;
  const float inv_d = 1.0f / (float)a.d;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, ++turn) {
    const float rstd = a.rstd[r];
    HalfIn<T, kRagged> hdy[2];
    uint4 codes[2];
    float scale[2], along = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t i = threadIdx.x * 16 + j * step;
      hdy[j].zero();
      codes[j] = make_uint4(0, 0, 0, 0);
      scale[j] = 0.f;
      if (!kRagged && !at[j].live) continue;
      hdy[j].load(py + r * a.dy_ld + i, at[j], extent_of(py, a.rows, a.dy_ld, a.d));
      codes[j] = load_codes<kRagged>(a.codes + r * a.c_ld + i, at[j]);
      if (at[j].live) scale[j] = pow2_of(a.scales[r * a.s_ld + i / kGroup]) * rstd;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t i = threadIdx.x * 16 + j * step;
      if (!at[j].live) continue;
      HalfIn<T, kRagged> hw;
      hw.template load<true>(pw + i, at[j], in_w);
      float dy[16], xh[16], w[16];
      hdy[j].get(dy, at[j]);
      hw.get(w, at[j]);
      unpack_half(codes[j], scale[j], xh);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        along = fmaf(dy[k] * w[k], xh[k], along);
        acc[j][k] = fmaf(dy[k], xh[k], acc[j][k]);
      }
    }
    along = cta_sum(along, ws[turn & 1]) * inv_d;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t i = threadIdx.x * 16 + j * step;
      if (!kRagged && !at[j].live) continue;  // ragged rows are stored by whole warps
      HalfIn<T, kRagged> hw, hdh;
      hw.zero();
      hdh.zero();
      if (kRagged || at[j].live) {
        hw.template load<true>(pw + i, at[j], in_w);
        if (a.dh) hdh.load(ph + r * a.dh_ld + i, at[j], extent_of(ph, a.rows, a.dh_ld, a.d));
      }
      float dy[16], xh[16], w[16], dh[16];
      hdy[j].get(dy, at[j]);
      hw.get(w, at[j]);
      hdh.get(dh, at[j]);
      unpack_half(codes[j], scale[j], xh);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        dh[k] += rstd * (dy[k] * w[k] - xh[k] * along);
        xh[k] *= w[k];
      }
      put_values<kRagged>(static_cast<T*>(a.dx) + r * a.dx_ld + i, dh, at[j]);
      if (a.y) put_values<kRagged>(static_cast<T*>(a.y) + r * a.y_ld + i, xh, at[j]);
    }
  }
  if (!a.dw) return;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    put_part<kRagged>(a.part + (int64_t)blockIdx.x * a.d + threadIdx.x * 16 + j * step, acc[j], at[j].live);
}

// ---------------------------------------------------------------------------------------------
// Rows that no CTA holds: read again from L2 for each use.
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) add_rmsnorm_pack_long_kernel(const NormFwd a) {
  __shared__ float ws[32];
  const int64_t r = blockIdx.x, padded = (a.d + kGroup - 1) / kGroup * kGroup;
  float ss = 0.f;
  for (int64_t i = threadIdx.x; i < a.d; i += kThreads) {
    const float v = residual<T>(a, r, i);
    ss = fmaf(v, v, ss);
  }
  const float rstd = rstd_of(cta_sum(ss, ws), a);
  if (threadIdx.x == 0) a.rstd[r] = rstd;
  for (int64_t i = threadIdx.x; i < padded; i += kThreads) {  // whole warps: a group is a warp's 32 lanes
    const float v = i < a.d ? residual<T>(a, r, i) : 0.f;
    int s;
    const uint32_t c = pack_lane(v, &s);
    if ((threadIdx.x & 31) == 0) a.scales[r * a.s_ld + i / kGroup] = (uint8_t)s;
    if (i >= a.d) continue;
    a.codes[r * a.c_ld + i] = (uint8_t)c;
    if (a.h) static_cast<T*>(a.h)[r * a.h_ld + i] = from_float<T>(v);
    static_cast<T*>(a.y)[r * a.y_ld + i] = from_float<T>(v * rstd * to_float(static_cast<const T*>(a.w)[i]));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rmsnorm_bwd_long_kernel(const NormBwd a) {
  __shared__ float ws[32];
  const int64_t r = blockIdx.x;
  const float rstd = a.rstd[r];
  const T *dy = static_cast<const T*>(a.dy) + r * a.dy_ld, *w = static_cast<const T*>(a.w);
  float along = 0.f;
  for (int64_t i = threadIdx.x; i < a.d; i += kThreads) {
    const float xh = unpack_one(a.codes[r * a.c_ld + i], a.scales[r * a.s_ld + i / kGroup]) * rstd;
    along = fmaf(to_float(dy[i]) * to_float(w[i]), xh, along);
  }
  along = cta_sum(along, ws) / (float)a.d;
  for (int64_t i = threadIdx.x; i < a.d; i += kThreads) {
    const float xh = unpack_one(a.codes[r * a.c_ld + i], a.scales[r * a.s_ld + i / kGroup]) * rstd;
    const float wi = to_float(w[i]);
    float dx = rstd * (to_float(dy[i]) * wi - xh * along);
    if (a.dh) dx += to_float(static_cast<const T*>(a.dh)[r * a.dh_ld + i]);
    static_cast<T*>(a.dx)[r * a.dx_ld + i] = from_float<T>(dx);
    if (a.y) static_cast<T*>(a.y)[r * a.y_ld + i] = from_float<T>(xh * wi);
  }
}

// part[p][i] = sum of dy x^ over the p-th share of the rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) rmsnorm_dw_part_kernel(const NormBwd a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.d) return;
  const int64_t share = (a.rows + a.parts - 1) / a.parts, r0 = blockIdx.y * share, r1 = min(r0 + share, a.rows);
  float sum = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float xh = unpack_one(a.codes[r * a.c_ld + i], a.scales[r * a.s_ld + i / kGroup]) * a.rstd[r];
    sum = fmaf(to_float(static_cast<const T*>(a.dy)[r * a.dy_ld + i]), xh, sum);
  }
  a.part[blockIdx.y * a.d + i] = sum;
}

// dw = the partial sums, always added in the same order: a warp takes every kSumWarps-th of 32 columns' partials.
constexpr int kSumWarps = 32;
template <typename T>
__global__ void __launch_bounds__(kSumWarps * 32) rmsnorm_dw_sum_kernel(const NormBwd a) {
  chain_wait();
  __shared__ float ws[kSumWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (i < a.d) {
#pragma unroll 8
    for (int p = warp; p < a.parts; p += kSumWarps) sum += a.part[p * a.d + i];
  }
  ws[warp][lane] = sum;
  __syncthreads();
  if (warp || i >= a.d) return;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kSumWarps; ++w) sum += ws[w][lane];
  static_cast<T*>(a.dw)[i] = from_float<T>(sum);
}

// Threads of a CTA: 16 values each (32 in rows over kHalfRow), eight warps where a warp holds rows.
int threads_of(int64_t d) {
  if (d <= kWarpRow) return kThreads;
  return (int)(d <= kHalfRow ? (d + 511) / 512 : (d + 1023) / 1024) * 32;
}
// Lanes of a row of up to kWarpRow values: a power of two, two at least (a group).
int lanes_of(int64_t d) {
  int n = 2;
  while (n * 16 < d) n *= 2;
  return n;
}
// Partial sums of dw: the CTAs of the backward kernel.  About 1024 threads an SM (the registers of more would not
// fit); fewer where a CTA's rows one after another would be less than 8, down to two CTAs an SM, since a CTA's partial sums
// cost what a row does.  us with at least 1, 2, 4, 8, 16 rows: 3295 x 768 bf16 13.9, 12.5, 9.8, 11.4, 12.0; 2048 x 4096 17.6, 17.5,
// 17.5, 14.7, 14.8; 5374 x 530 25.0, 25.0, 26.7, 26.2, 38.7.  No number is the best of all three: 8 is within a sixth of each
// size's best, 4 and fewer lose a fifth at the second or more at the first.
int parts_of(int64_t rows, int64_t d) {
  if (d > kMaxRow) return (int)std::max<int64_t>(1, std::min<int64_t>(rows / 8, 128));
  const int64_t at_once = d <= kWarpRow ? kWarps * (32 / lanes_of(d)) : 1;  // rows of a CTA
  const int64_t turns = (rows + at_once - 1) / at_once;
  const int64_t few = std::min<int64_t>(turns, 2 * 148);
  return (int)std::min<int64_t>(std::max<int64_t>((turns + 7) / 8, few), 148 * (1024 / threads_of(d)));
}

}  // namespace
}  // namespace gsa

using namespace gsa;

extern "C" {

int gsa_add_rmsnorm_pack(int dtype, int64_t rows, int64_t d, const void* x, int64_t x_ld, const void* a, int64_t a_ld,
                         const void* weight, float eps, void* h, int64_t h_ld, void* y, int64_t y_ld, uint8_t* codes,
                         int64_t c_ld, uint8_t* scales, int64_t s_ld, float* rstd, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || d < 1 || rows > 0x7fffffffLL) return GSA_ERR_BAD_ARG;
  if (rows == 0) return GSA_OK;
  if (!x || x_ld < 0 || (a && a_ld < 0) || !weight || !y || y_ld < d || (h && (!a || h_ld < d)) || !rstd ||
      !packed_ok(codes, c_ld, scales, s_ld, d))
    return GSA_ERR_BAD_ARG;
  const int lanes = lanes_of(std::min<int64_t>(d, kWarpRow));
  const NormFwd p{rows, d, x,     a,      weight, x_ld, a_ld, eps,  h,
                  y,    h_ld, y_ld, codes, scales, c_ld, s_ld, rstd, lanes};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const int threads = threads_of(d);
    const bool whole = d % 16 == 0 && halves_ok<T>(x, x_ld) && (!a || halves_ok<T>(a, a_ld)) &&
                       (!h || halves_ok<T>(h, h_ld)) && halves_ok<T>(y, y_ld) && halves_ok<T>(weight, 0);
    auto go = [&](auto ragged) {
      constexpr bool kRagged = decltype(ragged)::value;
      const unsigned row_grid = (unsigned)rows;
      if (d <= kWarpRow) {
        const int64_t per = kWarps * (32 / lanes);
        add_rmsnorm_pack16_kernel<T, kRagged, true, 1, kThreads>
            <<<(unsigned)((rows + per - 1) / per), kThreads, 0, s>>>(p);
      } else if (d <= kHalfRow) {
        add_rmsnorm_pack16_kernel<T, kRagged, false, 1, 512><<<row_grid, threads, 0, s>>>(p);
      } else if (d <= kMaxRow) {
        if constexpr (kRagged)  // 32 values a thread would leave one CTA an SM
          add_rmsnorm_pack16_kernel<T, true, false, 1, 1024><<<row_grid, (unsigned)((d + 511) / 512 * 32), 0, s>>>(p);
        else
          add_rmsnorm_pack16_kernel<T, false, false, 2, 512><<<row_grid, threads, 0, s>>>(p);
      } else {
        add_rmsnorm_pack_long_kernel<T><<<row_grid, kThreads, 0, s>>>(p);
      }
    };
    whole ? go(std::false_type()) : go(std::true_type());
  });
  return launch_status();
}

int64_t gsa_rmsnorm_packed_workspace_size(int64_t rows, int64_t d) {
  return rows > 0 && d > 0 ? parts_of(rows, d) * d * (int64_t)sizeof(float) : 0;
}

int gsa_rmsnorm_packed_backward(int dtype, int64_t rows, int64_t d, const void* dy, int64_t dy_ld, const void* dh,
                                int64_t dh_ld, const void* weight, const uint8_t* codes, int64_t c_ld,
                                const uint8_t* scales, int64_t s_ld, const float* rstd, void* dx, int64_t dx_ld,
                                void* y, int64_t y_ld, void* dw, void* workspace, int64_t workspace_bytes,
                                gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || d < 1 || rows > 0x7fffffffLL) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (!dw) return GSA_OK;
    return cudaMemsetAsync(dw, 0, d * (dtype == GSA_DTYPE_BF16 ? 2 : 4), s) == cudaSuccess ? GSA_OK : GSA_ERR_CUDA;
  }
  if (!dy || dy_ld < 0 || (dh && dh_ld < 0) || !weight || !rstd || !dx || dx_ld < d || (y && y_ld < d) ||
      !packed_ok(codes, c_ld, scales, s_ld, d))
    return GSA_ERR_BAD_ARG;
  if (dw && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
             workspace_bytes < gsa_rmsnorm_packed_workspace_size(rows, d)))
    return GSA_ERR_WORKSPACE;
  const NormBwd p{rows, d,    dy, dh, weight, dy_ld, dh_ld, codes, scales, c_ld,
                  s_ld, rstd, dx, y,  dw,     dx_ld, y_ld,  static_cast<float*>(workspace), parts_of(rows, d),
                  lanes_of(std::min<int64_t>(d, kWarpRow))};
  int status = GSA_OK;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const int threads = threads_of(d);
    const bool whole = d % 16 == 0 && halves_ok<T>(dy, dy_ld) && (!dh || halves_ok<T>(dh, dh_ld)) &&
                       halves_ok<T>(dx, dx_ld) && (!y || halves_ok<T>(y, y_ld)) && halves_ok<T>(weight, 0);
    auto go = [&](auto ragged) {
      constexpr bool kRagged = decltype(ragged)::value;
      if (d <= kWarpRow) {
        rmsnorm_bwd16_kernel<T, kRagged, true><<<p.parts, kThreads, 0, s>>>(p);
      } else if (d <= kHalfRow) {
        rmsnorm_bwd16_kernel<T, kRagged, false><<<p.parts, threads, 0, s>>>(p);
      } else if (d <= kMaxRow) {
        rmsnorm_bwd32_kernel<T, kRagged><<<p.parts, threads, 0, s>>>(p);
      } else {
        rmsnorm_bwd_long_kernel<T><<<(unsigned)rows, kThreads, 0, s>>>(p);
        if (dw)
          rmsnorm_dw_part_kernel<T><<<dim3((unsigned)((d + kThreads - 1) / kThreads), p.parts), kThreads, 0, s>>>(p);
      }
    };
    whole ? go(std::false_type()) : go(std::true_type());
    status = launch_status();
    if (status == GSA_OK && dw &&
        launch_chained(rmsnorm_dw_sum_kernel<T>, (unsigned)((d + 31) / 32), kSumWarps * 32, 0, s, p) != cudaSuccess)
      status = GSA_ERR_LAUNCH;
  });
  return status;
}

}  // extern "C"
