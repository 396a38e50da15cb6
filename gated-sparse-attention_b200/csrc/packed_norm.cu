// Residual add + RMSNorm that keeps the sum in 8 bits for its backward pass (the form: packed.cuh).
//
//   h = x + a, r = (mean h^2 + eps)^(-1/2), y = h r w, h kept packed with r; backward, with x^ = h^ r:
//   dx = r (dy w - x^ mean(dy w x^)) + dh,  dw = sum_rows dy x^,  y again = x^ w
//
// Products, sums and statistics are in 32 bits; an output is rounded once, to its type.  h is rounded to its type
// before the norm, since the residual stream that the backward pass differentiates is what the tensor holds.
//
// Bound by the bytes that it moves: a row is held in registers, so every tensor is read once and written once.  A thread
// holds 16 neighbouring values (half a group: 32-byte accesses, one shuffle for the scale) where rows are whole
// multiples of that and aligned, else 16 values a row's threads apart (a group a warp).  A CTA takes a row, or a
// warp one of up to 512 values (several, where rows are shorter still).  The backward pass keeps its CTAs for all rows:
// each sums dw beside dx over its rows in order, and a last kernel adds the CTAs' sums in order.
#include <algorithm>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWarpRow = 512;   // values of a row that a warp holds
constexpr int kLaneRow = 8192;  // values of an unaligned row that a CTA holds, 16 a thread
constexpr int kMaxRow = 16384;  // values of an aligned row that a CTA holds, 16 or 32 a thread

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
template <typename T, bool kWarpRows, int kHalves, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) add_rmsnorm_pack16_kernel(const NormFwd a) {
  __shared__ float ws[32];
  const int lane = threadIdx.x & 31, per = kWarpRows ? 32 / a.lanes : 1;
  const int64_t r = kWarpRows ? ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * per + lane / a.lanes : blockIdx.x;
  const int64_t i0 = (kWarpRows ? lane & (a.lanes - 1) : threadIdx.x) * 16;
  const int64_t step = (int64_t)blockDim.x * 16;  // between a thread's halves
  float v[kHalves][16], ss = 0.f;
#pragma unroll
  for (int j = 0; j < kHalves; ++j) {
    const int64_t i = i0 + j * step;
    const bool live = i < a.d && r < a.rows;
    Half<T> hx, ha;
    hx.zero();
    ha.zero();
    if (live) {
      hx.load(static_cast<const T*>(a.x) + r * a.x_ld + i);
      if (a.a) ha.load(static_cast<const T*>(a.a) + r * a.a_ld + i);
    }
    hx.get(v[j]);
    if (a.a) {
      float t[16];
      ha.get(t);
#pragma unroll
      for (int k = 0; k < 16; ++k) v[j][k] += t[k];
      hx.set(v[j]);
      if (live && a.h) hx.store(static_cast<T*>(a.h) + r * a.h_ld + i);
      hx.get(v[j]);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) ss = fmaf(v[j][k], v[j][k], ss);
  }
  const float rstd = rstd_of(row_sum<kWarpRows>(ss, a.lanes, ws), a);
  if (i0 == 0 && r < a.rows) a.rstd[r] = rstd;
#pragma unroll
  for (int j = 0; j < kHalves; ++j) {
    const int64_t i = i0 + j * step;
    const bool live = i < a.d && r < a.rows;
    if (live) {
      Half<T> hw;
      hw.load_shared(static_cast<const T*>(a.w) + i);
      float t[16];
      hw.get(t);
#pragma unroll
      for (int k = 0; k < 16; ++k) t[k] = v[j][k] * rstd * t[k];
      store_half(static_cast<T*>(a.y) + r * a.y_ld + i, t);
    }
    uint4 q;
    const int s = pack_half(v[j], &q);
    if (!live) continue;
    store_codes(a.codes + r * a.c_ld + i, q);
    if ((threadIdx.x & 1) == 0) a.scales[r * a.s_ld + i / kGroup] = (uint8_t)s;
  }
}

// What the backward pass reads of 16 values of a row.
template <typename T>
struct RowIn {
  Half<T> dy, dh;
  uint4 codes;
  float scale, rstd;
  __device__ __forceinline__ void load(const NormBwd& a, int64_t r, int64_t i) {
    dy.zero();
    dh.zero();
    codes = make_uint4(0, 0, 0, 0);
    scale = rstd = 0.f;
    if (r >= a.rows || i >= a.d) return;
    dy.load(static_cast<const T*>(a.dy) + r * a.dy_ld + i);
    codes = load_codes(a.codes + r * a.c_ld + i);
    if (a.dh) dh.load(static_cast<const T*>(a.dh) + r * a.dh_ld + i);
    scale = pow2_of(a.scales[r * a.s_ld + i / kGroup]);
    rstd = a.rstd[r];
  }
};

// The columns' sums of a CTA whose warps held rows: acc[k] of column i + k, added over the warps in order.
template <int K>
__device__ __forceinline__ void warp_rows_part(const NormBwd& a, const float* acc, float* part, float (*col)[kWarpRow],
                                               int first, int stride, bool writes) {
  if (writes)
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (first + k * stride < kWarpRow) col[threadIdx.x >> 5][first + k * stride] = acc[k];
  __syncthreads();
  for (int c = threadIdx.x; c < a.d; c += kThreads) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += col[w][c];
    part[c] = t;
  }
}

// Rows blockIdx.x, blockIdx.x + gridDim.x, ... (or as many for each warp); part[blockIdx.x] = the CTA's sum of dy x^ over
// its rows, in that order.  The next row is loaded before this row's sum is waited for.
template <typename T, bool kWarpRows>
__global__ void __launch_bounds__(kWarpRows ? kThreads : 512) rmsnorm_bwd16_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  __shared__ float col[kWarpRows ? kWarps : 1][kWarpRow];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = kWarpRows ? 32 / a.lanes : 1;
  const int64_t i = (kWarpRows ? lane & (a.lanes - 1) : threadIdx.x) * 16;
  Half<T> hw;
  hw.zero();
  if (i < a.d) hw.load_shared(static_cast<const T*>(a.w) + i);
  float acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
  const int64_t step = (int64_t)gridDim.x * (kWarpRows ? kWarps : 1) * per;
  int64_t base = (kWarpRows ? (int64_t)blockIdx.x * kWarps + warp : blockIdx.x) * per;
  const int slot = kWarpRows ? lane / a.lanes : 0;
  RowIn<T> in;
  in.load(a, base + slot, i);
  const float inv_d = 1.0f / (float)a.d;
  for (int turn = 0; base < a.rows; ++turn, base += step) {
    const RowIn<T> cur = in;
    const int64_t r = base + slot;
    in.load(a, r + step, i);
    float dy[16], xh[16], w[16];
    cur.dy.get(dy);
    hw.get(w);
    unpack_half(cur.codes, cur.scale, xh);
    float along = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      xh[k] *= cur.rstd;
      along = fmaf(dy[k] * w[k], xh[k], along);
      acc[k] = fmaf(dy[k], xh[k], acc[k]);
    }
    along = row_sum<kWarpRows>(along, a.lanes, ws[turn & 1]) * inv_d;
    if (i < a.d && r < a.rows) {
      float dh[16];
      cur.dh.get(dh);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        dh[k] += cur.rstd * (dy[k] * w[k] - xh[k] * along);
        xh[k] *= w[k];
      }
      store_half(static_cast<T*>(a.dx) + r * a.dx_ld + i, dh);
      if (a.y) store_half(static_cast<T*>(a.y) + r * a.y_ld + i, xh);
    }
  }
  if (!a.dw) return;
  float* part = a.part + (int64_t)blockIdx.x * a.d;
  if (kWarpRows) {
    for (int o = a.lanes; o < 32; o <<= 1)  // the warp's rows side by side
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[k] += __shfl_xor_sync(0xffffffffu, acc[k], o);
    warp_rows_part<16>(a, acc, part, col, (int)i, 1, lane < a.lanes);
  } else if (i < a.d) {
#pragma unroll
    for (int k = 0; k < 16; k += 4)
      *reinterpret_cast<float4*>(part + i + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
  }
}

// Rows of more than 8192 values: 32 a thread.  Their sums of dw leave no registers to load ahead, or for the weights.
template <typename T>
__global__ void __launch_bounds__(512) rmsnorm_bwd32_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  const int64_t step = (int64_t)blockDim.x * 16;
  float acc[2][16];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[j][k] = 0.f;
  const float inv_d = 1.0f / (float)a.d;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, ++turn) {
    const float rstd = a.rstd[r];
    Half<T> hdy[2];
    uint4 codes[2];
    float scale[2], along = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t i = threadIdx.x * 16 + j * step;
      hdy[j].zero();
      codes[j] = make_uint4(0, 0, 0, 0);
      scale[j] = 0.f;
      if (i >= a.d) continue;
      hdy[j].load(static_cast<const T*>(a.dy) + r * a.dy_ld + i);
      codes[j] = load_codes(a.codes + r * a.c_ld + i);
      scale[j] = pow2_of(a.scales[r * a.s_ld + i / kGroup]) * rstd;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t i = threadIdx.x * 16 + j * step;
      if (i >= a.d) continue;
      Half<T> hw;
      hw.load_shared(static_cast<const T*>(a.w) + i);
      float dy[16], xh[16], w[16];
      hdy[j].get(dy);
      hw.get(w);
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
      if (i >= a.d) continue;
      Half<T> hw, hdh;
      hw.load_shared(static_cast<const T*>(a.w) + i);
      hdh.zero();
      if (a.dh) hdh.load(static_cast<const T*>(a.dh) + r * a.dh_ld + i);
      float dy[16], xh[16], w[16], dh[16];
      hdy[j].get(dy);
      hw.get(w);
      hdh.get(dh);
      unpack_half(codes[j], scale[j], xh);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        dh[k] += rstd * (dy[k] * w[k] - xh[k] * along);
        xh[k] *= w[k];
      }
      store_half(static_cast<T*>(a.dx) + r * a.dx_ld + i, dh);
      if (a.y) store_half(static_cast<T*>(a.y) + r * a.y_ld + i, xh);
    }
  }
  if (!a.dw) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t i = threadIdx.x * 16 + j * step;
    if (i >= a.d) continue;
#pragma unroll
    for (int k = 0; k < 16; k += 4)
      *reinterpret_cast<float4*>(a.part + (int64_t)blockIdx.x * a.d + i + k) =
          make_float4(acc[j][k], acc[j][k + 1], acc[j][k + 2], acc[j][k + 3]);
  }
}

// ---------------------------------------------------------------------------------------------
// Unaligned rows: K values a thread, a row's threads apart.
// ---------------------------------------------------------------------------------------------
template <typename T, bool kWarpRows, int K>
__global__ void __launch_bounds__(kWarpRows ? kThreads : 512) add_rmsnorm_pack_kernel(const NormFwd a) {
  __shared__ float ws[32];
  const int lane = threadIdx.x & 31, stride = kWarpRows ? 32 : blockDim.x, d = (int)a.d;
  const int64_t r = kWarpRows ? (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  if (r >= a.rows) return;
  const int i0 = kWarpRows ? lane : threadIdx.x;
  const T *x = static_cast<const T*>(a.x) + r * a.x_ld, *add = static_cast<const T*>(a.a) + r * a.a_ld;
  const T* w = static_cast<const T*>(a.w);
  T *h = static_cast<T*>(a.h) + r * a.h_ld, *y = static_cast<T*>(a.y) + r * a.y_ld;
  uint8_t *codes = a.codes + r * a.c_ld, *scales = a.scales + r * a.s_ld;
  T vx[K], va[K];  // all loads before the first use
#pragma unroll
  for (int k = 0; k < K; ++k) vx[k] = i0 + k * stride < d ? x[i0 + k * stride] : from_float<T>(0.f);
  if (a.a)
#pragma unroll
    for (int k = 0; k < K; ++k) va[k] = i0 + k * stride < d ? add[i0 + k * stride] : from_float<T>(0.f);
  float v[K], ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = to_float(vx[k]);
    if (a.a) v[k] = to_float(from_float<T>(v[k] + to_float(va[k])));
    ss = fmaf(v[k], v[k], ss);
  }
  const float rstd = rstd_of(row_sum<kWarpRows>(ss, 32, ws), a);
  if (i0 == 0) a.rstd[r] = rstd;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = i0 + k * stride;
    if (i - lane >= d) break;  // whole warps: a group is a warp's 32 lanes
    int s;
    const uint32_t c = pack_lane(v[k], &s);
    if (lane == 0) scales[i / kGroup] = (uint8_t)s;
    if (i < d) {
      codes[i] = (uint8_t)c;
      if (a.h) h[i] = from_float<T>(v[k]);
      y[i] = from_float<T>(v[k] * rstd * to_float(w[i]));
    }
  }
}

template <typename T, bool kWarpRows, int K>
__global__ void __launch_bounds__(kWarpRows ? kThreads : 512) rmsnorm_bwd_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  __shared__ float col[kWarpRows ? kWarps : 1][kWarpRow];
  const int lane = threadIdx.x & 31, stride = kWarpRows ? 32 : blockDim.x, d = (int)a.d;
  const int i0 = kWarpRows ? lane : threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * (kWarpRows ? kWarps : 1);
  int64_t r = kWarpRows ? (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  const T* w = static_cast<const T*>(a.w);
  float acc[K];
#pragma unroll
  for (int k = 0; k < K; ++k) acc[k] = 0.f;
  const float inv_d = 1.0f / (float)a.d;
  for (int turn = 0; r < a.rows; r += step, ++turn) {
    const float rstd = a.rstd[r];
    const T *dy = static_cast<const T*>(a.dy) + r * a.dy_ld, *dh = static_cast<const T*>(a.dh) + r * a.dh_ld;
    T *dx = static_cast<T*>(a.dx) + r * a.dx_ld, *y = static_cast<T*>(a.y) + r * a.y_ld;
    const uint8_t *codes = a.codes + r * a.c_ld, *scales = a.scales + r * a.s_ld;
    T vy[K], vh[K];  // all loads before the first use
    uint8_t vc[K], vs[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + k * stride;
      vy[k] = i < d ? dy[i] : from_float<T>(0.f);
      vc[k] = i < d ? codes[i] : (uint8_t)0;
      vs[k] = i < d ? scales[i / kGroup] : (uint8_t)0;
    }
    if (a.dh)
#pragma unroll
      for (int k = 0; k < K; ++k) vh[k] = i0 + k * stride < d ? dh[i0 + k * stride] : from_float<T>(0.f);
    float xh[K], along = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xh[k] = unpack_one(vc[k], vs[k]) * rstd;
      const float g = to_float(vy[k]), wi = i0 + k * stride < d ? to_float(w[i0 + k * stride]) : 0.f;
      along = fmaf(g * wi, xh[k], along);
      acc[k] = fmaf(g, xh[k], acc[k]);
    }
    along = row_sum<kWarpRows>(along, 32, ws[turn & 1]) * inv_d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + k * stride;
      if (i < d) {
        const float wi = to_float(w[i]);
        float g = rstd * (to_float(vy[k]) * wi - xh[k] * along);
        if (a.dh) g += to_float(vh[k]);
        dx[i] = from_float<T>(g);
        if (a.y) y[i] = from_float<T>(xh[k] * wi);
      }
    }
  }
  if (!a.dw) return;
  float* part = a.part + (int64_t)blockIdx.x * a.d;
  if (kWarpRows) {
    warp_rows_part<K>(a, acc, part, col, i0, stride, true);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (i0 + k * stride < d) part[i0 + k * stride] = acc[k];
  }
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

// Threads of a CTA: 16 values each (32 in rows over kLaneRow), eight warps where a warp holds rows.
int threads_of(int64_t d) {
  if (d <= kWarpRow) return kThreads;
  return (int)(d <= kLaneRow ? (d + 511) / 512 : (d + 1023) / 1024) * 32;
}
// Lanes of an aligned row of up to kWarpRow values: a power of two, two at least (a group).
int lanes_of(int64_t d) {
  int n = 2;
  while (n * 16 < d) n *= 2;
  return n;
}
// Partial sums of dw: the CTAs of the backward kernel.  About 1024 threads an SM (the registers of more would not
// fit), and one row at least for each warp or CTA.
int parts_of(int64_t rows, int64_t d) {
  if (d > kMaxRow) return (int)std::max<int64_t>(1, std::min<int64_t>(rows / 8, 128));
  const int64_t per = d <= kWarpRow ? kWarps : 1;
  return (int)std::min<int64_t>((rows + per - 1) / per, 148 * (1024 / threads_of(d)));
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
    const bool aligned = d % 16 == 0 && halves_ok<T>(x, x_ld) && (!a || halves_ok<T>(a, a_ld)) &&
                         (!h || halves_ok<T>(h, h_ld)) && halves_ok<T>(y, y_ld) && halves_ok<T>(weight, 0);
    const unsigned row_grid = (unsigned)rows, warp_grid = (unsigned)((rows + kWarps - 1) / kWarps);
    if (aligned && d <= kWarpRow) {
      const int64_t per = kWarps * (32 / lanes);
      add_rmsnorm_pack16_kernel<T, true, 1, kThreads><<<(unsigned)((rows + per - 1) / per), kThreads, 0, s>>>(p);
    } else if (aligned && d <= kLaneRow) {
      add_rmsnorm_pack16_kernel<T, false, 1, 512><<<row_grid, threads, 0, s>>>(p);
    } else if (aligned && d <= kMaxRow) {
      add_rmsnorm_pack16_kernel<T, false, 2, 512><<<row_grid, threads, 0, s>>>(p);
    } else if (d <= 128) {
      add_rmsnorm_pack_kernel<T, true, 4><<<warp_grid, kThreads, 0, s>>>(p);
    } else if (d <= kWarpRow) {
      add_rmsnorm_pack_kernel<T, true, 16><<<warp_grid, kThreads, 0, s>>>(p);
    } else if (d <= kLaneRow) {
      add_rmsnorm_pack_kernel<T, false, 16><<<row_grid, threads, 0, s>>>(p);
    } else {
      add_rmsnorm_pack_long_kernel<T><<<row_grid, kThreads, 0, s>>>(p);
    }
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
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const int threads = threads_of(d);
    const bool aligned = d % 16 == 0 && halves_ok<T>(dy, dy_ld) && (!dh || halves_ok<T>(dh, dh_ld)) &&
                         halves_ok<T>(dx, dx_ld) && (!y || halves_ok<T>(y, y_ld)) && halves_ok<T>(weight, 0);
    if (aligned && d <= kWarpRow) {
      rmsnorm_bwd16_kernel<T, true><<<p.parts, kThreads, 0, s>>>(p);
    } else if (aligned && d <= kLaneRow) {
      rmsnorm_bwd16_kernel<T, false><<<p.parts, threads, 0, s>>>(p);
    } else if (aligned && d <= kMaxRow) {
      rmsnorm_bwd32_kernel<T><<<p.parts, threads, 0, s>>>(p);
    } else if (d <= 128) {
      rmsnorm_bwd_kernel<T, true, 4><<<p.parts, kThreads, 0, s>>>(p);
    } else if (d <= kWarpRow) {
      rmsnorm_bwd_kernel<T, true, 16><<<p.parts, kThreads, 0, s>>>(p);
    } else if (d <= kLaneRow) {
      rmsnorm_bwd_kernel<T, false, 16><<<p.parts, threads, 0, s>>>(p);
    } else {
      rmsnorm_bwd_long_kernel<T><<<(unsigned)rows, kThreads, 0, s>>>(p);
      if (dw) rmsnorm_dw_part_kernel<T><<<dim3((unsigned)((d + kThreads - 1) / kThreads), p.parts), kThreads, 0, s>>>(p);
    }
    if (dw) launch_chained(rmsnorm_dw_sum_kernel<T>, (unsigned)((d + 31) / 32), kSumWarps * 32, 0, s, p);
  });
  return launch_status();
}

}  // extern "C"
