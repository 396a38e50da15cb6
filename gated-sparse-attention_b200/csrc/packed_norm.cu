// Residual add + RMSNorm that keeps the sum in 8 bits for its backward pass (the form: packed.cuh).
//
//   h = x + a, r = (mean h^2 + eps)^(-1/2), y = h r w, h kept packed with r; backward, with x^ = h^ r:
//   dx = r (dy w - x^ mean(dy w x^)) + dh,  dw = sum_rows dy x^,  y again = x^ w
//
// Products, sums and statistics are in 32 bits; an output is rounded once, to its type.  h is rounded to its type
// before the norm, since the residual stream that the backward pass differentiates is what the tensor holds.
#include <algorithm>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Sum over the CTA, the same value in every thread; ws: kWarps floats, free for the next sum on return.
__device__ __forceinline__ float block_sum(float v, float* ws) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += ws[w];
  __syncthreads();
  return t;
}

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
};

template <typename T>
__device__ __forceinline__ float residual(const NormFwd& a, int64_t r, int64_t i) {
  float v = to_float(static_cast<const T*>(a.x)[r * a.x_ld + i]);
  if (a.a) v = to_float(from_float<T>(v + to_float(static_cast<const T*>(a.a)[r * a.a_ld + i])));
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) add_rmsnorm_pack_kernel(const NormFwd a) {
  __shared__ float ws[kWarps];
  const int64_t r = blockIdx.x, padded = (a.d + kGroup - 1) / kGroup * kGroup;
  float ss = 0.f;
  for (int64_t i = threadIdx.x; i < a.d; i += kThreads) {
    const float v = residual<T>(a, r, i);
    ss = fmaf(v, v, ss);
  }
  const float rstd = 1.0f / sqrtf(block_sum(ss, ws) / (float)a.d + a.eps);
  if (threadIdx.x == 0) a.rstd[r] = rstd;
  for (int64_t i = threadIdx.x; i < padded; i += kThreads) {  // whole warps: a group is a warp's 32 lanes
    const float v = i < a.d ? residual<T>(a, r, i) : 0.f;
    int s;
    const uint32_t c = pack_lane(v, &s);
    if (i < a.c_ld) a.codes[r * a.c_ld + i] = (uint8_t)c;
    if ((threadIdx.x & 31) == 0) a.scales[r * a.s_ld + i / kGroup] = (uint8_t)s;
    if (i < a.d) {
      if (a.h) static_cast<T*>(a.h)[r * a.h_ld + i] = from_float<T>(v);
      static_cast<T*>(a.y)[r * a.y_ld + i] = from_float<T>(v * rstd * to_float(static_cast<const T*>(a.w)[i]));
    }
  }
}

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
};

template <typename T>
__global__ void __launch_bounds__(kThreads) rmsnorm_bwd_kernel(const NormBwd a) {
  __shared__ float ws[kWarps];
  const int64_t r = blockIdx.x;
  const float rstd = a.rstd[r];
  const T *dy = static_cast<const T*>(a.dy) + r * a.dy_ld, *w = static_cast<const T*>(a.w);
  float along = 0.f;
  for (int64_t i = threadIdx.x; i < a.d; i += kThreads) {
    const float xh = unpack_one(a.codes[r * a.c_ld + i], a.scales[r * a.s_ld + i / kGroup]) * rstd;
    along = fmaf(to_float(dy[i]) * to_float(w[i]), xh, along);
  }
  along = block_sum(along, ws) / (float)a.d;
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

// ---------------------------------------------------------------------------------------------
// A row in registers, 16 values a thread (half a group: one shuffle gives its scale): one CTA a row, or one warp a
// row for rows of up to 512 values.  Every tensor is read once and written once.
// ---------------------------------------------------------------------------------------------
constexpr int kWarpRow = 512;    // values of a row that a warp holds
constexpr int kMaxRow = 16384;   // values of a row that a CTA of 1024 threads holds

// Sum over the threads of a row, the same value in each of them.
template <bool kWarpRows>
__device__ __forceinline__ float row_sum(float v, float* ws) {
  v = warp_sum(v);
  if (kWarpRows) return v;
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? ws[lane] : 0.f);
}

template <typename T, bool kWarpRows, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) add_rmsnorm_pack16_kernel(const NormFwd a) {
  __shared__ float ws[32];
  const int64_t r = kWarpRows ? (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarpRows && r >= a.rows) return;
  const int64_t i = (kWarpRows ? threadIdx.x & 31 : threadIdx.x) * 16;
  const bool live = i < a.d;
  Half<T> hx, ha, hw;
  hx.zero();
  ha.zero();
  hw.zero();
  if (live) {
    hx.load(static_cast<const T*>(a.x) + r * a.x_ld + i);
    if (a.a) ha.load(static_cast<const T*>(a.a) + r * a.a_ld + i);
    hw.load_shared(static_cast<const T*>(a.w) + i);
  }
  float v[16], t[16];
  hx.get(v);
  if (a.a) {
    ha.get(t);
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] += t[k];
    hx.set(v);
    if (live && a.h) hx.store(static_cast<T*>(a.h) + r * a.h_ld + i);
    hx.get(v);
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) ss = fmaf(v[k], v[k], ss);
  const float rstd = 1.0f / sqrtf(row_sum<kWarpRows>(ss, ws) / (float)a.d + a.eps);
  if (live) {
    hw.get(t);
#pragma unroll
    for (int k = 0; k < 16; ++k) t[k] = v[k] * rstd * t[k];
    store_half(static_cast<T*>(a.y) + r * a.y_ld + i, t);
  }
  uint4 q;
  const int s = pack_half(v, &q);
  if (i == 0) a.rstd[r] = rstd;
  if (!live) return;
  store_codes(a.codes + r * a.c_ld + i, q);
  if ((threadIdx.x & 1) == 0) a.scales[r * a.s_ld + i / kGroup] = (uint8_t)s;
}

// What the backward pass reads of a row; the next row's is loaded before this row's sum is waited for.
template <typename T>
struct RowIn {
  Half<T> dy, dh;
  uint4 codes;
  float scale, rstd;
  __device__ __forceinline__ void load(const NormBwd& a, int64_t r, int64_t i, bool live) {
    dy.zero();
    dh.zero();
    codes = make_uint4(0, 0, 0, 0);
    scale = rstd = 0.f;
    if (r >= a.rows || !live) return;
    dy.load(static_cast<const T*>(a.dy) + r * a.dy_ld + i);
    codes = load_codes(a.codes + r * a.c_ld + i);
    if (a.dh) dh.load(static_cast<const T*>(a.dh) + r * a.dh_ld + i);
    scale = pow2_of(a.scales[r * a.s_ld + i / kGroup]);
    rstd = a.rstd[r];
  }
};

// Rows blockIdx.x, blockIdx.x + gridDim.x, ... (of kWarps rows each for warp rows); part[blockIdx.x] = the CTA's sum of
// dy x^ over its rows, in that order.
template <typename T, bool kWarpRows, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) rmsnorm_bwd16_kernel(const NormBwd a) {
  __shared__ float ws[2][32];
  __shared__ float col[kWarpRows ? kWarps : 1][kWarpRows ? kWarpRow : 1];
  const int warp = threadIdx.x >> 5;
  const int64_t per = kWarpRows ? kWarps : 1;
  const int64_t i = (kWarpRows ? threadIdx.x & 31 : threadIdx.x) * 16;
  const bool live = i < a.d;
  Half<T> hw;
  hw.zero();
  if (live) hw.load_shared(static_cast<const T*>(a.w) + i);
  float acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
  RowIn<T> in;
  int64_t r = blockIdx.x * per + (kWarpRows ? warp : 0);
  in.load(a, r, i, live);
  const float inv_d = 1.0f / (float)a.d;
  for (int turn = 0; r < a.rows; ++turn) {
    const RowIn<T> cur = in;
    const int64_t next = r + gridDim.x * per;
    in.load(a, next, i, live);
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
    along = row_sum<kWarpRows>(along, ws[turn & 1]) * inv_d;
    if (live) {
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
    r = next;
  }
  if (!a.dw) return;
  float* part = a.part + (int64_t)blockIdx.x * a.d;
  if (kWarpRows) {
#pragma unroll
    for (int k = 0; k < 16; ++k) col[warp][i + k] = acc[k];
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += col[w][c];
      part[c] = t;
    }
  } else if (live) {
#pragma unroll
    for (int k = 0; k < 16; k += 4)
      *reinterpret_cast<float4*>(part + i + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
  }
}

// dw = the partial sums, always added in the same order: a warp takes every kSumWarps-th of 32 columns' partials.
constexpr int kSumWarps = 16;
template <typename T>
__global__ void __launch_bounds__(kSumWarps * 32) rmsnorm_dw_sum_kernel(const NormBwd a) {
  chain_wait();
  __shared__ float ws[kSumWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (i < a.d) {
#pragma unroll 4
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

// Partial sums of dw: the CTAs of the backward kernel.  About 1024 threads an SM (the registers of more would not
// fit), and at least one row of a CTA or warp each.
int threads_of(int64_t d) { return d <= kWarpRow ? kThreads : (int)((d + 511) / 512 * 32); }
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
  const NormFwd p{rows, d, x, a, weight, x_ld, a_ld, eps, h, y, h_ld, y_ld, codes, scales, c_ld, s_ld, rstd};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const int threads = threads_of(d);
    if (d % 16 || d > kMaxRow || !halves_ok<T>(x, x_ld) || (a && !halves_ok<T>(a, a_ld)) ||
        (h && !halves_ok<T>(h, h_ld)) || !halves_ok<T>(y, y_ld) || !halves_ok<T>(weight, 0))
      add_rmsnorm_pack_kernel<T><<<(unsigned)rows, kThreads, 0, s>>>(p);
    else if (d <= kWarpRow)
      add_rmsnorm_pack16_kernel<T, true, kThreads><<<(unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, s>>>(p);
    else if (threads <= 512)
      add_rmsnorm_pack16_kernel<T, false, 512><<<(unsigned)rows, threads, 0, s>>>(p);
    else
      add_rmsnorm_pack16_kernel<T, false, 1024><<<(unsigned)rows, threads, 0, s>>>(p);
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
  if (dw && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < gsa_rmsnorm_packed_workspace_size(rows, d))) return GSA_ERR_WORKSPACE;
  const NormBwd p{rows, d,    dy,   dh, weight, dy_ld, dh_ld, codes, scales, c_ld,
                  s_ld, rstd, dx,   y,  dw,     dx_ld, y_ld,  static_cast<float*>(workspace), parts_of(rows, d)};
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const int threads = threads_of(d);
    if (d % 16 || d > kMaxRow || !halves_ok<T>(dy, dy_ld) || (dh && !halves_ok<T>(dh, dh_ld)) ||
        !halves_ok<T>(dx, dx_ld) || (y && !halves_ok<T>(y, y_ld)) || !halves_ok<T>(weight, 0)) {
      rmsnorm_bwd_kernel<T><<<(unsigned)rows, kThreads, 0, s>>>(p);
      if (dw) rmsnorm_dw_part_kernel<T><<<dim3((unsigned)((d + kThreads - 1) / kThreads), p.parts), kThreads, 0, s>>>(p);
    } else if (d <= kWarpRow) {
      rmsnorm_bwd16_kernel<T, true, kThreads><<<p.parts, kThreads, 0, s>>>(p);
    } else if (threads <= 512) {
      rmsnorm_bwd16_kernel<T, false, 512><<<p.parts, threads, 0, s>>>(p);
    } else {
      rmsnorm_bwd16_kernel<T, false, 1024><<<p.parts, threads, 0, s>>>(p);
    }
    if (dw) launch_chained(rmsnorm_dw_sum_kernel<T>, (unsigned)((d + 31) / 32), kSumWarps * 32, 0, s, p);
  });
  return launch_status();
}

}  // extern "C"
