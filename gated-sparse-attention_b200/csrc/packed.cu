// Activations kept in 8 bits for the backward pass (the form: packed.cuh), and the two decoder-layer products
// that use them: the residual add with its RMSNorm, and the SwiGLU product.  All are bound by the bytes
// that they move.
//
//   pack / unpack   x -> codes, scales -> x^
//   silu_mul        z = g sigma(g) u, (g, u) kept packed; backward, from the packed g^, u^:
//                   dg = dz u^ sigma (1 + g^ (1 - sigma)), du = dz g^ sigma, z again for the weight gradient of the
//                   product that reads it
//   add_rmsnorm     h = x + a, r = (mean h^2 + eps)^(-1/2), y = h r w, h kept packed with r; backward, with
//                   x^ = h^ r:  dx = r (dy w - x^ mean(dy w x^)) + dh,  dw = sum_rows dy x^,  y again = x^ w
//
// Products, sums and statistics are in 32 bits; an output is rounded once, to its type.  h is rounded to its type
// before the norm, since the residual stream that the backward pass differentiates is what the tensor holds.
#include <algorithm>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// One group by one warp, a value a lane: its code and the scale byte; returns the code (in the low byte).
__device__ __forceinline__ uint32_t pack_lane(float x, int* scale) {
  const int s = scale_byte(__reduce_max_sync(0xffffffffu, finite_abs_bits(x)));
  *scale = s;
  return to_e4m3x2(inf_to_nan(x) * inv_pow2_of(s), 0.f) & 0xffu;
}

__device__ __forceinline__ float unpack_one(uint8_t code, uint8_t scale) {
  return from_e4m3x2(code).x * pow2_of(scale);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(int64_t rows, int64_t n, const T* x, int64_t x_ld,
                                                        uint8_t* codes, int64_t c_ld, uint8_t* scales, int64_t s_ld) {
  const int64_t groups = (n + kGroup - 1) / kGroup, total = rows * groups;
  const int lane = threadIdx.x & 31;
  for (int64_t g = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); g < total; g += (int64_t)gridDim.x * kWarps) {
    const int64_t r = g / groups, i = (g - r * groups) * kGroup + lane;
    int s;
    const uint32_t c = pack_lane(i < n ? to_float(x[r * x_ld + i]) : 0.f, &s);
    if (i < c_ld) codes[r * c_ld + i] = (uint8_t)c;
    if (lane == 0) scales[r * s_ld + i / kGroup] = (uint8_t)s;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack_kernel(int64_t rows, int64_t n, const uint8_t* codes, int64_t c_ld,
                                                          const uint8_t* scales, int64_t s_ld, T* x, int64_t x_ld) {
  const int64_t total = rows * n;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t r = e / n, i = e - r * n;
    x[r * x_ld + i] = from_float<T>(unpack_one(codes[r * c_ld + i], scales[r * s_ld + i / kGroup]));
  }
}

__device__ __forceinline__ float sigmoid32(float x) { return 1.0f / (1.0f + expf(-x)); }

// gu rows hold g then u; the packed rows 2r and 2r + 1 are row r's g and u.
template <typename T>
__global__ void __launch_bounds__(kThreads) silu_mul_pack_kernel(int64_t rows, int64_t n, const T* gu, int64_t gu_ld,
                                                                 T* z, int64_t z_ld, uint8_t* codes, int64_t c_ld,
                                                                 uint8_t* scales, int64_t s_ld) {
  const int64_t groups = (n + kGroup - 1) / kGroup, total = rows * groups;
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5); w < total; w += (int64_t)gridDim.x * kWarps) {
    const int64_t r = w / groups, i = (w - r * groups) * kGroup + lane;
    const float g = i < n ? to_float(gu[r * gu_ld + i]) : 0.f;
    const float u = i < n ? to_float(gu[r * gu_ld + n + i]) : 0.f;
    if (i < n) z[r * z_ld + i] = from_float<T>(g * sigmoid32(g) * u);
    int sg, su;
    const uint32_t cg = pack_lane(g, &sg), cu = pack_lane(u, &su);
    if (i < c_ld) {
      codes[2 * r * c_ld + i] = (uint8_t)cg;
      codes[(2 * r + 1) * c_ld + i] = (uint8_t)cu;
    }
    if (lane == 0) {
      scales[2 * r * s_ld + i / kGroup] = (uint8_t)sg;
      scales[(2 * r + 1) * s_ld + i / kGroup] = (uint8_t)su;
    }
  }
}

struct SwigluGrad {
  float dg, du, z;
};
__device__ __forceinline__ SwigluGrad swiglu_grad(float dz, float g, float u) {
  const float sig = sigmoid32(g), silu = g * sig;
  return {dz * u * (sig * (1.0f + g * (1.0f - sig))), dz * silu, silu * u};
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    silu_mul_bwd_kernel(int64_t rows, int64_t n, const T* dz, int64_t dz_ld, const uint8_t* codes, int64_t c_ld,
                        const uint8_t* scales, int64_t s_ld, T* dgu, int64_t dgu_ld, T* z, int64_t z_ld) {
  const int64_t total = rows * n;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kThreads) {
    const int64_t r = e / n, i = e - r * n, r2 = 2 * r;
    const float g = unpack_one(codes[r2 * c_ld + i], scales[r2 * s_ld + i / kGroup]);
    const float u = unpack_one(codes[(r2 + 1) * c_ld + i], scales[(r2 + 1) * s_ld + i / kGroup]);
    const SwigluGrad d = swiglu_grad(to_float(dz[r * dz_ld + i]), g, u);
    dgu[r * dgu_ld + i] = from_float<T>(d.dg);
    dgu[r * dgu_ld + n + i] = from_float<T>(d.du);
    if (z) z[r * z_ld + i] = from_float<T>(d.z);
  }
}

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

// dw = the partial sums, always added in the same order.
template <typename T>
__global__ void __launch_bounds__(kThreads) rmsnorm_dw_sum_kernel(const NormBwd a) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.d) return;
  float sum = 0.f;
  for (int p = 0; p < a.parts; ++p) sum += a.part[p * a.d + i];
  static_cast<T*>(a.dw)[i] = from_float<T>(sum);
}

int parts_of(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(rows / 8, 128)); }

unsigned grid_of(int64_t blocks) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, 148 * 32)); }

int launched() { return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH; }

bool type_ok(int dtype) { return dtype == GSA_DTYPE_F32 || dtype == GSA_DTYPE_BF16; }

// Packed rows of n values: whole 16-byte pieces of codes, a scale byte for each group.
bool packed_ok(const uint8_t* codes, int64_t c_ld, const uint8_t* scales, int64_t s_ld, int64_t n) {
  return codes && scales && c_ld >= (n + 15) / 16 * 16 && c_ld % 16 == 0 &&
         reinterpret_cast<uintptr_t>(codes) % 16 == 0 && s_ld >= (n + kGroup - 1) / kGroup;
}

// Calls f with a value of the element type.
template <typename F>
void typed(int dtype, F f) {
  if (dtype == GSA_DTYPE_BF16)
    f(__nv_bfloat16());
  else
    f(float());
}

}  // namespace
}  // namespace gsa

using namespace gsa;

extern "C" {

int gsa_pack_e4m3(int dtype, int64_t rows, int64_t n, const void* x, int64_t x_ld, uint8_t* codes, int64_t c_ld,
                  uint8_t* scales, int64_t s_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!x || x_ld < 0 || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = grid_of((rows * ((n + kGroup - 1) / kGroup) + kWarps - 1) / kWarps);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    pack_kernel<T><<<grid, kThreads, 0, s>>>(rows, n, static_cast<const T*>(x), x_ld, codes, c_ld, scales, s_ld);
  });
  return launched();
}

int gsa_unpack_e4m3(int dtype, int64_t rows, int64_t n, const uint8_t* codes, int64_t c_ld, const uint8_t* scales,
                    int64_t s_ld, void* x, int64_t x_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!x || x_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = grid_of((rows * n + kThreads - 1) / kThreads);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    unpack_kernel<T><<<grid, kThreads, 0, s>>>(rows, n, codes, c_ld, scales, s_ld, static_cast<T*>(x), x_ld);
  });
  return launched();
}

int gsa_silu_mul_pack(int dtype, int64_t rows, int64_t n, const void* gu, int64_t gu_ld, void* z, int64_t z_ld,
                      uint8_t* codes, int64_t c_ld, uint8_t* scales, int64_t s_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!gu || gu_ld < 0 || !z || z_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = grid_of((rows * ((n + kGroup - 1) / kGroup) + kWarps - 1) / kWarps);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    silu_mul_pack_kernel<T><<<grid, kThreads, 0, s>>>(rows, n, static_cast<const T*>(gu), gu_ld, static_cast<T*>(z),
                                                      z_ld, codes, c_ld, scales, s_ld);
  });
  return launched();
}

int gsa_silu_mul_packed_backward(int dtype, int64_t rows, int64_t n, const void* dz, int64_t dz_ld,
                                 const uint8_t* codes, int64_t c_ld, const uint8_t* scales, int64_t s_ld, void* dgu,
                                 int64_t dgu_ld, void* z, int64_t z_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!dz || dz_ld < 0 || !dgu || dgu_ld < 2 * n || (z && z_ld < n) || !packed_ok(codes, c_ld, scales, s_ld, n))
    return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = grid_of((rows * n + kThreads - 1) / kThreads);
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    silu_mul_bwd_kernel<T><<<grid, kThreads, 0, s>>>(rows, n, static_cast<const T*>(dz), dz_ld, codes, c_ld, scales,
                                                     s_ld, static_cast<T*>(dgu), dgu_ld, static_cast<T*>(z), z_ld);
  });
  return launched();
}

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
  typed(dtype, [&](auto e) { add_rmsnorm_pack_kernel<decltype(e)><<<(unsigned)rows, kThreads, 0, s>>>(p); });
  return launched();
}

int64_t gsa_rmsnorm_packed_workspace_size(int64_t rows, int64_t d) {
  return rows > 0 && d > 0 ? parts_of(rows) * d * (int64_t)sizeof(float) : 0;
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
  if (dw && (!workspace || workspace_bytes < gsa_rmsnorm_packed_workspace_size(rows, d))) return GSA_ERR_WORKSPACE;
  const NormBwd p{rows, d,    dy,   dh, weight, dy_ld, dh_ld, codes, scales, c_ld,
                  s_ld, rstd, dx,   y,  dw,     dx_ld, y_ld,  static_cast<float*>(workspace), parts_of(rows)};
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    rmsnorm_bwd_kernel<T><<<(unsigned)rows, kThreads, 0, s>>>(p);
    if (!dw) return;
    const unsigned cols = (unsigned)((d + kThreads - 1) / kThreads);
    rmsnorm_dw_part_kernel<T><<<dim3(cols, p.parts), kThreads, 0, s>>>(p);
    rmsnorm_dw_sum_kernel<T><<<cols, kThreads, 0, s>>>(p);
  });
  return launched();
}

}  // extern "C"
