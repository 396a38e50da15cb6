// Activations kept in 8 bits for the backward pass (the form: packed.cuh), and the SwiGLU product that keeps its
// operands so.
//
//   pack / unpack   x -> codes, scales -> x^
//   silu_mul        z = g sigma(g) u, (g, u) kept packed; backward, from the packed g^, u^:
//                   dg = dz u^ sigma (1 + g^ (1 - sigma)), du = dz g^ sigma, z again for the weight gradient of the
//                   product that reads it
//
// Products are in 32 bits; an output is rounded once, to its type.  All are bound by the bytes that they move, so
// a thread holds 16 neighbouring values (half a group, 32-byte loads and stores, one shuffle for the scale) wherever
// the rows are whole multiples of that and aligned; rows that are not take a value a lane, four groups a warp.
#include <algorithm>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// 4 sigma(x) = 1 / ((1 + e^-x) / 4): the quarter keeps the reciprocal in the normal range for all e^-x that are, so that
// x sigma(x) has its relative accuracy over the whole range (a plain fast reciprocal gives 0 under 2^-126).  e^-x is
// 2^t times 2^lo with t = -x log2 e rounded and lo what that lost; beyond +-1e4 it is 0 or infinite in any case.
__device__ __forceinline__ float sigmoid_times4(float x) {
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.925963e-8f, kLn2 = 0.693147181f;  // log2 e as a sum of two
  const float c = fminf(fmaxf(x, -1e4f), 1e4f);
  const float t = -c * kLog2e, lo = fmaf(-c, kLog2eLow, fmaf(-c, kLog2e, -t));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e *= fmaf(lo, kLn2, 1.0f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0.25f, 0.25f)));
  return r;
}
__device__ __forceinline__ float silu_mul(float g, float u) { return 0.25f * g * sigmoid_times4(g) * u; }

struct SwigluGrad {
  float dg, du, z;
};
__device__ __forceinline__ SwigluGrad swiglu_grad(float dz, float g, float u) {
  const float s4 = sigmoid_times4(g), sig = 0.25f * s4, silu = 0.25f * g * s4;
  return {dz * u * (sig * (1.0f + g * (1.0f - sig))), dz * silu, silu * u};
}

// ---------------------------------------------------------------------------------------------
// 16 values a thread.  A row is cut into 2 ceil(n / 32) halves, so that the two halves of a group are
// neighbouring lanes; the last may be empty.
// ---------------------------------------------------------------------------------------------
struct Cut {
  int64_t rows, halves, per_row;  // halves (or spans): rows * per_row
  uint64_t magic;
  int64_t n;
};
struct Place {
  int64_t r, i;
  bool live;
};
__device__ __forceinline__ Place place_of(const Cut& c, int skip = 0, int each = 1) {
  const int64_t e = (int64_t)blockIdx.x * each * kThreads + skip + threadIdx.x;
  const int64_t r = row_of(e, c.magic), i = (e - r * c.per_row) * 16;
  return {r, i, e < c.halves && i < c.n};
}

// Two halves a thread, both loaded first: one alone leaves too little in flight for HBM (69 us, 65 with two, for 32768 x
// 4096 bf16).
constexpr int kPackEach = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads) pack16_kernel(const Cut c, const T* x, int64_t x_ld, uint8_t* codes,
                                                          int64_t c_ld, uint8_t* scales, int64_t s_ld) {
  Place p[kPackEach];
  Half<T> h[kPackEach];
#pragma unroll
  for (int j = 0; j < kPackEach; ++j) {
    p[j] = place_of(c, j * kThreads, kPackEach);
    h[j].zero();
    if (p[j].live) h[j].load(x + p[j].r * x_ld + p[j].i);
  }
#pragma unroll
  for (int j = 0; j < kPackEach; ++j) {
    float v[16];
    h[j].get(v);
    uint4 q;
    const int s = pack_half(v, &q);
    if (p[j].live) {
      store_codes(codes + p[j].r * c_ld + p[j].i, q);
      if ((threadIdx.x & 1) == 0) scales[p[j].r * s_ld + p[j].i / kGroup] = (uint8_t)s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack16_kernel(const Cut c, const uint8_t* codes, int64_t c_ld,
                                                            const uint8_t* scales, int64_t s_ld, T* x, int64_t x_ld) {
  const Place p = place_of(c);
  if (!p.live) return;
  float v[16];
  unpack_half(load_codes(codes + p.r * c_ld + p.i), pow2_of(scales[p.r * s_ld + p.i / kGroup]), v);
  store_half(x + p.r * x_ld + p.i, v);
}

// gu rows hold g then u; the packed rows 2r and 2r + 1 are row r's g and u.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) silu_mul_pack16_kernel(const Cut c, const T* gu, int64_t gu_ld, T* z,
                                                                   int64_t z_ld, uint8_t* codes, int64_t c_ld,
                                                                   uint8_t* scales, int64_t s_ld) {
  const Place p = place_of(c);
  Half<T> hg, hu;
  hg.zero();
  hu.zero();
  if (p.live) {
    hg.load(gu + p.r * gu_ld + p.i);
    hu.load(gu + p.r * gu_ld + c.n + p.i);
  }
  float g[16], u[16];
  hg.get(g);
  hu.get(u);
  if (p.live) {
    float o[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = silu_mul(g[k], u[k]);
    store_half(z + p.r * z_ld + p.i, o);
  }
  uint4 qg, qu;
  const int sg = pack_half(g, &qg), su = pack_half(u, &qu);
  if (!p.live) return;
  store_codes(codes + 2 * p.r * c_ld + p.i, qg);
  store_codes(codes + (2 * p.r + 1) * c_ld + p.i, qu);
  if ((threadIdx.x & 1) == 0) {
    scales[2 * p.r * s_ld + p.i / kGroup] = (uint8_t)sg;
    scales[(2 * p.r + 1) * s_ld + p.i / kGroup] = (uint8_t)su;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    silu_mul_bwd16_kernel(const Cut c, const T* dz, int64_t dz_ld, const uint8_t* codes, int64_t c_ld,
                          const uint8_t* scales, int64_t s_ld, T* dgu, int64_t dgu_ld, T* z, int64_t z_ld) {
  const Place p = place_of(c);
  if (!p.live) return;
  const int64_t r2 = 2 * p.r, k0 = p.i / kGroup;
  float d[16], g[16], u[16];
  load_half(dz + p.r * dz_ld + p.i, d);
  unpack_half(load_codes(codes + r2 * c_ld + p.i), pow2_of(scales[r2 * s_ld + k0]), g);
  unpack_half(load_codes(codes + (r2 + 1) * c_ld + p.i), pow2_of(scales[(r2 + 1) * s_ld + k0]), u);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const SwigluGrad s = swiglu_grad(d[k], g[k], u[k]);
    d[k] = s.dg;
    g[k] = s.du;
    u[k] = s.z;
  }
  store_half(dgu + p.r * dgu_ld + p.i, d);
  store_half(dgu + p.r * dgu_ld + c.n + p.i, g);
  if (z) store_half(z + p.r * z_ld + p.i, u);
}

// ---------------------------------------------------------------------------------------------
// A value a lane, kLaneGroups groups of a row a warp.
// ---------------------------------------------------------------------------------------------
constexpr int kLaneGroups = 4;
constexpr int kSpan = kLaneGroups * kGroup;

// The warp's row and the lane's first value in it; false past the last.
__device__ __forceinline__ bool span_of(const Cut& c, int64_t* r, int64_t* i) {
  const int64_t w = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (w >= c.halves) return false;
  *r = c.per_row == 1 ? w : row_of(w, c.magic);
  *i = (w - *r * c.per_row) * kSpan + (threadIdx.x & 31);
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(const Cut c, const T* x, int64_t x_ld, uint8_t* codes,
                                                        int64_t c_ld, uint8_t* scales, int64_t s_ld) {
  int64_t r, i;
  if (!span_of(c, &r, &i)) return;
  float v[kLaneGroups];
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) v[k] = i + k * kGroup < c.n ? to_float(x[r * x_ld + i + k * kGroup]) : 0.f;
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) {
    int s;
    const uint32_t q = pack_lane(v[k], &s);  // by all lanes, in a group beyond the row too
    if (i + k * kGroup < c.n) {
      codes[r * c_ld + i + k * kGroup] = (uint8_t)q;
      if ((threadIdx.x & 31) == 0) scales[r * s_ld + i / kGroup + k] = (uint8_t)s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const Cut c, const uint8_t* codes, int64_t c_ld,
                                                          const uint8_t* scales, int64_t s_ld, T* x, int64_t x_ld) {
  int64_t r, i;
  if (!span_of(c, &r, &i)) return;
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k)
    if (i + k * kGroup < c.n)
      x[r * x_ld + i + k * kGroup] =
          from_float<T>(unpack_one(codes[r * c_ld + i + k * kGroup], scales[r * s_ld + i / kGroup + k]));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) silu_mul_pack_kernel(const Cut c, const T* gu, int64_t gu_ld, T* z,
                                                                 int64_t z_ld, uint8_t* codes, int64_t c_ld,
                                                                 uint8_t* scales, int64_t s_ld) {
  int64_t r, i;
  if (!span_of(c, &r, &i)) return;
  float g[kLaneGroups], u[kLaneGroups];
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) {
    const bool live = i + k * kGroup < c.n;
    g[k] = live ? to_float(gu[r * gu_ld + i + k * kGroup]) : 0.f;
    u[k] = live ? to_float(gu[r * gu_ld + c.n + i + k * kGroup]) : 0.f;
  }
  auto* cp = codes + 2 * r * c_ld + i;
  auto* sp = scales + 2 * r * s_ld + i / kGroup;
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) {
    int sg, su;
    const uint32_t cg = pack_lane(g[k], &sg), cu = pack_lane(u[k], &su);  // by all lanes
    if (i + k * kGroup < c.n) {
      z[r * z_ld + i + k * kGroup] = from_float<T>(silu_mul(g[k], u[k]));
      cp[k * kGroup] = (uint8_t)cg;
      cp[c_ld + k * kGroup] = (uint8_t)cu;
      if ((threadIdx.x & 31) == 0) {
        sp[k] = (uint8_t)sg;
        sp[s_ld + k] = (uint8_t)su;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    silu_mul_bwd_kernel(const Cut c, const T* dz, int64_t dz_ld, const uint8_t* codes, int64_t c_ld,
                        const uint8_t* scales, int64_t s_ld, T* dgu, int64_t dgu_ld, T* z, int64_t z_ld) {
  int64_t r, i;
  if (!span_of(c, &r, &i)) return;
  auto* cp = codes + 2 * r * c_ld + i;
  auto* sp = scales + 2 * r * s_ld + i / kGroup;
  float d[kLaneGroups], g[kLaneGroups], u[kLaneGroups];
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) {
    if (i + k * kGroup >= c.n) break;
    d[k] = to_float(dz[r * dz_ld + i + k * kGroup]);
    g[k] = unpack_one(cp[k * kGroup], sp[k]);
    u[k] = unpack_one(cp[c_ld + k * kGroup], sp[s_ld + k]);
  }
#pragma unroll
  for (int k = 0; k < kLaneGroups; ++k) {
    const int64_t at = i + k * kGroup;
    if (at >= c.n) break;
    const SwigluGrad q = swiglu_grad(d[k], g[k], u[k]);
    dgu[r * dgu_ld + at] = from_float<T>(q.dg);
    dgu[r * dgu_ld + c.n + at] = from_float<T>(q.du);
    if (z) z[r * z_ld + at] = from_float<T>(q.z);
  }
}

// Rows cut into halves of groups, one a thread, or into spans of kLaneGroups groups, one a warp.  False where a
// grid cannot hold them (beyond 2^31 CTAs: 2^41 values).
bool cut(int64_t rows, int64_t n, bool halves, Cut* c, unsigned* grid) {
  c->rows = rows;
  c->n = n;
  c->per_row = halves ? (n + kGroup - 1) / kGroup * 2 : (n + kSpan - 1) / kSpan;
  c->halves = rows * c->per_row;
  c->magic = c->per_row == 1 ? 0 : row_magic(rows, c->per_row);
  const int64_t each = halves ? kThreads : kWarps, blocks = (c->halves + each - 1) / each;
  *grid = (unsigned)blocks;
  return blocks <= 0x7fffffffLL;
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
  Cut c;
  unsigned grid = 0;
  bool fits = false;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(x);
    const bool halves = n % 16 == 0 && halves_ok<T>(x, x_ld);
    if (!(fits = cut(rows, n, halves, &c, &grid))) return;
    auto* kernel = halves ? pack16_kernel<T> : pack_kernel<T>;
    if (halves) grid = (grid + kPackEach - 1) / kPackEach;
    kernel<<<grid, kThreads, 0, s>>>(c, in, x_ld, codes, c_ld, scales, s_ld);
  });
  return fits ? launch_status() : GSA_ERR_BAD_ARG;
}

int gsa_unpack_e4m3(int dtype, int64_t rows, int64_t n, const uint8_t* codes, int64_t c_ld, const uint8_t* scales,
                    int64_t s_ld, void* x, int64_t x_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!x || x_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Cut c;
  unsigned grid = 0;
  bool fits = false;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    T* out = static_cast<T*>(x);
    const bool halves = n % 16 == 0 && halves_ok<T>(x, x_ld);
    if (!(fits = cut(rows, n, halves, &c, &grid))) return;
    auto* kernel = halves ? unpack16_kernel<T> : unpack_kernel<T>;
    kernel<<<grid, kThreads, 0, s>>>(c, codes, c_ld, scales, s_ld, out, x_ld);
  });
  return fits ? launch_status() : GSA_ERR_BAD_ARG;
}

int gsa_silu_mul_pack(int dtype, int64_t rows, int64_t n, const void* gu, int64_t gu_ld, void* z, int64_t z_ld,
                      uint8_t* codes, int64_t c_ld, uint8_t* scales, int64_t s_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!gu || gu_ld < 0 || !z || z_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Cut c;
  unsigned grid = 0;
  bool fits = false;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(gu);
    T* out = static_cast<T*>(z);
    const bool halves = n % 16 == 0 && halves_ok<T>(gu, gu_ld) && halves_ok<T>(z, z_ld);
    if (!(fits = cut(rows, n, halves, &c, &grid))) return;
    auto* kernel = halves ? silu_mul_pack16_kernel<T> : silu_mul_pack_kernel<T>;
    kernel<<<grid, kThreads, 0, s>>>(c, in, gu_ld, out, z_ld, codes, c_ld, scales, s_ld);
  });
  return fits ? launch_status() : GSA_ERR_BAD_ARG;
}

int gsa_silu_mul_packed_backward(int dtype, int64_t rows, int64_t n, const void* dz, int64_t dz_ld,
                                 const uint8_t* codes, int64_t c_ld, const uint8_t* scales, int64_t s_ld, void* dgu,
                                 int64_t dgu_ld, void* z, int64_t z_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!dz || dz_ld < 0 || !dgu || dgu_ld < 2 * n || (z && z_ld < n) || !packed_ok(codes, c_ld, scales, s_ld, n))
    return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Cut c;
  unsigned grid = 0;
  bool fits = false;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(dz);
    T *out = static_cast<T*>(dgu), *again = static_cast<T*>(z);
    const bool halves = n % 16 == 0 && halves_ok<T>(dz, dz_ld) && halves_ok<T>(dgu, dgu_ld) &&
                        (!z || halves_ok<T>(z, z_ld));
    if (!(fits = cut(rows, n, halves, &c, &grid))) return;
    auto* kernel = halves ? silu_mul_bwd16_kernel<T> : silu_mul_bwd_kernel<T>;
    kernel<<<grid, kThreads, 0, s>>>(c, in, dz_ld, codes, c_ld, scales, s_ld, out, dgu_ld, again, z_ld);
  });
  return fits ? launch_status() : GSA_ERR_BAD_ARG;
}

}  // extern "C"
