// Activations kept in 8 bits for the backward pass (the form: packed.cuh), and the SwiGLU product that keeps its
// operands so.
//
//   pack / unpack   x -> codes, scales -> x^
//   silu_mul        z = g sigma(g) u, (g, u) kept packed; backward, from the packed g^, u^:
//                   dg = dz u^ sigma (1 + g^ (1 - sigma)), du = dz g^ sigma, z again for the weight gradient of the
//                   product that reads it
//
// Products are in 32 bits; an output is rounded once, to its type.  All are bound by the bytes that they move, so
// a thread holds 16 neighbouring values (half a group, 32-byte loads and stores, one shuffle for the scale); where rows are
// not whole multiples of that, or not aligned, through aligned pieces (kRagged: packed.cuh).  Whole rows run at HBM's rate (of
// 6.55 TB/s for a copy): pack and unpack of 32768 x 4096 bf16 128 us, 6.4 TB/s; SwiGLU and its backward pass of 16384 x
// 11008 0.50 ms, 6.5 TB/s.  Ragged ones are bound by instructions: 32768 x 4090 bf16 155 us (5.2 TB/s) and 0.55 ms (4.4); fp32
// 16384 x 4090 124 us and 0.35 ms (5.4, 6.2).
#include <algorithm>

#include "packed.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// sigma(x) = s k with k a power of two, s = 1 / ((1 + e^-x) k): k = 1/4 keeps the reciprocal in the normal range as long as e^-x
// is in it.  Beyond (x < -87.3, where the 1 no longer counts) it is e^-x 2^-96 of which the reciprocal is taken, so that
// x sigma(x), formed as (k x) s, has its relative accuracy down to the smallest normal number (x = -91.8; a plain fast
// reciprocal gives 0 from -87.3 on).  e^-x is 2^t times 2^lo with t = -x log2 e rounded and lo what that lost; beyond +-1e4 it is 0
// or infinite in any case.
struct Sigmoid {
  float s, k;
};
__device__ __forceinline__ Sigmoid sigmoid_of(float x) {
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.925963e-8f, kLn2 = 0.693147181f;  // log2 e as a sum of two
  const float c = fminf(fmaxf(x, -1e4f), 1e4f);
  const float t = -c * kLog2e, lo = fmaf(-c, kLog2eLow, fmaf(-c, kLog2e, -t));
  const bool far = t > 126.f;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(far ? t - 96.f : t));
  e *= fmaf(lo, kLn2, 1.0f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0.25f, 0.25f)));
  return {r, far ? 0x1p-98f : 0.25f};
}
__device__ __forceinline__ float silu_mul(float g, float u) {
  const Sigmoid q = sigmoid_of(g);
  return q.k * g * q.s * u;
}

struct SwigluGrad {
  float dg, du, z;
};
__device__ __forceinline__ SwigluGrad swiglu_grad(float dz, float g, float u) {
  const Sigmoid q = sigmoid_of(g);
  const float sig = q.k * q.s, silu = q.k * g * q.s;
  // sig may be under the normal range, where silu carries the sum
  return {dz * u * fmaf(silu, 1.0f - sig, sig), dz * silu, silu * u};
}

// A row is cut into 2 ceil(n / 32) halves of 16 values, one a thread, so that the two halves of a group are neighbouring
// lanes; the last may be empty.
struct Cut {
  int64_t rows, halves, per_row;  // halves: rows * per_row
  uint64_t magic;
  int64_t n;
};
struct Place {
  int64_t r, i;
  Spot at;
};
template <bool kRagged>
__device__ __forceinline__ Place place_of(const Cut& c, int skip = 0, int each = 1) {
  const int64_t e = (int64_t)blockIdx.x * each * kThreads + skip + threadIdx.x;
  const int64_t r = row_of(e, c.magic), i = (e - r * c.per_row) * 16;
  return {r, i, spot_of<kRagged>(i, c.n, e < c.halves)};
}

// Two halves a thread, both loaded first: one alone leaves too little in flight for HBM (69 us, 65 with two, for 32768 x
// 4096 bf16).
constexpr int kPackEach = 2;

template <typename T, bool kRagged>
__global__ void __launch_bounds__(kThreads) pack16_kernel(const Cut c, const T* x, int64_t x_ld, uint8_t* codes,
                                                          int64_t c_ld, uint8_t* scales, int64_t s_ld) {
  const Extent in = extent_of(x, c.rows, x_ld, c.n);
  Place p[kPackEach];
  HalfIn<T, kRagged> h[kPackEach];
#pragma unroll
  for (int j = 0; j < kPackEach; ++j) {
    p[j] = place_of<kRagged>(c, j * kThreads, kPackEach);
    h[j].zero();
    if (kRagged || p[j].at.live) h[j].load(x + p[j].r * x_ld + p[j].i, p[j].at, in);
  }
#pragma unroll
  for (int j = 0; j < kPackEach; ++j) {
    float v[16];
    h[j].get(v, p[j].at);
    uint4 q;
    const int s = pack_half(v, &q);
    if (p[j].at.live) {
      store_codes(codes + p[j].r * c_ld + p[j].i, q);
      if ((threadIdx.x & 1) == 0) scales[p[j].r * s_ld + p[j].i / kGroup] = (uint8_t)s;
    }
  }
}

template <typename T, bool kRagged>
__global__ void __launch_bounds__(kThreads) unpack16_kernel(const Cut c, const uint8_t* codes, int64_t c_ld,
                                                            const uint8_t* scales, int64_t s_ld, T* x, int64_t x_ld) {
  const Place p = place_of<kRagged>(c);
  if (!kRagged && !p.at.live) return;
  uint4 q = make_uint4(0, 0, 0, 0);
  float scale = 0.f;
  if (kRagged || p.at.live) {
    q = load_codes<kRagged>(codes + p.r * c_ld + p.i, p.at);
    if (p.at.live) scale = pow2_of(scales[p.r * s_ld + p.i / kGroup]);
  }
  float v[16];
  unpack_half(q, scale, v);
  put_values<kRagged>(x + p.r * x_ld + p.i, v, p.at);
}

// gu rows hold g then u; the packed rows 2r and 2r + 1 are row r's g and u.
template <typename T, bool kRagged>
__global__ void __launch_bounds__(kThreads, kRagged && sizeof(T) == 4 ? 3 : 4)
    silu_mul_pack16_kernel(const Cut c, const T* gu, int64_t gu_ld, T* z, int64_t z_ld, uint8_t* codes, int64_t c_ld,
                           uint8_t* scales, int64_t s_ld) {
  const Place p = place_of<kRagged>(c);
  const Extent in = extent_of(gu, c.rows, gu_ld, 2 * c.n);
  HalfIn<T, kRagged> hg, hu;
  hg.zero();
  hu.zero();
  if (kRagged || p.at.live) {
    hg.load(gu + p.r * gu_ld + p.i, p.at, in);
    hu.load(gu + p.r * gu_ld + c.n + p.i, p.at, in);
  }
  float g[16], u[16];
  hg.get(g, p.at);
  hu.get(u, p.at);
  if (kRagged || p.at.live) {
    float o[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = silu_mul(g[k], u[k]);
    put_values<kRagged>(z + p.r * z_ld + p.i, o, p.at);
  }
  uint4 qg, qu;
  const int sg = pack_half(g, &qg), su = pack_half(u, &qu);
  if (!p.at.live) return;
  store_codes(codes + 2 * p.r * c_ld + p.i, qg);
  store_codes(codes + (2 * p.r + 1) * c_ld + p.i, qu);
  if ((threadIdx.x & 1) == 0) {
    scales[2 * p.r * s_ld + p.i / kGroup] = (uint8_t)sg;
    scales[(2 * p.r + 1) * s_ld + p.i / kGroup] = (uint8_t)su;
  }
}

template <typename T, bool kRagged>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && !kRagged ? 4 : 3)
    silu_mul_bwd16_kernel(const Cut c, const T* dz, int64_t dz_ld, const uint8_t* codes, int64_t c_ld,
                          const uint8_t* scales, int64_t s_ld, T* dgu, int64_t dgu_ld, T* z, int64_t z_ld) {
  const Place p = place_of<kRagged>(c);
  if (!kRagged && !p.at.live) return;
  const int64_t r2 = 2 * p.r, k0 = p.i / kGroup;
  HalfIn<T, kRagged> hd;
  uint4 qg = make_uint4(0, 0, 0, 0), qu = qg;
  float sg = 0.f, su = 0.f;
  hd.zero();
  if (p.at.live) {
    hd.load(dz + p.r * dz_ld + p.i, p.at, extent_of(dz, c.rows, dz_ld, c.n));
    qg = load_codes<kRagged>(codes + r2 * c_ld + p.i, p.at);
    qu = load_codes<kRagged>(codes + (r2 + 1) * c_ld + p.i, p.at);
    sg = pow2_of(scales[r2 * s_ld + k0]);
    su = pow2_of(scales[(r2 + 1) * s_ld + k0]);
  }
  float d[16], g[16], u[16];
  unpack_half(qg, sg, g);
  unpack_half(qu, su, u);
  hd.get(d, p.at);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const SwigluGrad s = swiglu_grad(d[k], g[k], u[k]);
    d[k] = s.dg;
    g[k] = s.du;
    u[k] = s.z;
  }
  put_values<kRagged>(dgu + p.r * dgu_ld + p.i, d, p.at);
  put_values<kRagged>(dgu + p.r * dgu_ld + c.n + p.i, g, p.at);
  if (z) put_values<kRagged>(z + p.r * z_ld + p.i, u, p.at);
}

// False where a grid cannot hold the halves (beyond 2^31 CTAs: 2^43 values).
bool cut(int64_t rows, int64_t n, Cut* c, unsigned* grid) {
  c->rows = rows;
  c->n = n;
  c->per_row = (n + kGroup - 1) / kGroup * 2;
  c->halves = rows * c->per_row;
  c->magic = row_magic(rows, c->per_row);
  const int64_t blocks = (c->halves + kThreads - 1) / kThreads;
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
  if (!cut(rows, n, &c, &grid)) return GSA_ERR_BAD_ARG;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(x);
    const bool whole = n % 16 == 0 && halves_ok<T>(x, x_ld);
    auto* kernel = whole ? pack16_kernel<T, false> : pack16_kernel<T, true>;
    kernel<<<(grid + kPackEach - 1) / kPackEach, kThreads, 0, s>>>(c, in, x_ld, codes, c_ld, scales, s_ld);
  });
  return launch_status();
}

int gsa_unpack_e4m3(int dtype, int64_t rows, int64_t n, const uint8_t* codes, int64_t c_ld, const uint8_t* scales,
                    int64_t s_ld, void* x, int64_t x_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!x || x_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Cut c;
  unsigned grid = 0;
  if (!cut(rows, n, &c, &grid)) return GSA_ERR_BAD_ARG;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    T* out = static_cast<T*>(x);
    const bool whole = n % 16 == 0 && halves_ok<T>(x, x_ld);
    auto* kernel = whole ? unpack16_kernel<T, false> : unpack16_kernel<T, true>;
    kernel<<<grid, kThreads, 0, s>>>(c, codes, c_ld, scales, s_ld, out, x_ld);
  });
  return launch_status();
}

int gsa_silu_mul_pack(int dtype, int64_t rows, int64_t n, const void* gu, int64_t gu_ld, void* z, int64_t z_ld,
                      uint8_t* codes, int64_t c_ld, uint8_t* scales, int64_t s_ld, gsa_stream_t stream) {
  if (!type_ok(dtype) || rows < 0 || n < 0) return GSA_ERR_BAD_ARG;
  if (rows == 0 || n == 0) return GSA_OK;
  if (!gu || gu_ld < 0 || !z || z_ld < n || !packed_ok(codes, c_ld, scales, s_ld, n)) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Cut c;
  unsigned grid = 0;
  if (!cut(rows, n, &c, &grid)) return GSA_ERR_BAD_ARG;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(gu);
    T* out = static_cast<T*>(z);
    const bool whole = n % 16 == 0 && halves_ok<T>(gu, gu_ld) && halves_ok<T>(z, z_ld);
    auto* kernel = whole ? silu_mul_pack16_kernel<T, false> : silu_mul_pack16_kernel<T, true>;
    kernel<<<grid, kThreads, 0, s>>>(c, in, gu_ld, out, z_ld, codes, c_ld, scales, s_ld);
  });
  return launch_status();
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
  if (!cut(rows, n, &c, &grid)) return GSA_ERR_BAD_ARG;
  typed(dtype, [&](auto e) {
    using T = decltype(e);
    const T* in = static_cast<const T*>(dz);
    T *out = static_cast<T*>(dgu), *again = static_cast<T*>(z);
    const bool whole = n % 16 == 0 && halves_ok<T>(dz, dz_ld) && halves_ok<T>(dgu, dgu_ld) &&
                       (!z || halves_ok<T>(z, z_ld));
    auto* kernel = whole ? silu_mul_bwd16_kernel<T, false> : silu_mul_bwd16_kernel<T, true>;
    kernel<<<grid, kThreads, 0, s>>>(c, in, dz_ld, codes, c_ld, scales, s_ld, out, dgu_ld, again, z_ld);
  });
  return launch_status();
}

}  // extern "C"
