// The 8-bit form that activations are kept in for the backward pass: e4m3 values with one power-of-two scale
// for each group of 32 along the last dimension.
//
//   scale byte s stands for 2^(s - 127): the least power of two (s >= 0) with max|x| <= 448 * 2^(s - 127)
//   code = e4m3(x * 2^(127 - s)), to nearest even;  value = code * 2^(s - 127)
//
// Scaling by a power of two is exact, so a value is rounded once, to 4 significant bits (fewer below 2^-14 of
// its group's largest).  The scale goes by the finite values of the group; a NaN or an infinity becomes NaN.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "kernels.cuh"

namespace gsa {

constexpr int kGroup = 32;

// Scale byte of a group from the bits of its largest finite |x| (fp32).  448 = 1.75 * 2^8: the byte is the
// exponent field less 8, one more where the significand is above 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  const int s = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return max(s, 0);
}
__device__ __forceinline__ float pow2_of(int s) {  // 2^(s - 127); s = 0 is below the normal range
  return __int_as_float(s ? s << 23 : 0x00400000);
}
__device__ __forceinline__ float inv_pow2_of(int s) { return __int_as_float((254 - s) << 23); }  // s <= 247

// Two values to two e4m3 codes (x0 in the low byte).  The conversion saturates infinities, which have no
// code: they go in as NaN.
__device__ __forceinline__ uint16_t to_e4m3x2(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a >= 0x7f800000u ? 0u : a;
}
__device__ __forceinline__ float inf_to_nan(float x) { return isinf(x) ? __int_as_float(0x7fc00000) : x; }

// One value a lane: a warp's 32 are a group.  Returns the code (in the low byte).
__device__ __forceinline__ uint32_t pack_lane(float x, int* scale) {
  const int s = scale_byte(__reduce_max_sync(0xffffffffu, finite_abs_bits(x)));
  *scale = s;
  return to_e4m3x2(inf_to_nan(x) * inv_pow2_of(s), 0.f) & 0xffu;
}
__device__ __forceinline__ float unpack_one(uint8_t code, uint8_t scale) {
  return from_e4m3x2(code).x * pow2_of(scale);
}

// ---------------------------------------------------------------------------------------------
// 16 values a thread: half a group.  Their loads and stores are 32-byte ones (a whole sector a thread), kept out
// of L1, where nothing reads them twice.
// ---------------------------------------------------------------------------------------------
struct Words8 {
  uint32_t w[8];
};
__device__ __forceinline__ Words8 load32(const void* p) {
  Words8 r;
  asm("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
      : "l"(p));
  return r;
}
// The same through L1, for what neighbouring CTAs read again.
__device__ __forceinline__ Words8 load32_shared(const void* p) {
  Words8 r;
  asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
      : "l"(p));
  return r;
}
__device__ __forceinline__ void store32(void* p, const Words8& r) {
  asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]),
               "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
               : "memory");
}

// 16 values in their type, and their conversions.
template <typename T>
struct Half;
template <>
struct Half<__nv_bfloat16> {
  Words8 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = load32(p); }
  __device__ __forceinline__ void load_shared(const __nv_bfloat16* p) { a = load32_shared(p); }
  __device__ __forceinline__ void zero() { a = Words8{}; }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = __uint_as_float(a.w[i] << 16);
      v[2 * i + 1] = __uint_as_float(a.w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      a.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { store32(p, a); }
};
template <>
struct Half<float> {
  Words8 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = load32(p);
    b = load32(p + 8);
  }
  __device__ __forceinline__ void load_shared(const float* p) {
    a = load32_shared(p);
    b = load32_shared(p + 8);
  }
  __device__ __forceinline__ void zero() { a = b = Words8{}; }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = __uint_as_float(a.w[i]);
      v[8 + i] = __uint_as_float(b.w[i]);
    }
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a.w[i] = __float_as_uint(v[i]);
      b.w[i] = __float_as_uint(v[8 + i]);
    }
  }
  __device__ __forceinline__ void store(float* p) const {
    store32(p, a);
    store32(p + 8, b);
  }
};

// ---------------------------------------------------------------------------------------------
// Rows that are not whole multiples of 16 values, or not aligned to 32 bytes ("ragged"): a thread still holds 16
// neighbouring ones.  It reads the aligned 16-byte pieces that they lie in and writes aligned pieces, of which two
// neighbouring lanes share one: the right one puts it together.  Which register holds which value goes by the
// row's offset, one of a few cases with code of its own, so that taking a value costs no shift beside its
// conversion.  Only pieces at a row's ends and at a warp's go word by word.
// ---------------------------------------------------------------------------------------------

// Calls f with one of eight offsets, 0 to 7, at compile time.
template <typename F>
__device__ __forceinline__ void by_offset(int offset, F f) {
  switch (offset) {
    case 0: f(std::integral_constant<int, 0>()); break;
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 5: f(std::integral_constant<int, 5>()); break;
    case 6: f(std::integral_constant<int, 6>()); break;
    default: f(std::integral_constant<int, 7>());
  }
}

// The values of a row that a thread holds (0 to 16), and whether the lanes beside it hold their neighbours.
struct Spot {
  int live;
  bool left, right;
};
template <bool kRagged>
__device__ __forceinline__ Spot spot_of(int64_t i, int64_t n, bool row) {
  row = row && i < n;
  if (!kRagged) return {row ? 16 : 0, false, false};
  const int lane = threadIdx.x & 31;
  return {row ? (int)min((int64_t)16, n - i) : 0, row && i > 0 && lane > 0, row && i + 16 < n && lane < 31};
}

// The bytes of a tensor: pieces that reach out of it are read value by value.
struct Extent {
  const char *lo, *hi;
};
template <typename T>
__device__ __forceinline__ Extent extent_of(const T* x, int64_t rows, int64_t ld, int64_t n) {
  return {reinterpret_cast<const char*>(x), reinterpret_cast<const char*>(x + (rows - 1) * ld + n)};
}

// 16 values as they are read, and their conversion.  Whole rows are loaded where the spot is live, several tensors under one
// condition; ragged ones see to that themselves (measured: the other way round each is 5-10% slower).
template <typename T, bool kRagged>
struct HalfIn {
  Half<T> h;
  __device__ __forceinline__ void zero() { h.zero(); }
  template <bool kShared = false>
  __device__ __forceinline__ void load(const T* p, const Spot& at, const Extent&) {
    if (kShared)
      h.load_shared(p);
    else
      h.load(p);
  }
  __device__ __forceinline__ void get(float* v, const Spot&) const { h.get(v); }
};
template <typename T>
struct HalfIn<T, true> {
  static constexpr int kSize = (int)sizeof(T), kPieces = kSize + 1;
  uint32_t w[4 * kPieces];
  int offset;  // of the first value in w, in bytes
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 4 * kPieces; ++i) w[i] = 0;
    offset = 0;
  }
  __device__ __forceinline__ void piece(int j, const char* q) {
    const uint4 t = __ldg(reinterpret_cast<const uint4*>(q) + j);
    w[4 * j] = t.x;
    w[4 * j + 1] = t.y;
    w[4 * j + 2] = t.z;
    w[4 * j + 3] = t.w;
  }
  template <bool kShared = false>
  __device__ __forceinline__ void load(const T* p, const Spot& at, const Extent& in) {
    zero();
    if (!at.live) return;
    offset = (int)(reinterpret_cast<uintptr_t>(p) & 15);
    const char* q = reinterpret_cast<const char*>(p) - offset;
    if (q >= in.lo && q + 16 * kPieces <= in.hi) {
#pragma unroll
      for (int j = 0; j < kPieces - 1; ++j) piece(j, q);
      if (offset) piece(kPieces - 1, q);
      return;
    }
#pragma unroll
    for (int b = 0; b < 16 * kPieces; b += kSize) {
      if (b < offset || b >= offset + at.live * kSize) continue;
      if (kSize == 2)
        w[b / 4] |= (uint32_t)*reinterpret_cast<const uint16_t*>(q + b) << (b % 4 * 8);
      else
        w[b / 4] = *reinterpret_cast<const uint32_t*>(q + b);
    }
  }
  __device__ __forceinline__ void get(float* v, const Spot& at) const {
    if (kSize == 2) {
      by_offset(offset / 2, [&](auto o) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int b = 2 * (decltype(o)::value + k);
          v[k] = __uint_as_float(b % 4 ? w[b / 4] & 0xffff0000u : w[b / 4] << 16);
        }
      });
    } else {
      uint32_t t[18];
#pragma unroll
      for (int i = 0; i < 18; ++i) t[i] = offset & 8 ? w[(i + 2) % (4 * kPieces)] : w[i % (4 * kPieces)];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(offset & 4 ? t[i + 1] : t[i]);
    }
    if (at.live < 16)
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k >= at.live) v[k] = 0.f;
  }
};

// 16 values as whole words from the start of the piece that they begin in, offset bytes before them; zeros around them.
__device__ __forceinline__ void lay_out(const __nv_bfloat16*, const float* v, int offset, uint32_t* t) {
  by_offset(offset / 2, [&](auto o) {
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      const int k = 2 * i - decltype(o)::value;  // the low value's
      const __nv_bfloat162 h = __floats2bfloat162_rn(k >= 0 && k < 16 ? v[k & 15] : 0.f,
                                                     k >= -1 && k < 15 ? v[(k + 1) & 15] : 0.f);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  });
}
__device__ __forceinline__ void lay_out(const float*, const float* v, int offset, uint32_t* t) {
  by_offset(offset / 4, [&](auto o) {
#pragma unroll
    for (int i = 0; i < 24; ++i) {
      const int k = i - decltype(o)::value;
      t[i] = k >= 0 && k < 16 ? __float_as_uint(v[k & 15]) : 0u;
    }
  });
}
__device__ __forceinline__ void store_piece(char* p, const uint32_t (&w)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_piece(char* p, const uint32_t (&w)[8]) {
  store32(p, Words8{{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]}});
}

// Stores a thread's 16 values at p; ragged ones by every lane of the warp together, in pieces of eight values: fp32 ones
// are whole sectors, which bf16's 16 bytes are not (but with sectors the registers' turns cost more: 85 us against 98 for
// 32768 x 4090 unpacked; for fp32 it is 77 against 58).
template <bool kRagged, typename T>
__device__ __forceinline__ void put_values(T* p, const float* v, const Spot& at) {
  if (!kRagged) {
    if (!at.live) return;
    Half<T> h;
    h.set(v);
    h.store(p);
    return;
  }
  constexpr int kSize = (int)sizeof(T), kShift = kSize / 2, kBytes = 8 * kSize, kWords = kBytes / 4;
  const int offset = (int)(reinterpret_cast<uintptr_t>(p) & (kBytes - 1));
  uint32_t t[3 * kWords];
  lay_out(p, v, offset, t);
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const uint32_t before = __shfl_up_sync(0xffffffffu, t[2 * kWords + i], 1);
    if (at.left) t[i] |= before;
  }
  char* q = reinterpret_cast<char*>(p) - offset;
  const int b0 = at.left ? 0 : offset, b1 = at.right ? 2 * kBytes : offset + at.live * kSize;  // this lane's bytes
  int parts = 0;  // pieces of which this lane has a part
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = t[kWords * j + i];
    if (b0 <= kBytes * j && b1 >= kBytes * (j + 1))
      store_piece(q + kBytes * j, w);
    else if (b0 < kBytes * (j + 1) && b1 > kBytes * j && b1 > b0)
      parts |= 1 << j;
  }
  while (parts) {
    const int j = __ffs(parts) - 1;
    parts &= parts - 1;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = t[i];
#pragma unroll
      for (int m = 1; m < 3; ++m) w[i] = j == m ? t[kWords * m + i] : w[i];
    }
    const int lo = max(b0 - kBytes * j, 0) >> kShift, hi = min(b1 - kBytes * j, kBytes) >> kShift;
    const uint32_t mine = (1u << hi) - (1u << lo);
    char* to = q + kBytes * j;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (!(mine >> k & 1u)) continue;
      if (kSize == 2)
        reinterpret_cast<uint16_t*>(to)[k] = (uint16_t)(w[k / 2] >> (k % 2 * 16));
      else
        reinterpret_cast<uint32_t*>(to)[k] = w[k % kWords];
    }
  }
}

// A group held by two neighbouring lanes (every lane of the warp calls this): the scale byte, and this lane's 16
// codes.  Lanes without values pass zeros.
__device__ __forceinline__ int pack_half(float* v, uint4* codes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  if (m >= 0x7f800000u) {  // rare: the scale goes by the finite values, infinities convert as NaN
    m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      m = max(m, finite_abs_bits(v[i]));
      v[i] = inf_to_nan(v[i]);
    }
  }
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const int s = scale_byte(m);
  const float f = inv_pow2_of(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = to_e4m3x2(v[4 * i] * f, v[4 * i + 1] * f) |
           (uint32_t)to_e4m3x2(v[4 * i + 2] * f, v[4 * i + 3] * f) << 16;
  *codes = make_uint4(w[0], w[1], w[2], w[3]);
  return s;
}

__device__ __forceinline__ void unpack_half(const uint4& codes, float scale, float* v) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = from_e4m3x2((uint16_t)w[i]), hi = from_e4m3x2((uint16_t)(w[i] >> 16));
    v[4 * i] = lo.x * scale;
    v[4 * i + 1] = lo.y * scale;
    v[4 * i + 2] = hi.x * scale;
    v[4 * i + 3] = hi.y * scale;
  }
}

__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
  uint4 r;
  asm("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
      : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
      : "l"(p));
  return r;
}
// The same for a spot as HalfIn loads it; the codes behind a ragged row's end as zeros, whatever the buffer holds there.
template <bool kRagged>
__device__ __forceinline__ uint4 load_codes(const uint8_t* p, const Spot& at) {
  if (kRagged && !at.live) return make_uint4(0, 0, 0, 0);
  uint4 r = load_codes(p);
  if (kRagged && at.live < 16) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = min(max(at.live - 4 * i, 0), 4);
      w[i] = k == 4 ? w[i] : w[i] & ((1u << (8 * k)) - 1u);
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}
__device__ __forceinline__ void store_codes(uint8_t* p, const uint4& c) {
  asm volatile("st.global.L1::no_allocate.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(c.x), "r"(c.y), "r"(c.z),
               "r"(c.w)
               : "memory");
}

// floor(n / d) for n d < 2^64, d > 1, with m = ceil(2^64 / d); d = 1 (a single row) is passed as m = 0 and gives 0
// for n < d of the one row.
__device__ __forceinline__ int64_t row_of(int64_t n, uint64_t m) { return (int64_t)__umul64hi((uint64_t)n, m); }
inline uint64_t row_magic(int64_t rows, int64_t d) { return rows == 1 ? 0 : ~0ull / (uint64_t)d + 1; }

inline bool type_ok(int dtype) { return dtype == GSA_DTYPE_F32 || dtype == GSA_DTYPE_BF16; }

// Packed rows of n values: whole 16-byte pieces of codes, a scale byte for each group.
inline bool packed_ok(const uint8_t* codes, int64_t c_ld, const uint8_t* scales, int64_t s_ld, int64_t n) {
  return codes && scales && c_ld >= (n + 15) / 16 * 16 && c_ld % 16 == 0 &&
         reinterpret_cast<uintptr_t>(codes) % 16 == 0 && s_ld >= (n + kGroup - 1) / kGroup;
}

// Calls f with a value of the element type.
template <typename F>
inline void typed(int dtype, F f) {
  if (dtype == GSA_DTYPE_BF16)
    f(__nv_bfloat16());
  else
    f(float());
}

inline int launch_status() { return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH; }

// Whether rows of a tensor can be read or written 16 values at a time.
template <typename T>
inline bool halves_ok(const void* p, int64_t ld) {
  return reinterpret_cast<uintptr_t>(p) % 32 == 0 && ld % 16 == 0;
}
template <>
inline bool halves_ok<float>(const void* p, int64_t ld) {
  return reinterpret_cast<uintptr_t>(p) % 32 == 0 && ld % 8 == 0;
}

}  // namespace gsa
