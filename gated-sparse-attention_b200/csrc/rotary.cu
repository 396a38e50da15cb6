// Rotary positions on q and k: y = R(p) x on the first rd values of every head, the rest passed through.
//
//   angle_i = p f_i,  c_i = m cos(angle_i),  s_i = m sin(angle_i)   (m: the attention factor)
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s;  backward (the transpose): s -> -s
//   half pairs: (x_i, x_{i + rd/2});  interleaved pairs: (x_{2i}, x_{2i+1})
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there, so that far positions keep their
// angle (p f of 2^20 radians in 32 bits is off by 2^-4); sine and cosine of the fraction are 32-bit.  A CTA takes
// a few tokens, evaluates each token's rd/2 angles once into shared memory (all its heads share them) and
// then streams the tokens' heads.  Bound by the bytes of q and k, read once and written once: 131,072 tokens of 40 heads
// of 128 in bf16 take 0.396 ms, 6.8 TB/s.
//
// A thread owns one place of a token -- a head and V neighbouring pairs of it (or 2 V pass-through values) -- and
// walks the CTA's tokens with it, four in flight, so the place is worked out once.  V values are one
// load: 16 bytes where rd, D, the strides and the addresses are multiples of that, else 4 values, 2 or 1.
#include <algorithm>

#include "kernels.cuh"

namespace gsa {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxTokens = 64;
constexpr int kFlight = 4;        // tokens whose loads are in flight
constexpr int kMaxAngles = 4096;  // (token, pair) entries of the shared table: 32 KB

struct Side {  // q or k: strides in elements
  const void* in;
  void* out;
  int heads;
  int64_t ib, il, ih, ob, ol, oh;
};

struct RotaryArgs {
  Side q, k;
  int64_t B, L;
  int D, rd;
  const int64_t* pos;
  int64_t pb, pl;
  const double* freq;  // [rd/2], or NULL: the tables
  const void* cos_tab;
  const void* sin_tab;
  int tab_dtype;
  int64_t tab_ld, tab_rows;
  float factor;
  int inverse;
  int tokens;  // per CTA
  int beside;  // tokens that the CTA's threads take at a time
  int items;   // places of a token
  int turn_units, units;  // of a head: units that turn, all
  int* err;
};

// (c, s) of one token's pair i.
__device__ __forceinline__ float2 angle_of(const RotaryArgs& a, int64_t p, int i) {
  float c, s;
  if (a.freq) {
    constexpr double kInvTwoPi = 0.15915494309189533577;
    const double turns = (double)p * a.freq[i] * kInvTwoPi;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  } else if (p < 0 || p >= a.tab_rows) {
    set_error(a.err, GSA_ERR_INDEX);
    c = s = __int_as_float(0x7fc00000);
  } else {
    c = load_elem(a.cos_tab, p * a.tab_ld + i, a.tab_dtype);
    s = load_elem(a.sin_tab, p * a.tab_ld + i, a.tab_dtype);
  }
  c *= a.factor;
  s *= a.factor;
  return make_float2(c, a.inverse ? -s : s);
}

// One value of a pair: each product and the sum rounded by itself (no contraction), as torch evaluates it.
__device__ __forceinline__ float turn0(float x0, float x1, float2 cs) { return fadd(fmul(x0, cs.x), -fmul(x1, cs.y)); }
__device__ __forceinline__ float turn1(float x0, float x1, float2 cs) { return fadd(fmul(x1, cs.x), fmul(x0, cs.y)); }

// V values as one load or store.
template <int kBytes>
struct Raw;
template <>
struct Raw<16> {
  using type = uint4;
};
template <>
struct Raw<8> {
  using type = uint2;
};
template <>
struct Raw<4> {
  using type = uint32_t;
};
template <>
struct Raw<2> {
  using type = uint16_t;
};
template <typename T, int V>
union Vec {
  typename Raw<sizeof(T) * V>::type raw;
  T v[V];
  __device__ __forceinline__ Vec() : raw{} {}
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const decltype(raw)*>(p)); }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<decltype(raw)*>(p), raw); }
};

// One place of a token: where its two vectors are, relative to the token's head 0.
struct Place {
  int64_t in, out;  // of the head
  int i0, i1;       // the vectors' first values; i1 < 0: the second is not there
  int unit;         // among those that turn; < 0: passes through
  bool is_k;
};

template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ Place place_of(const RotaryArgs& a, int item) {
  const int h = item / a.units, u = item - h * a.units, half = a.rd / 2;
  Place p;
  p.is_k = h >= a.q.heads;
  const Side& s = p.is_k ? a.k : a.q;
  const int hh = p.is_k ? h - a.q.heads : h;
  p.in = hh * s.ih;
  p.out = hh * s.oh;
  if (u < a.turn_units) {
    p.i0 = kInterleaved ? 2 * u * V : u * V;
    p.i1 = kInterleaved ? p.i0 + V : p.i0 + half;
    p.unit = u;
  } else {
    p.i0 = a.rd + (u - a.turn_units) * 2 * V;
    p.i1 = p.i0 + V < a.D ? p.i0 + V : -1;
    p.unit = -1;
  }
  return p;
}

// Where angle i of a token is among its rd/2: with vectors of 4 or 8, two of a unit's side by side and then the next
// unit's, so that neighbouring threads' 16-byte loads are next to each other (a unit's V in a row are on the same
// banks as its neighbours': 429 us against 396 for 131,072 tokens of 40 heads, 130 against 105 for 122,189 of 10).
template <int V>
__device__ __forceinline__ int slot_of(int i, int units) {
  return V <= 2 ? i : i % V / 2 * 2 * units + i / V * 2 + i % 2;
}
template <int V>
__device__ __forceinline__ void angles_of(const float2* token, int unit, int units, float2* cs) {
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    const float4 c = reinterpret_cast<const float4*>(token)[j * units + unit];
    cs[2 * j] = make_float2(c.x, c.y);
    cs[2 * j + 1] = make_float2(c.z, c.w);
  }
}

// x0, x1: the unit's two vectors, turned in place.  cs: the unit's V angles.
template <typename T, int V, bool kInterleaved>
__device__ __forceinline__ void turn(Vec<T, V>& x0, Vec<T, V>& x1, const float2* cs) {
  if (kInterleaved) {
    // values 2j, 2j + 1 of the 2 V are pair j
    T w[2 * V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[j] = x0.v[j];
      w[V + j] = x1.v[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 c = cs[j];
      const float a = to_float(w[2 * j]), b = to_float(w[2 * j + 1]);
      w[2 * j] = from_float<T>(turn0(a, b, c));
      w[2 * j + 1] = from_float<T>(turn1(a, b, c));
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x0.v[j] = w[j];
      x1.v[j] = w[V + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 c = cs[j];
      const float a = to_float(x0.v[j]), b = to_float(x1.v[j]);
      x0.v[j] = from_float<T>(turn0(a, b, c));
      x1.v[j] = from_float<T>(turn1(a, b, c));
    }
  }
}

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kMaxThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ __align__(16) float2 angles[];
  __shared__ int64_t base[kMaxTokens][4];  // element offsets of the token: q in, q out, k in, k out
  __shared__ int64_t at_pos[kMaxTokens];
  const int half = a.rd / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n_tok = (int)min((int64_t)a.tokens, a.B * a.L - t0);
  for (int tok = threadIdx.x; tok < n_tok; tok += blockDim.x) {
    const int64_t t = t0 + tok, b = t / a.L, l = t - b * a.L;
    at_pos[tok] = a.pos[b * a.pb + l * a.pl];
    base[tok][0] = b * a.q.ib + l * a.q.il;
    base[tok][1] = b * a.q.ob + l * a.q.ol;
    base[tok][2] = b * a.k.ib + l * a.k.il;
    base[tok][3] = b * a.k.ob + l * a.k.ol;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_tok * half; e += blockDim.x) {
    const int tok = e / half;
    angles[tok * half + slot_of<V>(e - tok * half, a.turn_units)] = angle_of(a, at_pos[tok], e - tok * half);
  }
  __syncthreads();
  // one token at a time: its places over all threads, in rounds; more: a place of one of them each
  const int tok1 = a.beside == 1 ? 0 : threadIdx.x / a.items;
  const int item1 = a.beside == 1 ? threadIdx.x : threadIdx.x - tok1 * a.items;
  if (tok1 >= a.beside) return;
  for (int item = item1; item < a.items; item += a.beside == 1 ? blockDim.x : a.items) {
    const Place p = place_of<T, V, kInterleaved>(a, item);
    const Side& s = p.is_k ? a.k : a.q;
    const T* in = static_cast<const T*>(s.in) + p.in;
    T* out = static_cast<T*>(s.out) + p.out;
    const int64_t* at = &base[0][p.is_k ? 2 : 0];
    if (p.unit < 0 && in == out) continue;  // rotated in place: the rest is where it belongs
    // four tokens' loads before the first store, which may be to the same tensor
    for (int tok0 = tok1; tok0 < n_tok; tok0 += kFlight * a.beside) {
      Vec<T, V> x0[kFlight], x1[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int tok = tok0 + j * a.beside;
        if (tok >= n_tok) break;
        const T* x = in + at[4 * tok];
        x0[j].load(x + p.i0);
        if (p.i1 >= 0) x1[j].load(x + p.i1);
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int tok = tok0 + j * a.beside;
        if (tok >= n_tok) break;
        T* y = out + at[4 * tok + 1];
        if (V <= 2) {
          if (p.unit >= 0) turn<T, V, kInterleaved>(x0[j], x1[j], &angles[tok * half + p.unit * V]);
        } else if (p.unit >= 0) {
          float2 cs[V];
          angles_of<V>(angles + tok * half, p.unit, a.turn_units, cs);
          turn<T, V, kInterleaved>(x0[j], x1[j], cs);
        }
        x0[j].store(y + p.i0);
        if (p.i1 >= 0) x1[j].store(y + p.i1);
      }
    }
  }
}

bool side_ok(const gsa_rotary_side* s, int64_t D) {
  return s->in && s->out && s->heads > 0 && s->in_h >= 0 && s->in_l >= 0 && s->in_b >= 0 &&
         (s->heads == 1 || s->out_h >= D) && s->out_l >= 0 && s->out_b >= 0;
}

Side side_of(const gsa_rotary_side* s) {
  if (!s) return Side{};
  return Side{s->in, s->out, s->heads, s->in_b, s->in_l, s->in_h, s->out_b, s->out_l, s->out_h};
}

bool vec_ok(const Side& s, int64_t V, int64_t esz) {
  const int64_t all = s.ib | s.il | s.ih | s.ob | s.ol | s.oh;
  return all % V == 0 && (reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) % (V * esz) == 0;
}

// Whether vectors of V values tile the heads: whole vectors of the turned part (of each of its halves), and of the
// rest.
bool tiles(const RotaryArgs& a, int interleaved, int64_t V, int64_t esz) {
  return (interleaved ? a.rd % (2 * V) : a.rd / 2 % V) == 0 && a.D % V == 0 && vec_ok(a.q, V, esz) &&
         (a.k.heads == 0 || vec_ok(a.k, V, esz));
}

template <typename T, int V>
int launch_vec(RotaryArgs a, int interleaved, cudaStream_t stream) {
  a.turn_units = a.rd / 2 / V;
  a.units = a.turn_units + (a.D - a.rd + 2 * V - 1) / (2 * V);
  a.items = (a.q.heads + a.k.heads) * a.units;
  // threads: all places of one token in as few even rounds as fit, or those of several tokens where they are few
  a.beside = a.items < 48 ? 128 / a.items : 1;
  const int rounds = (a.items + kMaxThreads - 1) / kMaxThreads;
  const int threads = (a.beside > 1 ? a.beside * a.items + 31 : (a.items + rounds - 1) / rounds + 31) / 32 * 32;
  // tokens a CTA: up to eight a thread, which spreads the angles' cost, once that leaves four CTAs for each SM (131,072
  // tokens: 0.396 ms; 0.402 with sixteen, 0.411 with 32)
  const int64_t n = a.B * a.L;
  const int most = std::min(std::min(+kMaxTokens, 8 * a.beside), kMaxAngles / (a.rd / 2));
  a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(most, n / (4 * 148)));
  a.beside = std::min(a.beside, a.tokens);
  const int64_t grid = (n + a.tokens - 1) / a.tokens;
  if (grid > 0x7fffffffLL) return GSA_ERR_BAD_ARG;
  const size_t smem = (size_t)a.tokens * (a.rd / 2) * sizeof(float2);
  if (interleaved)
    rotary_kernel<T, V, true><<<(unsigned)grid, threads, smem, stream>>>(a);
  else
    rotary_kernel<T, V, false><<<(unsigned)grid, threads, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
}

template <typename T>
int launch_typed(const RotaryArgs& a, int interleaved, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  if (tiles(a, interleaved, kWide, sizeof(T))) return launch_vec<T, kWide>(a, interleaved, stream);
  if (kWide > 4 && tiles(a, interleaved, 4, sizeof(T))) return launch_vec<T, 4>(a, interleaved, stream);
  if (tiles(a, interleaved, 2, sizeof(T))) return launch_vec<T, 2>(a, interleaved, stream);
  return launch_vec<T, 1>(a, interleaved, stream);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

extern "C" int gsa_rotary(int dtype, int64_t B, int64_t L, int32_t D, int32_t rd, const gsa_rotary_side* q,
                          const gsa_rotary_side* k, const int64_t* positions, int64_t pos_bstride, int64_t pos_lstride,
                          const double* inv_freq, const void* cos_tab, const void* sin_tab, int tab_dtype,
                          int64_t tab_ld, int64_t tab_rows, float factor, int interleaved, int inverse,
                          gsa_stream_t stream) {
  if (B < 0 || L < 0 || D < 1 || D > 1024 || rd < 2 || rd > D || rd % 2 ||
      (dtype != GSA_DTYPE_F32 && dtype != GSA_DTYPE_BF16))
    return GSA_ERR_BAD_ARG;
  if (B * L == 0) return GSA_OK;
  if (!q || !side_ok(q, D) || (k && !side_ok(k, D)) || !positions || q->heads + (k ? k->heads : 0) > 1024)
    return GSA_ERR_BAD_ARG;
  if (!inv_freq && (!cos_tab || !sin_tab || tab_rows < 1 || tab_ld < rd / 2 ||
                    (tab_dtype != GSA_DTYPE_F32 && tab_dtype != GSA_DTYPE_BF16)))
    return GSA_ERR_BAD_ARG;
  RotaryArgs a{};
  a.q = side_of(q);
  a.k = side_of(k);
  a.B = B;
  a.L = L;
  a.D = D;
  a.rd = rd;
  a.pos = positions;
  a.pb = pos_bstride;
  a.pl = pos_lstride;
  a.freq = inv_freq;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.tab_dtype = tab_dtype;
  a.tab_ld = tab_ld;
  a.tab_rows = tab_rows;
  a.factor = factor;
  a.inverse = inverse;
  if (!inv_freq) {  // only a position outside the tables is an error of the device's
    const int st = device_error_word(&a.err);
    if (st) return st;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == GSA_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(a, interleaved, s)
                                 : launch_typed<float>(a, interleaved, s);
}
