// Rotary positions on q and k: y = R(p) x on the first rd values of every head, the rest passed through.
//
//   angle_i = p f_i,  c_i = m cos(angle_i),  s_i = m sin(angle_i)   (m: the attention factor)
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s;  backward (the transpose): s -> -s
//   half pairs: (x_i, x_{i + rd/2});  interleaved pairs: (x_{2i}, x_{2i+1})
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there, so that far positions keep their
// angle (p f of 2^20 radians in 32 bits is off by 2^-4); sine and cosine of the fraction are 32-bit.  A CTA takes
// a few tokens, evaluates each token's rd/2 angles once into shared memory (all its heads share them) and
// then streams the tokens' heads.  Bound by the bytes of q and k, read once and written once.
#include <algorithm>

#include "kernels.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;
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
  int units;   // of a head: pairs, then pass-through values
  uint32_t m_units, m_heads;
  int* err;
};

// n / d for n * d < 2^32 with m = ceil(2^32 / d); d = 1 has no 32-bit m and is passed as m = 0.
__device__ __forceinline__ uint32_t fast_div(uint32_t n, uint32_t m) { return m ? __umulhi(n, m) : n; }

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

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 angles[];
  __shared__ int64_t base[kMaxTokens][4];  // element offsets of the token: q in, q out, k in, k out
  const int half = a.rd / 2;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n_tok = (int)min((int64_t)a.tokens, a.B * a.L - t0);
  if ((int)threadIdx.x < n_tok) {
    const int64_t t = t0 + threadIdx.x, b = t / a.L, l = t - b * a.L;
    base[threadIdx.x][0] = b * a.q.ib + l * a.q.il;
    base[threadIdx.x][1] = b * a.q.ob + l * a.q.ol;
    base[threadIdx.x][2] = b * a.k.ib + l * a.k.il;
    base[threadIdx.x][3] = b * a.k.ob + l * a.k.ol;
  }
  for (int e = threadIdx.x; e < n_tok * half; e += kThreads) {
    const int64_t t = t0 + e / half, b = t / a.L, l = t - b * a.L;
    angles[e] = angle_of(a, a.pos[b * a.pb + l * a.pl], e % half);
  }
  __syncthreads();
  const int heads = a.q.heads + a.k.heads;
  const uint32_t items = (uint32_t)n_tok * heads * a.units;
  for (uint32_t it = threadIdx.x; it < items; it += kThreads) {
    const uint32_t row = fast_div(it, a.m_units), u = it - row * a.units;
    const uint32_t tok = fast_div(row, a.m_heads), h = row - tok * heads;
    const bool is_k = (int)h >= a.q.heads;
    const Side& s = is_k ? a.k : a.q;
    const int hh = is_k ? h - a.q.heads : h;
    const T* in = static_cast<const T*>(s.in) + base[tok][is_k ? 2 : 0] + hh * s.ih;
    T* out = static_cast<T*>(s.out) + base[tok][is_k ? 3 : 1] + hh * s.oh;
    if ((int)u < half) {
      const int i0 = kInterleaved ? 2 * u : u, i1 = kInterleaved ? 2 * u + 1 : u + half;
      const float2 cs = angles[tok * half + u];
      const float x0 = to_float(in[i0]), x1 = to_float(in[i1]);
      out[i0] = from_float<T>(turn0(x0, x1, cs));
      out[i1] = from_float<T>(turn1(x0, x1, cs));
    } else {
      const int i = a.rd + (u - half);
      out[i] = in[i];
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

uint32_t magic(uint32_t d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); }

template <typename T>
int launch_typed(const RotaryArgs& a, int interleaved, cudaStream_t stream) {
  const int64_t T_all = a.B * a.L, grid = (T_all + a.tokens - 1) / a.tokens;
  if (grid > 0x7fffffffLL) return GSA_ERR_BAD_ARG;
  const size_t smem = (size_t)a.tokens * (a.rd / 2) * sizeof(float2);
  if (interleaved)
    rotary_kernel<T, true><<<(unsigned)grid, kThreads, smem, stream>>>(a);
  else
    rotary_kernel<T, false><<<(unsigned)grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
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
  int st = device_error_word(&a.err);
  if (st) return st;
  const int heads = a.q.heads + a.k.heads;
  a.units = rd / 2 + (D - rd);
  const int per_token = heads * a.units;
  a.tokens = std::max(1, std::min(std::min((int)kMaxTokens, kMaxAngles / (rd / 2)), (4 * kThreads + per_token - 1) / per_token));
  a.m_units = magic(a.units);
  a.m_heads = magic(heads);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == GSA_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(a, interleaved, s)
                                 : launch_typed<float>(a, interleaved, s);
}
