// Next-token loss with its gradient: position t of a sequence predicts labels[t + 1]; labels equal to
// ignore_index do not count.
//
//   loss = mean over the counted positions of (log sum_v e^{x_v} - x_target)
//   grad = (softmax(x) - onehot(target)) / count, zero in the rows that do not count
//
// A CTA takes a row (a warp takes one of up to kWarpRow values): its maximum and sum in one pass (online), then the
// gradient from a second reading, which the L2 serves -- the rows in flight, 2 for each SM, are 76 MB of 128,256
// bf16 logits.  So HBM sees each logit once and each gradient value once, which bounds it.
//
// Exponentials are 2^((x - m) log2 e) with the difference first: rows masked with the type's lowest value keep
// their weights, which x log2 e - m log2 e would lose to overflow.  Sums are in 32 bits within a row and in 64
// across rows; each CTA adds its rows in order and one CTA adds the CTAs' sums in order, so a loss is the same bits
// every time.
#include <algorithm>

#include "kernels.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPerSm = 2;
constexpr int kMaxGrid = 148 * 4;
constexpr int kCounters = 64;         // CTAs of the count kernel
constexpr int64_t kSelfCount = 16384;  // labels up to which every CTA counts for itself
constexpr int kWarpRow = 2048;
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;

struct Workspace {
  double sums[kMaxGrid];      // of each CTA's rows
  int64_t counts[kCounters];  // of the count kernel's CTAs
  int64_t count;
};

struct LossArgs {
  int64_t B, L, V;
  const void* logits;
  int64_t xb, xl;
  const int64_t* labels;
  int64_t lb, ll;
  int64_t ignore;
  Workspace* ws;
  void* grad;  // or NULL: the loss alone
  int64_t gb, gl;
  float* loss;
  int* err;
  int counted;  // ws->counts holds the count
};

template <typename S>
__device__ __forceinline__ S warp_all_sum(S v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// This CTA's share of the labels that count: those after the first of each sequence that are not ignore_index.
__device__ __forceinline__ int64_t count_labels(const LossArgs& a, int64_t cta, int64_t ctas) {
  int64_t n = 0;
  const int64_t per = a.L - 1, total = a.B * per;
  for (int64_t e = cta * kThreads + threadIdx.x; e < total; e += ctas * kThreads) {
    const int64_t b = e / per, t = e - b * per + 1;
    n += a.labels[b * a.lb + t * a.ll] != a.ignore;
  }
  return n;
}

__device__ __forceinline__ int64_t block_sum_i64(int64_t n, int64_t* ws) {
  n = warp_all_sum(n);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) n += ws[w];
  return n;
}

__global__ void __launch_bounds__(kThreads) lm_loss_count_kernel(const LossArgs a) {
  __shared__ int64_t ws[kWarps];
  const int64_t n = block_sum_i64(count_labels(a, blockIdx.x, gridDim.x), ws);
  if (threadIdx.x == 0) a.ws->counts[blockIdx.x] = n;
}

// e^d for d <= 0.
__device__ __forceinline__ float exp_neg(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * kLog2e));
  return r;
}

// (maximum, sum of e^{x - maximum}) of two parts joined; a part without values above -inf is (-inf, 0).
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float f1 = m == top ? 1.f : exp_neg(m - top), f2 = m2 == top ? 1.f : exp_neg(m2 - top);
  s = s * f1 + s2 * f2;
  m = top;
}

// 16 bytes of logits as floats.
template <typename T>
struct Piece;
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void get(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 set(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Piece<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void get(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x);
    v[1] = __uint_as_float(r.y);
    v[2] = __uint_as_float(r.z);
    v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 set(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};

// How a row's V values are walked: whole 16-byte pieces from the first aligned one, and the values before and
// after them one by one.  Where x and grad are not aligned alike all values go one by one.
struct Walk {
  int first, pieces, edges, V;
  template <typename T>
  __device__ __forceinline__ Walk(const T* x, const T* g, int v) : V(v) {
    constexpr int n = 16 / sizeof(T);
    const uint32_t ax = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16), ag = (uint32_t)(reinterpret_cast<uintptr_t>(g) % 16);
    first = min((int)((16 - ax) % 16 / sizeof(T)), v);
    pieces = g && ax != ag ? 0 : (v - first) / n;
    edges = v - pieces * n;
    if (pieces == 0) first = v;
  }
  __device__ __forceinline__ int edge(int e) const { return e < first ? e : V - edges + e; }  // e < edges
};

// Adds a value to the thread's running (m, s).
__device__ __forceinline__ void add_value(float& m, float& s, float v) {
  if (v > m) {
    s *= exp_neg(m - v);
    m = v;
  }
  if (v != -INFINITY) s += exp_neg(v - m);
}

// A row by kRow threads (a warp, or the CTA); lane: the thread's number among them.  Returns the row's loss.
template <typename T, int kRow>
__device__ __forceinline__ float row_loss(const LossArgs& a, int64_t r, int lane, float inv_count, float* m_ws,
                                          float* s_ws) {
  constexpr int n = Piece<T>::n, kAhead = 4;
  const int64_t b = r / a.L, t = r - b * a.L;
  const T* x = static_cast<const T*>(a.logits) + b * a.xb + t * a.xl;
  T* g = a.grad ? static_cast<T*>(a.grad) + b * a.gb + t * a.gl : nullptr;
  const Walk walk(x, g, (int)a.V);
  const uint4* xp = reinterpret_cast<const uint4*>(x + walk.first);
  uint4* gp = reinterpret_cast<uint4*>(g + walk.first);
  const int64_t target = t + 1 < a.L ? a.labels[b * a.lb + (t + 1) * a.ll] : a.ignore;
  if (target == a.ignore) {
    if (g) {
      for (int i = lane; i < walk.pieces; i += kRow) __stcs(gp + i, make_uint4(0, 0, 0, 0));
      for (int e = lane; e < walk.edges; e += kRow) g[walk.edge(e)] = from_float<T>(0.f);
    }
    return 0.f;
  }
  const bool bad = target < 0 || target >= a.V;
  if (bad && lane == 0) set_error(a.err, GSA_ERR_INDEX);
  float m = -INFINITY, s = 0.f;
  for (int i0 = lane; i0 < walk.pieces; i0 += kAhead * kRow) {
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * kRow < walk.pieces) raw[j] = xp[i0 + j * kRow];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kRow >= walk.pieces) break;
      float v[n];
      Piece<T>::get(raw[j], v);
      float top = v[0];
#pragma unroll
      for (int k = 1; k < n; ++k) top = fmaxf(top, v[k]);
      if (top > m) {
        s *= exp_neg(m - top);
        m = top;
      }
      if (top == -INFINITY) continue;  // all of them masked: their weight is 0, and m may be -inf still
#pragma unroll
      for (int k = 0; k < n; ++k) s += exp_neg(v[k] - m);
    }
  }
  for (int e = lane; e < walk.edges; e += kRow) add_value(m, s, to_float(x[walk.edge(e)]));
  for (int o = 16; o > 0; o >>= 1)
    join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if (kRow > 32) {
    __syncthreads();  // the last row's parts have been read
    if ((threadIdx.x & 31) == 0) {
      m_ws[threadIdx.x >> 5] = m;
      s_ws[threadIdx.x >> 5] = s;
    }
    __syncthreads();
    m = m_ws[0];
    s = s_ws[0];
#pragma unroll
    for (int w = 1; w < kRow / 32; ++w) join(m, s, m_ws[w], s_ws[w]);
  }
  // a label out of range, a NaN or a logit of +inf: the row's loss and gradient are NaN
  const float d = bad || m == INFINITY ? __int_as_float(0x7fc00000) : m - to_float(x[target]);
  const float loss = d + logf(s);
  if (!g) return loss;
  const float inv = isnan(loss) ? loss : inv_count / s;
  const int at = (int)target - walk.first;  // in 16-byte pieces' values
  for (int i0 = lane; i0 < walk.pieces; i0 += kAhead * kRow) {
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * kRow < walk.pieces) raw[j] = __ldcs(xp + i0 + j * kRow);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kRow;
      if (i >= walk.pieces) break;
      float v[n];
      Piece<T>::get(raw[j], v);
#pragma unroll
      for (int k = 0; k < n; ++k) v[k] = exp_neg(v[k] - m) * inv;
      const int k0 = at - i * n;
      if (k0 >= 0 && k0 < n) {
#pragma unroll
        for (int k = 0; k < n; ++k)
          if (k == k0) v[k] -= inv_count;
      }
      __stcs(gp + i, Piece<T>::set(v));
    }
  }
  for (int e = lane; e < walk.edges; e += kRow) {
    const int i = walk.edge(e);
    float p = exp_neg(to_float(x[i]) - m) * inv;
    if (i == (int)target) p -= inv_count;
    g[i] = from_float<T>(p);
  }
  return loss;
}

template <typename T, int kRow>
__global__ void __launch_bounds__(kThreads, kPerSm) lm_loss_kernel(const LossArgs a) {
  __shared__ int64_t cnt_ws[kWarps];
  __shared__ float m_ws[kWarps], s_ws[kWarps];
  __shared__ double sum_ws[kWarps];
  chain_wait();
  int64_t count = 0;
  if (a.counted) {
    for (int i = 0; i < kCounters; ++i) count += a.ws->counts[i];
  } else {
    count = block_sum_i64(count_labels(a, 0, 1), cnt_ws);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws->count = count;
  const float inv_count = count ? 1.0f / (float)count : 0.f;
  constexpr int kRows = kThreads / kRow;
  const int64_t rows = a.B * a.L;
  double sum = 0;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kRow; r < rows; r += (int64_t)gridDim.x * kRows)
    sum += row_loss<T, kRow>(a, r, threadIdx.x % kRow, inv_count, m_ws, s_ws);
  if (kRow == 32) {
    if ((threadIdx.x & 31) == 0) sum_ws[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kWarps; ++w) sum += sum_ws[w];
  }
  if (threadIdx.x == 0) a.ws->sums[blockIdx.x] = sum;
}

// The mean of the rows' losses: NaN where no label counts (0 / 0).
__global__ void __launch_bounds__(32) lm_loss_mean_kernel(const LossArgs a, int parts) {
  chain_wait();
  double sum = 0;
  for (int i = threadIdx.x; i < parts; i += 32) sum += a.ws->sums[i];
  sum = warp_all_sum(sum);
  if (threadIdx.x == 0) *a.loss = (float)(sum / (double)(parts ? a.ws->count : 0));
}

template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(int64_t n, T* x, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    x[i] = from_float<T>(to_float(x[i]) * f);
}

template <typename T>
cudaError_t launch_rows(const LossArgs& a, int* grid, cudaStream_t s) {
  const int64_t rows = a.B * a.L;
  if (a.V <= kWarpRow) {
    *grid = (int)std::min<int64_t>((rows + kWarps - 1) / kWarps, 148 * kPerSm);
    return launch_chained(lm_loss_kernel<T, 32>, *grid, kThreads, 0, s, a);
  }
  *grid = (int)std::min<int64_t>(rows, 148 * kPerSm);
  return launch_chained(lm_loss_kernel<T, kThreads>, *grid, kThreads, 0, s, a);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

extern "C" {

int64_t gsa_next_token_loss_workspace_size(void) { return (int64_t)sizeof(Workspace); }

int gsa_next_token_loss(int dtype, int64_t B, int64_t L, int64_t V, const void* logits, int64_t x_bstride,
                        int64_t x_lstride, const int64_t* labels, int64_t lab_bstride, int64_t lab_lstride,
                        int64_t ignore_index, float* loss, void* grad, int64_t g_bstride, int64_t g_lstride,
                        void* workspace, int64_t workspace_bytes, gsa_stream_t stream) {
  if ((dtype != GSA_DTYPE_F32 && dtype != GSA_DTYPE_BF16) || B < 0 || L < 0 || V < 1 || V > (1 << 30) || !loss)
    return GSA_ERR_BAD_ARG;
  const int64_t rows = B * L;
  if (rows > 0 && (!logits || !labels || x_bstride < 0 || x_lstride < 0 || lab_bstride < 0 || lab_lstride < 0 ||
                   (grad && (g_lstride < V || (B > 1 && g_bstride < V)))))
    return GSA_ERR_BAD_ARG;
  if (!workspace || workspace_bytes < (int64_t)sizeof(Workspace) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return GSA_ERR_WORKSPACE;
  LossArgs a{B, L, V, logits, x_bstride, x_lstride, labels, lab_bstride, lab_lstride, ignore_index,
             static_cast<Workspace*>(workspace), grad, g_bstride, g_lstride, loss, nullptr, rows > kSelfCount};
  int st = device_error_word(&a.err);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int grid = 0;
  if (rows > 0) {
    if (a.counted) {
      lm_loss_count_kernel<<<kCounters, kThreads, 0, s>>>(a);
      if (cudaGetLastError() != cudaSuccess) return GSA_ERR_LAUNCH;
    }
    const cudaError_t e = dtype == GSA_DTYPE_BF16 ? launch_rows<__nv_bfloat16>(a, &grid, s)
                                                  : launch_rows<float>(a, &grid, s);
    if (e != cudaSuccess) return GSA_ERR_LAUNCH;
  }
  return launch_chained(lm_loss_mean_kernel, 1, 32, 0, s, a, grid) == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
}

int gsa_scale(int dtype, int64_t n, void* x, const float* factor, gsa_stream_t stream) {
  if ((dtype != GSA_DTYPE_F32 && dtype != GSA_DTYPE_BF16) || n < 0) return GSA_ERR_BAD_ARG;
  if (n == 0) return GSA_OK;
  if (!x || !factor) return GSA_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 8);
  if (dtype == GSA_DTYPE_BF16)
    scale_kernel<<<grid, 256, 0, s>>>(n, static_cast<__nv_bfloat16*>(x), factor);
  else
    scale_kernel<<<grid, 256, 0, s>>>(n, static_cast<float*>(x), factor);
  return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
}

}  // extern "C"
