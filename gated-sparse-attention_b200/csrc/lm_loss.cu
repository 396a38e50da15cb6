// Next-token loss with its gradient: position t of a sequence predicts labels[t + 1]; labels equal to
// ignore_index do not count.
//
//   loss = mean over the counted positions of (log sum_v e^{x_v} - x_target)
//   grad = (softmax(x) - onehot(target)) / count, zero in the rows that do not count
//
// One CTA per row: the row's maximum and sum in one pass (online), then the gradient from a second reading of
// the row, which the L2 holds (148 rows of 128,256 bf16 logits are 38 MB).  So HBM sees each logit once and
// each gradient value once, which bounds it.  Every CTA counts the labels by itself (they sit in L2), so the division
// by the count needs no launch of its own; the rows' losses are added by one CTA in a fixed order.
#include <algorithm>

#include "kernels.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

struct LossArgs {
  int64_t B, L, V;
  const void* logits;
  int64_t xb, xl;
  const int64_t* labels;
  int64_t lb, ll;
  int64_t ignore;
  float* row_loss;  // [B * L]: the loss of the rows that count, 0 for the others
  void* grad;       // or NULL: the loss alone
  int64_t gb, gl;
  float* loss;
  int* err;
};

__device__ __forceinline__ double block_sum_f64(double v, double* ws) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  for (int w = 0; w < kWarps; ++w) t += ws[w];
  return t;
}

// Labels that count: those after the first of each sequence that are not ignore_index.
__device__ __forceinline__ int64_t count_labels(const LossArgs& a, int64_t* ws) {
  int64_t n = 0;
  const int64_t per = a.L - 1, total = a.B * per;
  for (int64_t e = threadIdx.x; e < total; e += kThreads) {
    const int64_t b = e / per, t = e - b * per + 1;
    n += a.labels[b * a.lb + t * a.ll] != a.ignore;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < kWarps; ++w) n += ws[w];
  return n;
}

// (maximum, sum of e^{x - maximum}) of two parts joined; a part without finite values is (-inf, 0).
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float f1 = m == top ? 1.f : expf(m - top), f2 = m2 == top ? 1.f : expf(m2 - top);
  s = s * f1 + s2 * f2;
  m = top;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) lm_loss_kernel(const LossArgs a) {
  __shared__ int64_t cnt_ws[kWarps];
  __shared__ float m_ws[kWarps], s_ws[kWarps];
  const int64_t count = count_labels(a, cnt_ws);
  const float inv_count = count ? 1.0f / (float)count : 0.f;
  for (int64_t r = blockIdx.x; r < a.B * a.L; r += gridDim.x) {
    const int64_t b = r / a.L, t = r - b * a.L;
    const T* x = static_cast<const T*>(a.logits) + b * a.xb + t * a.xl;
    T* g = a.grad ? static_cast<T*>(a.grad) + b * a.gb + t * a.gl : nullptr;
    const int64_t target = t + 1 < a.L ? a.labels[b * a.lb + (t + 1) * a.ll] : a.ignore;
    if (target == a.ignore) {
      if (threadIdx.x == 0) a.row_loss[r] = 0.f;
      if (g)
        for (int64_t i = threadIdx.x; i < a.V; i += kThreads) g[i] = from_float<T>(0.f);
      continue;
    }
    const bool bad = target < 0 || target >= a.V;
    if (bad && threadIdx.x == 0) set_error(a.err, GSA_ERR_INDEX);
    float m = -INFINITY, s = 0.f;
    for (int64_t i = threadIdx.x; i < a.V; i += kThreads) {
      const float v = to_float(x[i]);
      if (v > m) {
        s = s * expf(m - v) + 1.f;
        m = v;
      } else if (v != -INFINITY) {
        s += expf(v - m);
      }
    }
    for (int o = 16; o > 0; o >>= 1)
      join(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      m_ws[threadIdx.x >> 5] = m;
      s_ws[threadIdx.x >> 5] = s;
    }
    __syncthreads();
    m = m_ws[0];
    s = s_ws[0];
    for (int w = 1; w < kWarps; ++w) join(m, s, m_ws[w], s_ws[w]);
    // a label out of range, or a logit of +inf: the row's loss and gradient are NaN
    const float lse = bad || m == INFINITY ? __int_as_float(0x7fc00000) : m + logf(s);
    if (threadIdx.x == 0) a.row_loss[r] = isnan(lse) ? lse : lse - to_float(x[target]);
    if (!g) continue;
    const float inv = isnan(lse) ? lse : inv_count / s;
    for (int64_t i = threadIdx.x; i < a.V; i += kThreads) {
      float p = expf(to_float(x[i]) - m) * inv;
      if (i == target) p -= inv_count;
      g[i] = from_float<T>(p);
    }
  }
}

// The mean of the rows' losses: NaN where no label counts (0 / 0).
__global__ void __launch_bounds__(kThreads) lm_loss_mean_kernel(const LossArgs a) {
  __shared__ int64_t cnt_ws[kWarps];
  __shared__ double ws[kWarps];
  const int64_t count = a.L > 1 ? count_labels(a, cnt_ws) : 0;
  double sum = 0;
  for (int64_t r = threadIdx.x; r < a.B * a.L; r += kThreads) sum += a.row_loss[r];
  sum = block_sum_f64(sum, ws);
  if (threadIdx.x == 0) *a.loss = (float)(sum / (double)count);
}

template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(int64_t n, T* x, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    x[i] = from_float<T>(to_float(x[i]) * f);
}

}  // namespace
}  // namespace gsa

using namespace gsa;

extern "C" {

int gsa_next_token_loss(int dtype, int64_t B, int64_t L, int64_t V, const void* logits, int64_t x_bstride,
                        int64_t x_lstride, const int64_t* labels, int64_t lab_bstride, int64_t lab_lstride,
                        int64_t ignore_index, float* row_loss, float* loss, void* grad, int64_t g_bstride,
                        int64_t g_lstride, gsa_stream_t stream) {
  if ((dtype != GSA_DTYPE_F32 && dtype != GSA_DTYPE_BF16) || B < 0 || L < 0 || V < 1 || !loss) return GSA_ERR_BAD_ARG;
  const int64_t rows = B * L;
  if (rows > 0 && (!logits || !labels || !row_loss || x_bstride < 0 || x_lstride < 0 || lab_bstride < 0 ||
                   lab_lstride < 0 || (grad && (g_lstride < V || (B > 1 && g_bstride < V)))))
    return GSA_ERR_BAD_ARG;
  LossArgs a{B, L, V, logits, x_bstride, x_lstride, labels, lab_bstride, lab_lstride, ignore_index,
             row_loss, grad, g_bstride, g_lstride, loss, nullptr};
  int st = device_error_word(&a.err);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows > 0) {
    const unsigned grid = (unsigned)std::min<int64_t>(rows, 148 * 4);
    if (dtype == GSA_DTYPE_BF16)
      lm_loss_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
    else
      lm_loss_kernel<float><<<grid, kThreads, 0, s>>>(a);
  }
  lm_loss_mean_kernel<<<1, kThreads, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
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
