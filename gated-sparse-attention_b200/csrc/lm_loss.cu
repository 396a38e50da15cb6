// Next-token loss with its gradient: position t of a sequence predicts labels[t + 1]; labels equal to
// ignore_index do not count.
//
//   loss = mean over the counted positions of (log sum_v e^{x_v} - x_target)
//   grad = (softmax(x) - onehot(target)) / count, zero in the rows that do not count
//
// A CTA takes a row (a warp one of up to 4 KB, two to eight lanes one of up to 1 KB): its maximum and sum in one pass (online), then the gradient
// from a second reading, which registers serve for short rows and the L2 for long ones, as far as it holds the rows in flight:
// 48 to 97 MB for rows of up to 320 KB, 148 rows beyond (so rows of more than some 850 KB come from HBM twice).  HBM sees
// each logit 1.24 times for rows of 250 KB, and each gradient value once; rows that do not count are not read at all.
// Exponentials are 2^(x log2 e - M) by one multiply-add (two values an instruction) and one ex2, M the rounded m log2 e:
// M is what the sums and the gradient share, so its rounding, a factor 2^r on all of them, cancels as long as 2^r does not
// leave the range: |r| is half a step of M, 4 up to kFar.  A row whose |M| is larger (masked throughout with any value or
// with -inf, or with a far largest one) is taken by differences first; beside a largest value within kFar, values under
// kLow weigh 0 and are not met at all (a thread that has seen nothing else would be left with an r of its own of
// any size).  Sums are in 32 bits within a row and in 64 across rows; each CTA adds its
// rows in order and one CTA adds the CTAs' sums in order, so a loss is the same bits every time.  8192 x 128256 bf16, every
// row counted: 0.79 ms, 5.4 TB/s; what keeps it from a copy's 6.55 is latency between the two passes of a row (no unit is busy
// for more than about two thirds).  The forms with six pieces in flight and 64 to 256 threads a row spill 16 to 60 bytes a thread.
#include <algorithm>

#include "kernels.cuh"

namespace gsa {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxGrid = 148 * 16;
constexpr int kCounters = 64;         // CTAs of the count kernel
constexpr int64_t kSelfCount = 2048;  // labels up to which every CTA counts for itself
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;
constexpr float kFar = 0x1p27f;   // of M
constexpr float kLow = -0x1p28f;  // of a logit: 1.7e8 under any largest value within kFar; |r| <= 16 down to there

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
  int counted;     // ws->counts holds the count
  uint64_t magic;  // ceil(2^64 / L), 0 for L = 1
};

struct Position {
  int64_t b, t;
};
// Sequence and token of row r < B L: by one multiplication, exact for r L < 2^64.
__device__ __forceinline__ Position position_of(const LossArgs& a, int64_t r) {
  const int64_t b = a.magic ? (int64_t)__umul64hi((uint64_t)r, a.magic) : r;
  return {b, r - b * a.L};
}
// What row r predicts: its label, or ignore_index past the end and for a sequence's last row.
__device__ __forceinline__ int64_t target_of(const LossArgs& a, int64_t r) {
  if (r >= a.B * a.L) return a.ignore;
  const Position p = position_of(a, r);
  return p.t + 1 < a.L ? a.labels[p.b * a.lb + (p.t + 1) * a.ll] : a.ignore;
}

template <typename S>
__device__ __forceinline__ S warp_all_sum(S v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// This CTA's share of the rows that count.
__device__ __forceinline__ int64_t count_labels(const LossArgs& a, int64_t cta, int64_t ctas) {
  int64_t n = 0;
  const int64_t rows = a.B * a.L;
#pragma unroll 4
  for (int64_t r = cta * blockDim.x + threadIdx.x; r < rows; r += ctas * blockDim.x) n += target_of(a, r) != a.ignore;
  return n;
}

__device__ __forceinline__ int64_t block_sum_i64(int64_t n, int64_t* ws) {
  n = warp_all_sum(n);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < blockDim.x >> 5; ++w) n += ws[w];
  return n;
}

// All rows that count, the same in every thread.
__device__ __forceinline__ int64_t total_count(const LossArgs& a, int64_t* ws) {
  if (!a.counted) return block_sum_i64(count_labels(a, 0, 1), ws);
  const int lane = threadIdx.x & 31;
  return warp_all_sum(a.ws->counts[lane] + a.ws->counts[lane + 32]);
}

__global__ void __launch_bounds__(kThreads) lm_loss_count_kernel(const LossArgs a) {
  __shared__ int64_t ws[kWarps];
  const int64_t n = block_sum_i64(count_labels(a, blockIdx.x, gridDim.x), ws);
  if (threadIdx.x == 0) a.ws->counts[blockIdx.x] = n;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two 32-bit values an instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^(x log2 e - M) of two values.
__device__ __forceinline__ uint64_t weight2(uint64_t x, uint64_t neg_m) {
  const float2 t = split(fma2(x, pair_of(kLog2e, kLog2e), neg_m));
  return pair_of(exp2_fast(t.x), exp2_fast(t.y));
}

__device__ __forceinline__ float warp_top(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// A part of a row: M, and the sum of 2^(x log2 e - M) over its values; (-inf, 0) where none is above kLow.
struct Part {
  float m, s;
};
// The lanes of this thread's row, where a warp holds rows of kRow lanes.
template <int kRow>
__device__ __forceinline__ uint32_t row_mask() {
  return kRow >= 32 ? 0xffffffffu : ((1u << (kRow & 31)) - 1u) << ((threadIdx.x & 31) / kRow * kRow);
}
// The parts of kLanes neighbouring lanes (a power of two) as one, the same in each of them.
template <int kLanes>
__device__ __forceinline__ Part join_lanes(Part p) {
  float top = p.m;
  if (kLanes >= 16) {  // of all the warp: the lanes beside hold the same parts
    top = warp_top(top);
  } else {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(row_mask<kLanes>(), top, o));
  }
  p.s *= p.m == top ? 1.f : exp2_fast(p.m - top);  // both may be -inf
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) p.s += __shfl_xor_sync(row_mask<kLanes>(), p.s, o);
  p.m = top;
  return p;
}
// The parts of kRow threads as one, the same in each of them; ws is free again after the CTA's next barrier.
template <int kRow>
__device__ __forceinline__ Part join_row(Part p, Part* ws) {
  if (kRow <= 32) return join_lanes<(kRow < 32 ? kRow : 32)>(p);
  p = join_lanes<32>(p);
  constexpr int kParts = kRow < 64 ? 1 : kRow / 32;
  const int lane = threadIdx.x & 31;
  if (lane == 0) ws[threadIdx.x >> 5] = p;
  __syncthreads();
  return join_lanes<kParts>(ws[lane % kParts]);
}

// 16 bytes of logits: n values as n / 2 pairs.
template <typename T>
struct Piece;
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ uint64_t wide(uint32_t w) {
    return pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void get(const uint4& r, uint64_t* v) {
    v[0] = wide(r.x);
    v[1] = wide(r.y);
    v[2] = wide(r.z);
    v[3] = wide(r.w);
  }
  // A running maximum over pieces, NaN once it has met one.
  uint32_t w;
  __device__ __forceinline__ Piece() : w(0xff80ff80u) {}
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ void meet(const uint4& r) { w = max2(w, max2(max2(r.x, r.y), max2(r.z, r.w))); }
  __device__ __forceinline__ float top() const {
    return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
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
  static __device__ __forceinline__ void get(const uint4& r, uint64_t* v) {
    v[0] = pair_of(__uint_as_float(r.x), __uint_as_float(r.y));
    v[1] = pair_of(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  float m;
  __device__ __forceinline__ Piece() : m(-INFINITY) {}
  __device__ __forceinline__ void meet(const uint4& r) {
    m = max_nan(m, max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)),
                           max_nan(__uint_as_float(r.z), __uint_as_float(r.w))));
  }
  __device__ __forceinline__ float top() const { return m; }
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

// Sum or maximum over the threads of a row, the same value in each of them; ws is free on entry and on return.
template <int kRow, bool kMax>
__device__ __forceinline__ float row_reduce(float v, float* ws) {
#pragma unroll
  for (int o = (kRow < 32 ? kRow : 32) / 2; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(row_mask<kRow>(), v, o);
    v = kMax ? fmaxf(v, w) : v + w;
  }
  if (kRow <= 32) return v;
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = v;
  __syncthreads();
  v = ws[0];
#pragma unroll
  for (int w = 1; w < kRow / 32; ++w) v = kMax ? fmaxf(v, ws[w]) : v + ws[w];
  __syncthreads();
  return v;
}

// A row of |M| past kFar, by differences first, a value at a time.  Rows with a NaN or a +inf, or of -inf alone, come out NaN.
template <typename T, int kRow>
__device__ __noinline__ double far_row(const T* x, T* g, int V, int target, int lane, float inv_count, float* ws) {
  if (kRow > 32) __syncthreads();  // ws has been read
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < V; i += kRow) m = fmaxf(m, to_float(x[i]));
  m = row_reduce<kRow, true>(m, ws);
  for (int i = lane; i < V; i += kRow) s += expf(to_float(x[i]) - m);
  s = row_reduce<kRow, false>(s, ws);
  if (g)
    for (int i = lane; i < V; i += kRow)
      g[i] = from_float<T>(expf(to_float(x[i]) - m) * (inv_count / s) - (i == target ? inv_count : 0.f));
  return (double)logf(s) - ((double)to_float(x[target]) - (double)m);
}

// The loss of a label far below the row's largest, in 64 bits (kept out of line: the registers of the usual case).
__device__ __noinline__ double far_label(float s, float m, float x_target) {
  return ((double)log2f(s) - ((double)x_target * kLog2e - m)) * kLn2;
}

// A row by kRow threads (neighbouring lanes, or the CTA); lane: the thread's number among them.  Returns the row's loss, or
// adds one that 32 bits may not hold to far.
template <typename T, int kRow, int kAhead>
__device__ __forceinline__ float row_loss(const LossArgs& a, int64_t r, int64_t target, int lane, float inv_count,
                                          Part* ws, double& far) {
  constexpr int n = Piece<T>::n;
  const Position pos = position_of(a, r);
  const T* x = static_cast<const T*>(a.logits) + pos.b * a.xb + pos.t * a.xl;
  T* g = a.grad ? static_cast<T*>(a.grad) + pos.b * a.gb + pos.t * a.gl : nullptr;
  const Walk walk(x, g, (int)a.V);
  const uint4* xp = reinterpret_cast<const uint4*>(x + walk.first);
  uint4* gp = reinterpret_cast<uint4*>(g + walk.first);
  if (target == a.ignore) {
    if (g) {
      for (int i = lane; i < walk.pieces; i += kRow) __stcs(gp + i, make_uint4(0, 0, 0, 0));
      for (int e = lane; e < walk.edges; e += kRow) g[walk.edge(e)] = from_float<T>(0.f);
    }
    return 0.f;
  }
  const float nan = __int_as_float(0x7fc00000);
  const bool bad = target < 0 || target >= a.V;
  if (bad && lane == 0) set_error(a.err, GSA_ERR_INDEX);
  const float x_target = bad ? nan : to_float(x[target]);
  const bool once = walk.pieces <= kAhead * kRow;  // the pieces stay in registers between the passes
  float top = -INFINITY;  // the thread's largest value
  Part p{-INFINITY, 0.f};
  uint4 raw[kAhead];
  for (int i0 = lane; i0 < walk.pieces; i0 += kAhead * kRow) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * kRow < walk.pieces) raw[j] = xp[i0 + j * kRow];
    // the largest of all of them first: one rescaling of the sum, and exponentials that wait for nothing
    Piece<T> most;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * kRow < walk.pieces) most.meet(raw[j]);
    const float here = most.top();
    if (here <= kLow) continue;
    if (here > top) {
      top = here;
      const float up = here * kLog2e;
      p.s *= exp2_fast(p.m - up);
      p.m = up;
    }
    const uint64_t neg_m = pair_of(-p.m, -p.m);
    uint64_t sum[n / 2];
#pragma unroll
    for (int k = 0; k < n / 2; ++k) sum[k] = 0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kRow >= walk.pieces) break;
      uint64_t v[n / 2];
      Piece<T>::get(raw[j], v);
#pragma unroll
      for (int k = 0; k < n / 2; ++k) sum[k] = add2(sum[k], weight2(v[k], neg_m));
    }
#pragma unroll
    for (int k = 1; k < n / 2; ++k) sum[0] = add2(sum[0], sum[k]);
    const float2 both = split(sum[0]);
    p.s += both.x + both.y;
  }
  for (int e = lane; e < walk.edges; e += kRow) {
    const float v = to_float(x[walk.edge(e)]);
    if (v <= kLow) continue;
    if (v > top) {
      top = v;
      p.s *= exp2_fast(p.m - v * kLog2e);
      p.m = v * kLog2e;
    }
    p.s += exp2_fast(fmaf(v, kLog2e, -p.m));
  }
  p = join_row<kRow>(p, ws);
  const float m = p.m, s = p.s;
  if (!(fabsf(m) < kFar) && !bad) {
    far += far_row<T, kRow>(x, g, walk.V, (int)target, lane, inv_count, &ws[0].m);
    return 0.f;
  }
  // a label out of range or a NaN: the row's loss and gradient are NaN
  float loss = bad ? nan : (log2f(s) - fmaf(x_target, kLog2e, -m)) * kLn2;
  if (loss == INFINITY) {  // x_target log2 e may leave the range of 32 bits where the loss does not
    far += far_label(s, m, x_target);
    loss = 0.f;
  }
  if (!g) return loss;
  const float inv = isnan(loss) ? loss : inv_count / s;
  const int at = bad ? -1 : (int)target - walk.first;  // among the pieces' values
  const uint64_t neg_m = pair_of(-m, -m), inv2 = pair_of(inv, inv);
  for (int i0 = lane; i0 < walk.pieces; i0 += kAhead * kRow) {
    if (!once) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kRow < walk.pieces) raw[j] = __ldcs(xp + i0 + j * kRow);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kRow;
      if (i >= walk.pieces) break;
      uint64_t v[n / 2];
      Piece<T>::get(raw[j], v);
      float q[n];
#pragma unroll
      for (int k = 0; k < n / 2; ++k) {
        const float2 both = split(mul2(weight2(v[k], neg_m), inv2));
        q[2 * k] = both.x;
        q[2 * k + 1] = both.y;
      }
      __stcs(gp + i, Piece<T>::set(q));
    }
  }
  // the label's value again, one less, by the thread that stored it
  if (at >= 0 && at < walk.pieces * n && at / n % kRow == lane)
    g[target] = from_float<T>(exp2_fast(fmaf(x_target, kLog2e, -m)) * inv - inv_count);
  for (int e = lane; e < walk.edges; e += kRow) {
    const int i = walk.edge(e);
    float q = exp2_fast(fmaf(to_float(x[i]), kLog2e, -m)) * inv;
    if (i == (int)target) q -= inv_count;
    g[i] = from_float<T>(q);
  }
  return loss;
}

// kThreads threads, kRow a row; a row's label is loaded while the one before it is worked on.
template <typename T, int kRow, int kCta, int kCtas, int kAhead>
__global__ void __launch_bounds__(kCta, kCtas) lm_loss_kernel(const LossArgs a) {
  constexpr int kRows = kCta / kRow, kW = kCta / 32;
  __shared__ int64_t cnt_ws[kW];
  __shared__ Part row_ws[2][kW];
  __shared__ double sum_ws[kW];
  chain_wait();
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kRow;
  const int64_t step = (int64_t)gridDim.x * kRows, rows = a.B * a.L;
  int64_t target = target_of(a, r);
  const int64_t count = total_count(a, cnt_ws);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.ws->count = count;
  const float inv_count = count ? 1.0f / (float)count : 0.f;
  double sum = 0;
  // two of row_ws in turn: a row's barrier is what frees the one before it
  for (int turn = 0; r < rows; r += step) {
    const int64_t next = target_of(a, r + step);
    const float loss = row_loss<T, kRow, kAhead>(a, r, target, threadIdx.x % kRow, inv_count, row_ws[turn], sum);
    sum += loss;
    if (target != a.ignore) turn ^= 1;
    target = next;
  }
  if (kRow <= 32) {
#pragma unroll
    for (int o = kRow; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) sum_ws[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kW; ++w) sum += sum_ws[w];
  }
  if (threadIdx.x == 0) a.ws->sums[blockIdx.x] = sum;
}

// The mean of the rows' losses: NaN where no label counts (0 / 0).
__global__ void __launch_bounds__(256) lm_loss_mean_kernel(const LossArgs a, int parts) {
  __shared__ double ws[8];
  chain_wait();
  double sum = 0;
  for (int i = threadIdx.x; i < parts; i += 256) sum += a.ws->sums[i];
  sum = warp_all_sum(sum);
  if ((threadIdx.x & 31) == 0) ws[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  sum = 0;
  for (int w = 0; w < 8; ++w) sum += ws[w];
  *a.loss = (float)(sum / (double)(parts ? a.ws->count : 0));
}

// x *= factor.  The gradient has been rounded to its type before its factor is known (the loss is formed first), so a factor that is
// no power of two rounds it a second time: by up to a half step more in bf16 than a gradient formed with the factor.
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(int64_t n, T* x, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    x[i] = from_float<T>(to_float(x[i]) * f);
}

template <typename T, int kRow, int kCta, int kCtas, int kAhead>
cudaError_t launch_rows(const LossArgs& a, int* grid, cudaStream_t s) {
  constexpr int kRows = kCta / kRow;
  *grid = (int)std::min<int64_t>((a.B * a.L + kRows - 1) / kRows, 148 * kCtas);
  return launch_chained(lm_loss_kernel<T, kRow, kCta, kCtas, kAhead>, *grid, kCta, 0, s, a);
}

// Threads a row: 1024 threads an SM in any case, on as many rows as their second reading finds in L2 -- 16 rows an SM of
// up to 20 KB (48 MB in flight), 8 of up to 48 KB, 4 of up to 112 KB, 2 of up to 320 KB, then 1.  Measured in TB/s with
// twice the threads a row | as here | with half: 8 KB rows 4.1 | 4.6 | -, 40 KB 4.8 | 5.1 | 4.6, 98 KB 4.6 | 4.8 | 4.4,
// 250 KB 4.9 | 5.0 | 4.4, 501 KB (fp32) - | 5.1 | 4.5.  Short rows take lanes of a warp, with four pieces of 16 bytes in
// flight (eight spill; us here | with eight lanes, or a warp over 1 KB, and eight pieces: 131,072 x 16 bf16 12 | 31, 71,652 x 52 fp32
// 13 | 21, 65,536 x 384 fp32 47 | 63, 131,072 x 333 bf16 57 | 57).
template <typename T>
cudaError_t launch_loss(const LossArgs& a, int* grid, cudaStream_t s) {
  const int64_t bytes = a.V * (int64_t)sizeof(T);
  if (bytes <= 64) return launch_rows<T, 2, 256, 4, 2>(a, grid, s);
  if (bytes <= 256) return launch_rows<T, 4, 256, 4, 4>(a, grid, s);
  if (bytes <= 1024) return launch_rows<T, 8, 256, 4, 4>(a, grid, s);
  if (bytes <= 4096) return launch_rows<T, 32, 256, 4, 4>(a, grid, s);
  if (bytes <= 20 << 10) return launch_rows<T, 64, 64, 16, 6>(a, grid, s);
  if (bytes <= 48 << 10) return launch_rows<T, 128, 128, 8, 6>(a, grid, s);
  if (bytes <= 112 << 10) return launch_rows<T, 256, 256, 4, 6>(a, grid, s);
  if (bytes <= 320 << 10) return launch_rows<T, 512, 512, 2, 6>(a, grid, s);
  return launch_rows<T, 1024, 1024, 1, 6>(a, grid, s);
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
             static_cast<Workspace*>(workspace), grad, g_bstride, g_lstride, loss, nullptr, rows > kSelfCount,
             L > 1 ? ~0ull / (uint64_t)L + 1 : 0};
  int st = device_error_word(&a.err);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int grid = 0;
  if (rows > 0) {
    if (a.counted) {
      lm_loss_count_kernel<<<kCounters, kThreads, 0, s>>>(a);
      if (cudaGetLastError() != cudaSuccess) return GSA_ERR_LAUNCH;
    }
    const cudaError_t e = dtype == GSA_DTYPE_BF16 ? launch_loss<__nv_bfloat16>(a, &grid, s)
                                                  : launch_loss<float>(a, &grid, s);
    if (e != cudaSuccess) return GSA_ERR_LAUNCH;
  }
  return launch_chained(lm_loss_mean_kernel, 1, 256, 0, s, a, grid) == cudaSuccess ? GSA_OK : GSA_ERR_LAUNCH;
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
